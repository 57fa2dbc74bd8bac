"""What the paged operators report, wherever they were called."""
import pytest
import torch

gpu = pytest.mark.gpu


def bad_free():
    """A free of a slot outside, on a cache of its own: reported as 11."""
    from thunderworld_b200 import PagedCache
    cache = PagedCache(4, 4, 1, 64, sequences=2, max_tokens=16)
    slots = torch.tensor([5], dtype=torch.int32, device='cuda')
    torch.cuda.synchronize()
    return lambda: cache.free(slots), cache


@gpu
def test_a_status_word_made_in_inference_mode_is_reset_outside(monkeypatch):
    from thunderworld_b200 import ops
    monkeypatch.setattr(ops, '_workspaces', {})
    monkeypatch.setattr(ops, '_status_words', {})
    with torch.inference_mode():
        free, cache = bad_free()
        free()
    with pytest.raises(RuntimeError, match='outside'):
        cache.check()
    ops.reset_device_status()
    assert ops.device_status() == 0
    torch.cuda.synchronize()


@gpu
def test_status_of_a_call_on_another_stream():
    """check() and device_status() wait for all streams of the device, reset_device_status() leaves nothing to a later moment."""
    from thunderworld_b200 import ops
    free, cache = bad_free()
    cache.check()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)                     # some 100 ms
        free()
    with pytest.raises(RuntimeError, match='outside'):
        cache.check()
    torch.cuda._sleep(200_000_000)
    ops.reset_device_status()
    with torch.cuda.stream(side):
        free()
    assert ops.device_status() == 11
    ops.reset_device_status()
    with torch.cuda.stream(side):
        assert ops.device_status() == 0
