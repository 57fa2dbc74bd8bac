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
