"""A DiTModel's blocks as modules: forward(x, mod) returns x, whoever calls it, so that hooks on a block see x and a block can be
replaced by a module that takes and returns the same. What the model computes does not depend on it, to the bit."""
import pytest
import torch
from test_gpu_dit_engine import make_inputs

gpu = pytest.mark.gpu


def build(blocks=4):
    from thunderworld_b200.cosmos.dit import DiTConfig, DiTModel
    from thunderworld_b200.cosmos.engine import StepEngine
    from thunderworld_b200.cosmos.settings import RunConfig
    cfg = DiTConfig(hidden=256, heads=2, ffn=512, blocks=blocks, seed=1)
    engine = StepEngine(RunConfig())
    model = DiTModel(cfg, engine)
    x, mod = make_inputs(cfg, 0)
    engine.warm_schedule(model, x=x, mod=mod)
    return model, x, mod


class Counting(torch.nn.Module):
    """A block in the place of another one, by the signature that blocks have."""

    def __init__(self, block):
        super().__init__()
        self.block, self.calls = block, 0

    def forward(self, x, mod):
        self.calls += 1
        return self.block(x, mod)


@gpu
@pytest.mark.parametrize('at', [(0,), (1,), (3,), (1, 2), (0, 1, 2, 3)])
def test_hooks_see_the_residual_stream(at):
    model, x, mod = build()
    with torch.no_grad():
        want = model(x, mod)
        stream, states = x.clone(), []
        for i, block in enumerate(model.blocks):
            assert block(stream, mod.permute(1, 2, 0, 3).contiguous()[i]) is stream
            states.append(stream.clone())
        seen, entered, handles = {}, {}, []
        for i in at:
            handles.append(model.blocks[i].register_forward_hook(lambda m, a, y, i=i: seen.update({i: y.clone()})))
            handles.append(model.blocks[i].register_forward_pre_hook(lambda m, a, i=i: entered.update({i: a[0].clone()})))
        got = model(x, mod)
        assert torch.equal(got, want) and sorted(seen) == sorted(at)
        for i in at:
            assert torch.equal(seen[i], states[i]) and torch.equal(entered[i], states[i - 1] if i else x)
        for h in handles:
            h.remove()
        seen.clear()
        assert torch.equal(model(x, mod), want) and not seen


@gpu
def test_global_hooks_see_every_block():
    from thunderworld_b200.cosmos.dit import DiTBlock
    model, x, mod = build()
    with torch.no_grad():
        want, seen = model(x, mod), []
        handle = torch.nn.modules.module.register_module_forward_hook(lambda m, a, y: seen.append(y) if isinstance(m, DiTBlock) else None)
        try:
            got = model(x, mod)
        finally:
            handle.remove()
    assert torch.equal(got, want) and len(seen) == 4 and all(y.shape == x.shape for y in seen)


@gpu
@pytest.mark.parametrize('at', [0, 2, 3])
def test_a_replaced_block(at):
    model, x, mod = build()
    with torch.no_grad():
        want = model(x, mod)
        model.blocks[at] = Counting(model.blocks[at])
        assert torch.equal(model(x, mod), want) and model.blocks[at].calls == 1
        model.blocks[at] = model.blocks[at].block
        inner = model.blocks[at].forward
        model.blocks[at].forward = lambda x, mod: inner(x, mod).clone()      # another tensor than the one it was given
        assert torch.equal(model(x, mod), want)
        model.blocks[at].forward = lambda x, mod: torch.zeros_like(x)
        assert not torch.equal(model(x, mod), want)


@gpu
def test_a_modulation_that_requires_gradients():
    """The blocks only read it; no gradient reaches it, as none ever did."""
    model, x, mod = build(2)
    with torch.no_grad():
        want = model(x, mod)
    got = model(x, mod.clone().requires_grad_())
    assert torch.equal(got, want) and not got.requires_grad
    stream = x.clone()
    assert model.blocks[0](stream, mod.permute(1, 2, 0, 3).contiguous()[0].requires_grad_()) is stream and not stream.requires_grad
    with pytest.raises(RuntimeError, match='inference'):
        model(x.clone().requires_grad_(), mod)
