"""The gated residual fused with the norms around it (`ops.gate_residual_norm_`) against its formula in 64 bits, and bit for
bit against the two kernels that it stands for.

Tolerances: x' and h are rounded to bf16 once, at most 2^-8 of the value (half a step); h is computed from the rounded x',
which both sides share when they round to the same side. The 32-bit part before a rounding carries a few 2^-24 per operation
and, through the sum of squares of up to 12288 terms held in 32 bits, less than 2^-16 relative; together under 2^-15. An x'
next to a rounding border may then fall to the other side: a whole step, 2^-7, in x' and in that element of h, and with shift
and scale h sees it times (1 + scale). So: |error of x'| <= 2^-7 |x'| + cancellation (2^-22 of the summands), h likewise."""
import pytest
import torch

gpu = pytest.mark.gpu
STEP = 2. ** -7


def formula(x, y, gate, post, post_weight, rs, weight, shift, scale, eps, rounded=None):
    x, y = x.double(), y.double()
    z = y
    if post:
        z = y / (y.square().mean(-1, keepdim=True) + eps).sqrt()
        if post_weight is not None:
            z = z * post_weight.double()
    new = rs * x + (z if gate is None else gate.double()[:, None] * z)
    size = (rs * x).abs() + (z if gate is None else gate.double()[:, None] * z).abs()
    held = (new.bfloat16() if rounded is None else rounded).double()
    h = held / (held.square().mean(-1, keepdim=True) + eps).sqrt()
    if weight is not None:
        h = h * weight.double()
    hsize = h.abs()
    if scale is not None:
        hsize = (h * (1 + scale.double()[:, None])).abs() + shift.double()[:, None].abs()
        h = h * (1 + scale.double()[:, None]) + shift.double()[:, None]
    return new, size, h, hsize


def inputs(b, t, n, seed, device='cuda'):
    g = torch.Generator().manual_seed(seed)
    r = lambda *s: torch.randn(*s, generator=g).bfloat16().to(device)  # noqa: E731
    return dict(x=r(b, t, n), y=r(b, t, n), gate=r(b, n), post_weight=r(n), weight=r(n), shift=r(b, n), scale=r(b, n))


@gpu
@pytest.mark.parametrize('b,t,n', [(1, 1, 8), (2, 1, 4096), (3, 7, 2040), (2, 33, 2048), (1, 300, 6144), (1, 5, 16384), (2, 19, 4104)])
@pytest.mark.parametrize('post', [None, 'plain', 'weighted'])
@pytest.mark.parametrize('modulate,gated', [(False, True), (True, True), (False, False)])
def test_formula(b, t, n, post, modulate, gated):
    from thunderworld_b200 import ops
    v = inputs(b, t, n, b * 1000 + t + n)
    gate = v['gate'] if gated else None
    weight = v['weight'] if not modulate else None
    shift, scale = (v['shift'], v['scale']) if modulate else (None, None)
    pw, rs = (v['post_weight'] if post == 'weighted' else None), (1. if post is None else .625)
    x = v['x'].clone()
    h, stats = ops.gate_residual_norm_(x, v['y'], gate, post_norm=post is not None, post_weight=pw, residual_scale=rs, weight=weight,
                                       shift=shift, scale=scale, eps=1e-6, want_factor=True, return_stats=True)
    new, size, want, hsize = formula(v['x'], v['y'], gate, post is not None, pw, rs, weight, shift, scale, 1e-6, rounded=x)
    assert (x.double() - new).abs().le(STEP * new.abs() + 2 ** -15 * size).all()
    assert (h.double() - want).abs().le(STEP * want.abs() + 2 ** -15 * hsize).all()
    top = h.float().abs().max()
    assert stats[1].item() == top.item() and abs(stats[0].item() - top.item() / 2688) <= 2 ** -23 * stats[0].item()


@gpu
@pytest.mark.parametrize('b,t,n', [(2, 3840, 4096), (2, 200, 256), (1, 9, 6144), (3, 5, 8), (1, 65, 16384)])
@pytest.mark.parametrize('weighted', [False, True])
def test_bits_of_the_two_kernels(b, t, n, weighted):
    from thunderworld_b200 import ops
    v = inputs(b, t, n, 3)
    weight = v['weight'] if weighted else None
    x0, x1 = v['x'].clone(), v['x'].clone()
    ops.gate_residual_(x0, v['gate'], v['y'])
    h0, f0 = ops.rms_norm(x0, weight, shift=v['shift'], scale=v['scale'], want_factor=True)
    for _ in range(2):                                            # the scratch comes back zeroed
        x1.copy_(v['x'])
        h1, f1 = ops.gate_residual_norm_(x1, v['y'], v['gate'], weight=weight, shift=v['shift'], scale=v['scale'], want_factor=True)
        assert torch.equal(x0, x1) and torch.equal(h0, h1) and torch.equal(f0, f1)


@gpu
def test_zero_rows_and_infinities_stay_in_their_rows():
    from thunderworld_b200 import ops
    v = inputs(1, 6, 512, 8)
    v['x'][0, 1], v['y'][0, 1] = 0, 0                              # an all-zero row: rsqrt(eps) times zero
    v['y'][0, 3, 7] = float('inf')
    v['y'][0, 4, 9] = float('nan')
    x = v['x'].clone()
    h = ops.gate_residual_norm_(x, v['y'], v['gate'], post_norm=True)
    assert not x[0, 1].any() and not h[0, 1].any()
    clean = [0, 1, 2, 5]
    assert torch.isfinite(h[0, clean].float()).all() and torch.isfinite(x[0, clean].float()).all()
    assert torch.isnan(h[0, 4].float()).any() and not torch.isfinite(h[0, 3].float()).all()
    z = torch.zeros(1, 2, 64, device='cuda', dtype=torch.bfloat16)
    _, f = ops.gate_residual_norm_(z, torch.zeros_like(z), want_factor=True)
    assert f.item() == 1.


@gpu
def test_graphs_replayed_side_by_side_keep_their_factors():
    """Two graphs captured on one stream and replayed on two: each has its own scratch for the factor."""
    from thunderworld_b200 import ops
    made = []
    for i in range(2):
        v = inputs(1, 2000, 2048, 20 + i)
        v['y'] *= 1 + 3 * i
        x = v['x'].clone()
        want_h, want_f = ops.gate_residual_norm_(x.clone(), v['y'], v['gate'], want_factor=True)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.copy_(v['x'])
            h, f = ops.gate_residual_norm_(x, v['y'], v['gate'], want_factor=True)
        made.append((graph, h, f, want_h, want_f, torch.cuda.Stream(), v, x))
    torch.cuda.synchronize()
    for _ in range(30):
        for graph, *_, stream, v, x in made:
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for _, h, f, want_h, want_f, *_ in made:
            assert torch.equal(h, want_h) and torch.equal(f, want_f)


@gpu
def test_gpu_refusals():
    from thunderworld_b200 import ops
    v = inputs(2, 4, 256, 1)
    call = ops.gate_residual_norm_
    with pytest.raises(ValueError, match='equal shapes'):
        call(v['x'], v['y'][:, :2].contiguous(), v['gate'])
    with pytest.raises(ValueError, match='share memory'):
        call(v['x'], v['x'], v['gate'])
    with pytest.raises(ValueError, match='batch'):
        call(v['x'], v['y'], v['gate'][:, :128].contiguous())
    with pytest.raises(ValueError, match='batch'):
        call(v['x'], v['y'], v['gate'], shift=v['shift'][:1].contiguous(), scale=v['scale'][:1].contiguous())
    with pytest.raises(ValueError, match='together'):
        call(v['x'], v['y'], v['gate'], shift=v['shift'])
    with pytest.raises(ValueError, match='hidden'):
        call(v['x'], v['y'], v['gate'], weight=v['weight'][:128].contiguous())
    with pytest.raises(ValueError, match='empty'):
        call(v['x'][:, :0].contiguous(), v['y'][:, :0].contiguous())
    with pytest.raises(ValueError, match='contiguous CUDA BF16'):
        call(v['x'].float(), v['y'])
    with pytest.raises(ValueError, match='contiguous CUDA BF16'):
        call(v['x'][..., ::2], v['y'][..., ::2])
    with pytest.raises(RuntimeError, match='inference'):
        call(v['x'], v['y'].clone().requires_grad_())
    with pytest.raises(RuntimeError, match='shape'):
        call(v['x'][..., :4].contiguous(), v['y'][..., :4].contiguous())
    with pytest.raises(RuntimeError, match='maximum'):
        big = torch.zeros(1, 1, 16392, device='cuda', dtype=torch.bfloat16)
        call(big, big.clone())


def test_refusals_without_a_gpu():
    import ctypes
    from thunderworld_b200 import _lib, ops
    x = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match='CUDA'):
        ops.gate_residual_norm_(x, x.clone())
    lib = _lib.load()
    ok = ctypes.c_void_p(256)
    assert lib.tw_gate_residual_norm(None, ok, None, None, 0, 1., None, None, None, ok, None, None, 1, 64, 1, 0., None) == 1
    assert lib.tw_gate_residual_norm(ok, ok, None, ok, 0, 1., None, None, None, ok, None, None, 1, 64, 1, 0., None) == 1
    assert lib.tw_gate_residual_norm(ok, ok, None, None, 0, 1., None, ok, None, ok, None, None, 1, 64, 1, 0., None) == 1
    assert lib.tw_gate_residual_norm(ok, ok, None, None, 0, 1., None, None, None, ok, ok, None, 1, 64, 1, 0., None) == 1
    assert lib.tw_gate_residual_norm(ok, ok, None, None, 0, 1., None, None, None, ok, None, None, 1, 63, 1, 0., None) == 2
    assert lib.tw_gate_residual_norm(ok, ok, None, None, 0, 1., None, None, None, ok, None, None, 1, 16392, 1, 0., None) == 9
    assert lib.tw_gate_residual_norm(ok, ctypes.c_void_p(260), None, None, 0, 1., None, None, None, ok, None, None, 1, 64, 1, 0., None) == 3
