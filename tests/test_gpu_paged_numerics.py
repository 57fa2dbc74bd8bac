"""Attention over a paged cache where probabilities are far apart and where values are infinite, against the formula in 64 bits.

Tolerances, as for the other tests of this operator: scores off by A (their 32-bit sums), a probability by a relative 2 A + 2^-20 more
for the exponential and its argument, and by its rounding: 2^-16 with bf16 pages (two bf16 values, the first truncated), with E4M3
pages 2^-12 of itself (f16) or 2^-25 of 2^-15 of the largest one of its warp, 2^-40; sums of n tokens (n / 16 + 16) 2^-22. The
result is rounded once, 2^-8."""
import math
import pytest
import torch

gpu = pytest.mark.gpu


def cache_of(k, v, page, seed):
    """Pools and table for k, v [sequences, hk, tokens, dim], pages in random order."""
    s, hk, n, dim = k.shape
    each = -(-n // page)
    order = torch.randperm(s * each, generator=torch.Generator().manual_seed(seed)).cuda()
    pools = []
    for x in (k, v):
        byte = x.view(torch.uint8) if x.dtype == torch.float8_e4m3fn else x
        pool = torch.zeros(s * each, hk, page, dim, device='cuda', dtype=byte.dtype)
        padded = torch.zeros(s, hk, each * page, dim, device='cuda', dtype=byte.dtype)
        padded[:, :, :n] = byte
        pool[order] = padded.view(s, hk, each, page, dim).transpose(1, 2).reshape(s * each, hk, page, dim)
        pools.append(pool.view(x.dtype))
    return pools[0], pools[1], order.view(s, each).int(), torch.full((s,), n, device='cuda', dtype=torch.int32)


def formula(q, k, v, scale):
    s, hq, dim = q.shape
    hk = k.shape[1]
    qq = q.double().view(s, hk, hq // hk, dim)
    score = scale * qq @ k.double().transpose(2, 3)
    size = scale * qq.abs() @ k.double().abs().transpose(2, 3)
    lse = torch.logsumexp(score, -1)
    p = torch.exp(score - lse[..., None])
    return p, score, size, lse


def check(out, lse, q, k, v, scale, fp8):
    s, hq, dim = q.shape
    p, score, size, want_lse = formula(q, k, v, scale)
    n = k.shape[2]
    want = p @ v.double()
    a = ((dim / 16 + 4) * 2. ** -22 * size + 2. ** -22 * score.abs()).amax(-1)
    e = 2 * (2 * a + 2. ** -20 + (2. ** -12 if fp8 else 2. ** -16) + (n / 16 + 16) * 2. ** -22)
    bound = 2. ** -8 * want.abs() + e[..., None] * (p @ v.double().abs())
    if fp8:
        bound = bound + 2. ** -39 * p.amax(-1)[..., None] * v.double().abs().sum(2)[:, :, None]
    off = (out.view(want.shape).double() - want).abs()
    assert (off <= bound).all(), float((off - bound).max())
    off = (lse.view(want_lse.shape).double() - want_lse).abs()
    assert (off <= 2 * a + 2. ** -20 + (n / 16 + 16) * 2. ** -22 + 2. ** -21 * want_lse.abs()).all(), float(off.max())


@gpu
@pytest.mark.parametrize('nats', [4, 12, 18, 24])
@pytest.mark.parametrize('hq,hk,dim', [(4, 2, 128), (4, 2, 64), (16, 1, 128), (32, 2, 64)])
@pytest.mark.parametrize('tokens', [2, 31, 200, 3000])
@pytest.mark.parametrize('fp8', [False, True])
def test_a_key_far_above_the_rest_whose_value_is_zero(nats, hq, hk, dim, tokens, fp8):
    """What an attention sink looks like: the result is that of the other tokens, e^-18 of the weight or less each."""
    from thunderworld_b200 import ops
    g = torch.Generator().manual_seed(nats * 1000 + tokens)
    q, scale = torch.ones(2, hq, dim), dim ** -.5
    k = torch.randint(-1, 2, (2, hk, tokens, dim), generator=g).float() / 16
    k[:, :, 0] = 0
    k[:, :, 0, :16] = round(nats / scale) / 16             # score `nats` (16 equal channels), a multiple of 1/16
    if fp8:
        k = k.to(torch.float8_e4m3fn).float()              # rounded: what counts is that it is far above
    v = torch.randn(2, hk, tokens, dim, generator=g).to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
    v.view(torch.uint8)[:, :, 0] = 0
    q, k, v = q.bfloat16().cuda(), k.to(v.dtype).cuda(), v.cuda()
    kp, vp, table, lengths = cache_of(k, v, 16, 1)
    out, lse = ops.paged_attention(q, kp, vp, table, lengths, return_lse=True)
    assert out.any()
    check(out, lse, q, k, v, scale, fp8)


@gpu
@pytest.mark.parametrize('fp8', [False, True])
def test_many_tokens_far_below_one(fp8):
    """Weight that lies in a hundred thousand tokens, each 2^-25 of the one above them."""
    from thunderworld_b200 import ops
    dim, n = 64, 100000
    k = torch.zeros(1, 1, n, dim)
    k[0, 0, 777, 0] = 18.
    q = torch.zeros(1, 2, dim)
    q[..., 0] = 1.
    v = (torch.rand(1, 1, n, dim, generator=torch.Generator().manual_seed(1)) + 8).to(torch.float8_e4m3fn if fp8 else torch.bfloat16)
    v.view(torch.uint8)[0, 0, 777] = 0
    q, k, v = q.bfloat16().cuda(), k.to(v.dtype).cuda(), v.cuda()
    kp, vp, table, lengths = cache_of(k, v, 64, 2)
    out, lse = ops.paged_attention(q, kp, vp, table, lengths, scale=1., return_lse=True)
    check(out, lse, q, k, v, 1., fp8)


@gpu
@pytest.mark.parametrize('hq,hk,dim', [(4, 2, 128), (16, 1, 128), (8, 1, 64), (24, 1, 64)])
@pytest.mark.parametrize('tokens', [1, 16, 50, 2000])
def test_infinite_values(hq, hk, dim, tokens):
    """bf16 values of +inf, -inf and both in one channel: the formula's infinity or NaN, and every other channel as without them."""
    from thunderworld_b200 import ops
    g = torch.Generator().manual_seed(tokens)
    q = torch.randn(3, hq, dim, generator=g).bfloat16().cuda()
    k, v = torch.randn(2, 3, hk, tokens, dim, generator=g).bfloat16().cuda()
    at = [int(i) for i in torch.randint(0, tokens, (4,), generator=g)]
    clean = ops.paged_attention(q, *cache_of(k, v, 16, 3))
    v[0, 0, at[0], 5] = math.inf
    v[1, 0, at[1], 40] = -math.inf
    v[2, hk - 1, at[2], 9], v[2, hk - 1, (at[2] + 1) % tokens, 9] = math.inf, -math.inf
    out = ops.paged_attention(q, *cache_of(k, v, 16, 3))
    p, *_ = formula(q, k, v, dim ** -.5)
    want = (p[..., None] * v.double()[:, :, None]).sum(-2).view(3, hq, dim)
    odd = ~want.isfinite()
    assert odd.sum() == 3 * hq // hk and torch.equal(out[odd].double().nan_to_num(7., 8., 9.), want[odd].nan_to_num(7., 8., 9.))
    assert torch.equal(out[~odd], clean[~odd])
