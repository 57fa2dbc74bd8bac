"""Attention of one token over a paged cache (`ops.paged_attention`) against its formula in 64 bits.

Tolerances. A score is a 32-bit sum of exact products, added by dim / 16 instructions: off by at most A = (dim / 16 + 4) 2^-22 times
the sum of the products' sizes, scale included; its multiplication by scale log2(e) adds 2^-22 of its size, which the test counts
into A. A probability is then off by a relative 2 A + 2^-21 (exponential: 2^-22), its rounding adds 2^-17 (two bf16 values) or, with
E4M3 pages, 2^-12 of itself or 2^-25 of the largest (f16); sums of n tokens in 32 bits add (n / 16 + 16) 2^-22. Numerator and
denominator together: twice that, of the sum of |p v|. The result is rounded once to bf16, half a step, 2^-8."""
import pytest
import torch

gpu = pytest.mark.gpu


def make(lens, hk, dim, page, fp8, seed, width=None, sequences=None, poison=True, strided=False):
    """A cache with the given lengths: pages in random order; NaN wherever nothing may be read."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pages, s = sum(need) + 3, sequences or len(lens)
    order = torch.randperm(pages, generator=g).tolist()
    width = width or max(1, max(need))
    table = torch.full((s, width), -1, dtype=torch.int32)
    pool = torch.randn(2, pages, hk, page, dim, generator=g)
    pool = (pool * 16).to(torch.float8_e4m3fn) if fp8 else pool.bfloat16()
    bits, nan = (pool.view(torch.uint8), 0x7f) if fp8 else (pool, float('nan'))
    live = torch.zeros(pages, page, dtype=torch.bool)
    for i, n in enumerate(lens):
        for j in range(need[i]):
            table[i, j] = order.pop()
            live[table[i, j], :n - j * page] = True
    if poison:
        bits.transpose(2, 3)[:, ~live] = nan
    kp, vp = pool[0].cuda(), pool[1].cuda()
    if strided:                                         # keys and values of a page side by side
        both = torch.stack([pool[0].view(torch.uint8) if fp8 else pool[0], pool[1].view(torch.uint8) if fp8 else pool[1]], 1).cuda()
        both = both.view(torch.float8_e4m3fn) if fp8 else both
        kp, vp = both[:, 0], both[:, 1]
    lengths = torch.zeros(s, dtype=torch.int32)
    lengths[:len(lens)] = torch.tensor(lens, dtype=torch.int32)
    scales = [(torch.rand(hk, generator=g) + .5).cuda() / 16 for _ in range(2)] if fp8 else [None, None]
    return kp, vp, table.cuda(), lengths.cuda(), scales


def check(out, lse, q, kp, vp, table, lengths, slots, scale, scales, hk, page, fp8, lens):
    batch, hq, dim = q.shape
    u8 = lambda p, at: (p.view(torch.uint8) if fp8 else p)[at].view(p.dtype).double()  # noqa: E731
    for b in range(batch):
        s = b if slots is None else int(slots[b])
        n = lens[s]
        if n == 0:
            assert not out[b].any() and (lse[b] == -float('inf')).all()
            continue
        at = table[s, :-(-n // page)].long()
        k, v = (u8(p, at).permute(1, 0, 2, 3).reshape(hk, -1, dim)[:, :n] for p in (kp, vp))
        if fp8:
            k, v = k * scales[0].double()[:, None, None], v * scales[1].double()[:, None, None]
        qq = q[b].double().view(hk, hq // hk, dim)
        score = scale * qq @ k.transpose(1, 2)
        size = abs(scale) * qq.abs() @ k.abs().transpose(1, 2)
        a = ((dim / 16 + 4) * 2. ** -22 * size + 2. ** -22 * score.abs()).amax(-1)
        want_lse = torch.logsumexp(score, -1)
        p = torch.exp(score - want_lse[..., None])
        want = p @ v
        e = 2 * (2 * a + 2. ** -21 + (2. ** -12 if fp8 else 2. ** -17) + (n / 16 + 16) * 2. ** -22)
        bound = 2. ** -8 * want.abs() + e[..., None] * (p @ v.abs()) + (2. ** -24 * p.amax(-1)[..., None] * v.abs().sum(1)[:, None] if fp8 else 0)
        off = (out[b].view(hk, -1, dim).double() - want).abs()
        assert (off <= bound).all(), (b, float((off - bound).max()))
        off = (lse[b].view(hk, -1).double() - want_lse).abs()
        assert (off <= 2 * a + 2. ** -20 + (n / 16 + 16) * 2. ** -22 + 2. ** -21 * want_lse.abs()).all(), (b, float(off.max()))


def run(lens, hq, hk, dim, page, fp8, seed=0, scale=None, **kw):
    from thunderworld_b200 import ops
    kp, vp, table, lengths, scales = make(lens, hk, dim, page, fp8, seed, **kw)
    q = torch.randn(len(lens), hq, dim, generator=torch.Generator().manual_seed(seed + 1)).bfloat16().cuda()
    out, lse = ops.paged_attention(q, kp, vp, table, lengths, scale=scale, k_scale=scales[0], v_scale=scales[1], return_lse=True)
    torch.cuda.synchronize()
    check(out, lse, q, kp, vp, table, lengths, None, dim ** -.5 if scale is None else scale, scales, hk, page, fp8, lens)
    assert ops.device_status() == 0
    return q, kp, vp, table, lengths, scales, out, lse


LENS = [[1], [16], [17, 0, 1], [63, 64, 65, 0, 128], [3840], [5, 1000, 0, 0, 77, 2049, 1, 64], [300] * 40, [0, 0], [8191, 1, 4096]]


@gpu
@pytest.mark.parametrize('lens', LENS, ids=lambda v: f'{len(v)}x{max(v)}')
@pytest.mark.parametrize('hq,hk,dim,page', [(8, 8, 128, 64), (32, 8, 128, 16), (12, 4, 64, 32), (16, 1, 64, 128), (6, 2, 128, 8)])
@pytest.mark.parametrize('fp8', [False, True])
def test_formula(lens, hq, hk, dim, page, fp8):
    run(lens, hq, hk, dim, page, fp8, seed=len(lens))


@gpu
@pytest.mark.parametrize('hq,hk', [(17, 1), (40, 2), (64, 1), (16, 16), (96, 32)])
@pytest.mark.parametrize('page', [1, 2, 4])
def test_groups_wider_than_a_tile_and_tiny_pages(hq, hk, page):
    run([130, 1, 0, 67], hq, hk, 64, page, True, seed=hq)
    run([130, 1, 0, 67], hq, hk, 128, page, False, seed=hq)


@gpu
@pytest.mark.parametrize('fp8', [False, True])
def test_many_sequences(fp8):
    g = torch.Generator().manual_seed(3)
    run([int(n) for n in torch.randint(0, 90, (700,), generator=g)], 4, 2, 64, 16, fp8, seed=9)


@gpu
@pytest.mark.parametrize('hq,hk,dim', [(16, 1, 128), (16, 1, 64), (8, 1, 128), (24, 2, 128), (4, 1, 128)])
@pytest.mark.parametrize('count', [2, 23, 37, 64, 101, 150])
def test_runs_that_begin_and_end_anywhere(hq, hk, dim, count):
    """Sequences of a few units, so that the CTAs' shares begin inside them, behind them and between two, and hold one, several or none."""
    lens = [int(n) for n in torch.randint(0, 400, (count,), generator=torch.Generator().manual_seed(count))]
    run(lens, hq, hk, dim, 16, count % 2 == 1, seed=count)


@gpu
@pytest.mark.parametrize('fp8', [False, True])
def test_sharp_scores_and_scale(fp8):
    """Scores of hundreds, so that one token has all the weight, and a negative scale."""
    run([500, 33], 8, 2, 128, 16, fp8, seed=4, scale=3.)
    run([500, 33], 8, 2, 64, 16, fp8, seed=5, scale=-.7)


@gpu
@pytest.mark.parametrize('fp8', [False, True])
def test_slots_strides_wide_table_and_out(fp8):
    from thunderworld_b200 import ops
    lens = [40, 700, 0, 129]
    kp, vp, table, lengths, scales = make(lens, 4, 128, 16, fp8, 6, width=60, sequences=9, strided=True)
    wide = torch.full((9, 100), 123456789, dtype=torch.int32, device='cuda')
    wide[:, :60] = table
    g = torch.Generator().manual_seed(7)
    heads = torch.randn(6, 3, 8, 128, generator=g).bfloat16().cuda()
    q = heads[:, 1]                                                      # strided rows, as sliced from a QKV projection
    slots = torch.tensor([3, 1, 1, 2, 0, 8], dtype=torch.int32, device='cuda')
    out = torch.full((6, 8, 128), 5., device='cuda', dtype=torch.bfloat16)
    got, lse = ops.paged_attention(q, kp, vp, wide[:, :60], lengths, slots=slots, k_scale=scales[0], v_scale=scales[1], return_lse=True, out=out)
    assert got is out
    check(out, lse, q, kp, vp, table, lengths, slots, 128 ** -.5, scales, 4, 16, fp8, lens + [0] * 5)
    turned = torch.randn(8, 6, 128, generator=g).bfloat16().cuda().transpose(0, 1)
    a = ops.paged_attention(turned, kp, vp, table, lengths, slots=slots, k_scale=scales[0], v_scale=scales[1])
    assert torch.equal(a, ops.paged_attention(turned.contiguous(), kp, vp, table, lengths, slots=slots, k_scale=scales[0], v_scale=scales[1]))


@gpu
def test_entries_that_lead_outside_are_left_out_and_reported():
    from thunderworld_b200 import ops
    lens = [100, 70, 64]
    kp, vp, table, lengths, scales = make(lens, 2, 64, 16, False, 1)
    q = torch.randn(4, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    clean = ops.paged_attention(q[:3], kp, vp, table, lengths)
    assert ops.device_status() == 0
    bad = table.clone()
    bad[0, 1], bad[1, 0] = 10 ** 6, -5
    slots = torch.tensor([0, 1, 2, 77], dtype=torch.int32, device='cuda')
    out, lse = ops.paged_attention(q, kp, vp, bad, lengths, slots=slots, return_lse=True)
    assert ops.device_status() == 11
    ops.reset_device_status()
    assert torch.equal(out[2], clean[2]) and not out[3].any() and (lse[3] == -float('inf')).all()
    for b, gone in ((0, range(16, 32)), (1, range(16))):                 # the other tokens' attention
        at = table[b, :-(-lens[b] // 16)].long()
        keep = [t for t in range(lens[b]) if t not in gone]
        k, v = (p[at].double().permute(1, 0, 2, 3).reshape(2, -1, 64)[:, keep] for p in (kp, vp))
        w = torch.softmax(q[b].double().view(2, 2, 64) @ k.transpose(1, 2) / 8, -1)
        assert (out[b].view(2, 2, 64).double() - w @ v).abs().max() < 2 ** -6
    over = lengths.clone()
    over[2], over[1] = 10 ** 6, -3                                       # longer than the table, negative
    out = ops.paged_attention(q[:3], kp, vp, table, over)
    assert ops.device_status() == 11 and not out[1].any()
    ops.reset_device_status()
    assert ops.device_status() == 0


@gpu
def test_tiny_pages_with_a_bad_entry():
    from thunderworld_b200 import ops
    kp, vp, table, lengths, _ = make([40], 1, 64, 4, False, 1)
    q = torch.randn(1, 2, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    at = table[0].long()
    bad = table.clone()
    bad[0, 3] = 999
    out = ops.paged_attention(q, kp, vp, bad, lengths)
    assert ops.device_status() == 11
    ops.reset_device_status()
    keep = [t for t in range(40) if t // 4 != 3]
    k, v = (p[at].double().permute(1, 0, 2, 3).reshape(1, -1, 64)[:, keep] for p in (kp, vp))
    assert (out.double() - torch.softmax(q.double() @ k.transpose(1, 2) / 8, -1) @ v).abs().max() < 2 ** -6


@gpu
def test_infinities_and_nan_in_live_places_stay_in_their_heads():
    from thunderworld_b200 import ops
    kp, vp, table, lengths, _ = make([50, 50], 2, 64, 16, False, 1)
    q = torch.randn(2, 4, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    clean = ops.paged_attention(q, kp, vp, table, lengths)
    vp[table[0, 1].long(), 0, 3, 5] = float('nan')
    vp[table[1, 0].long(), 1, 2, 7] = float('inf')
    out = ops.paged_attention(q, kp, vp, table, lengths)
    assert torch.isnan(out[0, :2, 5]).all() and not torch.isfinite(out[1, 2:, 7]).any()
    out[0, :2, 5], out[1, 2:, 7] = clean[0, :2, 5], clean[1, 2:, 7]
    assert torch.equal(out, clean)
    kp[table[0, 0].long(), 0, 0] = float('-inf')                          # scores of -inf, inf or nan by sign: as the formula, head by head
    k = kp[table[0].long()].double().permute(1, 0, 2, 3).reshape(2, -1, 64)[:, :50]
    want = torch.softmax(q[0].double().view(2, 2, 64) @ k.transpose(1, 2) / 8, -1)
    got = ops.paged_attention(q, kp, vp, table, lengths)
    assert torch.equal(torch.isnan(got[0, :2]).any(-1), torch.isnan(want[0]).any(-1))
    assert torch.equal(got[1, :2], out[1, :2])


@gpu
def test_streams_graphs_and_lengths_that_grow():
    """Two calls at once do not meet; a captured call reads the lengths and table of the replay."""
    from thunderworld_b200 import ops
    kp, vp, table, lengths, _ = make([2000, 31, 700], 4, 128, 16, False, 1, poison=False)
    q = torch.randn(3, 16, 128, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    want = [ops.paged_attention(q * i, kp, vp, table, lengths) for i in (1, 2)]
    qs = [q, q * 2]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(30):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, ops.paged_attention(qs[i], kp, vp, table, lengths)))
    torch.cuda.synchronize()
    assert all(torch.equal(y, want[i]) for i, y in got)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y = ops.paged_attention(q, kp, vp, table, lengths)
    for grown in ([2000, 31, 700], [1, 0, 64], [1999, 17, 33]):
        lengths.copy_(torch.tensor(grown, dtype=torch.int32))
        graph.replay()
        assert torch.equal(y, ops.paged_attention(q, kp, vp, table, lengths))


@gpu
def test_pool_past_32_bits():
    """A pool of more than 2^32 elements: pages at its end are read where they lie."""
    from thunderworld_b200 import ops
    pages, hk, page, dim = 70000, 8, 64, 128                              # 4.6e9 elements, 9.2 GB each half
    kp = torch.zeros((pages, hk, page, dim), device='cuda', dtype=torch.bfloat16)
    vp = torch.zeros_like(kp)
    at = torch.tensor([69999, 3, 33000, 65537], device='cuda')
    g = torch.Generator().manual_seed(1)
    small = torch.randn(2, 4, hk, page, dim, generator=g).bfloat16().cuda()
    kp[at], vp[at] = small[0], small[1]
    q = torch.randn(1, 16, dim, generator=g).bfloat16().cuda()
    lengths = torch.tensor([230], dtype=torch.int32, device='cuda')
    out = ops.paged_attention(q, kp, vp, at.int()[None], lengths)
    want = ops.paged_attention(q, small[0].contiguous(), small[1].contiguous(), torch.arange(4, device='cuda', dtype=torch.int32)[None], lengths)
    assert torch.equal(out, want) and out.any()


def _case(device):
    z = lambda *s, dtype=torch.int32: torch.zeros(s, dtype=dtype, device=device)  # noqa: E731
    return dict(q=z(2, 4, 64, dtype=torch.bfloat16), k_pages=z(3, 2, 16, 64, dtype=torch.bfloat16), v_pages=z(3, 2, 16, 64, dtype=torch.bfloat16),
                table=z(2, 5), lengths=z(2))


@gpu
def test_refusals():
    from thunderworld_b200 import ops
    ok = _case('cuda')
    ops.paged_attention(**ok)
    f8 = ok['k_pages'].to(torch.float8_e4m3fn)
    i32 = lambda *s: torch.zeros(s, dtype=torch.int32, device='cuda')  # noqa: E731
    for bad, match in ((dict(q=ok['q'].float()), 'BF16'), (dict(q=ok['q'][0]), 'BF16'), (dict(q=ok['q'][..., :32]), 'q must'), (dict(q=ok['q'][:, :3]), 'whole number'),
                       (dict(q=ok['q'][:0]), 'nonempty'), (dict(k_pages=ok['k_pages'][0]), 'alike'), (dict(k_pages=ok['k_pages'].half(), v_pages=ok['v_pages'].half()), 'bfloat16 or'),
                       (dict(k_pages=f8), 'bfloat16 or'), (dict(k_pages=ok['k_pages'][..., :32], v_pages=ok['v_pages'][..., :32]), '64 or 128'),
                       (dict(k_pages=ok['k_pages'][:, :, :12], v_pages=ok['v_pages'][:, :, :12]), 'power of two'),
                       (dict(k_pages=ok['k_pages'][:, :, ::2], v_pages=ok['v_pages'][:, :, ::2]), 'behind the other'),
                       (dict(table=i32(2, 5).long()), 'table'), (dict(table=i32(5)), 'table'), (dict(table=i32(5, 2).t()), 'table'), (dict(table=i32(2, 0)), 'table'),
                       (dict(lengths=i32(3)), 'lengths'), (dict(lengths=i32(2).long()), 'lengths'), (dict(lengths=i32(2).cpu()), 'lengths'),
                       (dict(slots=i32(3)), 'slots'), (dict(slots=i32(2).long()), 'slots'), (dict(table=i32(1, 5), lengths=i32(1)), 'slots'),
                       (dict(k_scale=torch.ones(2, device='cuda')), 'float8'), (dict(k_pages=f8, v_pages=f8, k_scale=torch.ones(3, device='cuda')), 'k_scale'),
                       (dict(k_pages=f8, v_pages=f8, v_scale=torch.ones(2)), 'v_scale'), (dict(out=torch.zeros(2, 4, 64, device='cuda')), 'out must'),
                       (dict(out=ok['q']), 'share memory')):
        with pytest.raises(ValueError, match=match):
            ops.paged_attention(**(ok | bad))
    with pytest.raises(RuntimeError, match='inference'):
        ops.paged_attention(**(ok | dict(q=ok['q'].clone().requires_grad_())))


def test_refusals_without_a_gpu():
    import ctypes
    from thunderworld_b200 import _lib, ops
    with pytest.raises(ValueError, match='CUDA'):
        ops.paged_attention(**_case('cpu'))
    lib = _lib.load()
    assert lib.tw_paged_attention(None, None) == 1 and lib.tw_paged_attention(ctypes.byref(_lib.PagedAttentionArgs()), None) == 1
    ok = dict(q=256, k_pages=256, v_pages=256, table=256, lengths=256, out=256, workspace=256, q_stride_batch=512, q_stride_head=128, k_stride_page=4096,
              k_stride_head=2048, v_stride_page=4096, v_stride_head=2048, table_stride=4, scale=1., batch=1, sequences=1, hq=4, hk=2, dim=128, page=16,
              pages=8, max_pages=4)
    for bad, status in ((dict(batch=0), 1), (dict(hq=3), 1), (dict(pages=0), 1), (dict(max_pages=0), 1), (dict(workspace=None), 1), (dict(dim=96), 2),
                        (dict(page=24), 2), (dict(max_pages=1 << 27), 9), (dict(k_pages=264), 3), (dict(v_stride_head=2044), 3), (dict(q=258), 3),
                        (dict(q_stride_head=127), 3), (dict(workspace=264), 3)):
        assert lib.tw_paged_attention(ctypes.byref(_lib.PagedAttentionArgs(**(ok | bad))), None) == status, bad
    size = lib.tw_paged_attention_workspace
    assert size(0, 4, 2, 128, 64) == 0 and size(1, 3, 2, 128, 64) == 0 and size(1, 4, 2, 128, 0) > 0
    assert size(4, 8, 2, 128, 10 ** 6) <= 148 * 3 * (2 * 4 * 130 * 4 + 16)


@gpu
@pytest.mark.parametrize('fp8', [False, True])
@pytest.mark.parametrize('hq,hk', [(4, 1), (16, 1), (6, 3)])
def test_spans_of_empty_sequences(hq, hk, fp8):
    """Between two sequences with tokens lie up to 200 without: a warp's cursor passes them and goes on in the right one."""
    g = torch.Generator().manual_seed(hq)
    lens = []
    for span in (0, 200, 1, 33, 0, 128, 64, 7, 199, 3):
        lens += [0] * span + [int(torch.randint(1, 500, (1,), generator=g))]
    run(lens + [0] * 90, hq, hk, 64, 16, fp8, seed=hk)
    run(lens + [0] * 90, hq, hk, 128, 4, fp8, seed=hk + 1)
