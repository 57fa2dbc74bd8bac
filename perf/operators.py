"""Cases of the token-at-a-time operators: matrix-vector products over packed NVFP4 weights, attention of one new
token over a paged key-value cache, the cache's page operations, and the gated residual fused with the norms around it.

`run` computes a case with elementary torch operations (own = False) or through the framework's entry points
(own = True). Sizes are those of the DiT configurations (hidden 2048 / 4096 / 6144, FFN 8192 / 16384 / 24576, 32 or 48
heads of 128 channels, 3840 tokens) and their odd neighbours."""
import math
import random
import torch

own = False
E2M1 = (0., .5, 1., 1.5, 2., 3., 4., 6., -0., -.5, -1., -1.5, -2., -3., -4., -6.)


# ---- cases -----------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one token through a 2048-wide output projection: a latency case
        dict(name='matvec 1x2048x2048', op='matvec', rows=1, n=2048, k=2048, tiles=0., prescale=False, bias=False),
        # one token through the QKV projection of the 4096-wide block
        dict(name='matvec 1x12288x4096', op='matvec', rows=1, n=12288, k=4096, tiles=0., prescale=True, bias=False),
        # a small batch of tokens through its FFN-up projection, with a bias
        dict(name='matvec 8x16384x4096', op='matvec', rows=8, n=16384, k=4096, tiles=0., prescale=True, bias=True),
        # an odd batch through the FFN-down projection of the 6144-wide block, a quarter of the residual tiles repaired
        dict(name='matvec 5x6144x24576 repaired', op='matvec', rows=5, n=6144, k=24576, tiles=.25, prescale=False, bias=False),
        # one sequence as long as the step's token count
        dict(name='attend 1x3840', op='attend', batch=1, hq=32, hk=8, dim=128, page=64, longest=3840, spread=0, fp8=False),
        # sequences of every length, one of them empty, on small pages
        dict(name='attend 24 ragged', op='attend', batch=24, hq=32, hk=8, dim=128, page=16, longest=8192, spread=5, fp8=False),
        # a long-context batch on an 8-bit cache
        dict(name='attend 48 long 8-bit', op='attend', batch=48, hq=32, hk=4, dim=128, page=64, longest=16384, spread=9, fp8=True),
        # a decode step's new keys and values of 64 sequences
        dict(name='append 64', op='append', batch=64, each=1, hk=8, dim=128, page=16, pages=4096, longest=900, spread=3, fp8=False),
        # a beam step: 32 sequences are forked, the 32 parents released
        dict(name='fork and free 32', op='fork', batch=32, hk=8, dim=128, page=64, pages=3200, longest=6000, spread=4, fp8=False),
        # a pool of which random halves were released is moved together
        dict(name='compact 2048', op='compact', batch=48, hk=8, dim=128, page=64, pages=2048, longest=4000, spread=7, fp8=False),
        # one token per CFG branch, norms before and after the block
        dict(name='norm 2x1x4096', op='norm', batch=2, tokens=1, hidden=4096, post=True, modulate=False),
        # the denoise step's residual stream
        dict(name='norm 2x3840x4096', op='norm', batch=2, tokens=3840, hidden=4096, post=False, modulate=True),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(('matvec', 'matvec', 'attend', 'attend', 'append', 'fork', 'compact', 'norm', 'norm'))
    if op == 'matvec':
        # the whole range of widths; with repaired tiles both sides lie on the 128 lattice
        tiles = rng.choice((0., 0., .1, .25, .5))
        k = 32 * _log(rng, 8, 768) if not tiles else 128 * _log(rng, 2, 192)
        n = _log(rng, 100, 20000) if not tiles else 128 * _log(rng, 2, 128)
        n = max(1, min(n, 150000000 // k)) if not tiles else max(1, min(n // 128, 150000000 // k // 128)) * 128
        return dict(op=op, rows=_log(rng, 1, 32), n=n, k=k, tiles=tiles, prescale=rng.random() < .5, bias=rng.random() < .5)
    if op == 'attend':
        hk = rng.choice((1, 2, 4, 8, 32))
        dim, fp8 = rng.choice((64, 128, 128)), rng.random() < .4
        longest = _log(rng, 1, 16384)
        batch = max(1, min(_log(rng, 1, 96), 370000000 // (longest * hk * dim * 4)))
        return dict(op=op, batch=batch, hq=hk * rng.choice((1, 3, 4, 8) if hk < 32 else (1, 2)), hk=hk, dim=dim,
                    page=rng.choice((1, 8, 16, 32, 64, 128)), longest=longest, spread=rng.randrange(1 << 20), fp8=fp8)
    if op == 'norm':
        hidden = 8 * _log(rng, 16, 1536)
        batch = rng.choice((1, 2, 3))
        tokens = max(1, min(_log(rng, 1, 4000), 31000000 // (batch * hidden)))
        return dict(op=op, batch=batch, tokens=tokens, hidden=hidden, post=rng.random() < .5, modulate=rng.random() < .5)
    c = dict(op=op, batch=_log(rng, 2, 48), hk=rng.choice((1, 2, 8)), dim=rng.choice((64, 128)), page=rng.choice((8, 16, 64)),
             longest=_log(rng, 8, 3000), spread=rng.randrange(1 << 20), fp8=rng.random() < .4)
    if op == 'append':
        c['each'] = _log(rng, 1, 200)
    most = -(-(c['longest'] + c.get('each', 0)) // c['page'])
    c['pages'] = c['batch'] * (most + 2) + rng.randrange(50)
    return c


def _lengths(case):
    """Tokens of every sequence, a property of the case: from one to the longest, one of them empty in larger batches."""
    r = random.Random(case['spread'])
    if case['batch'] == 1:
        return [case['longest']]
    got = [1 + int((case['longest'] - 1) * r.random() ** 1.5) for _ in range(case['batch'])]
    got[-1] = case['longest']
    if case['batch'] > 3:
        got[1] = 0
    return got


def _pages(tokens, page):
    return -(-tokens // page)


def _moves(case):
    """Whether each sequence of a compaction case has been released before (alternating from a random start)."""
    r = random.Random(case['spread'] + 1)
    return [r.random() < .5 for _ in range(case['batch'])]


def work(case):
    op = case['op']
    if op == 'matvec':
        r, n, k = case['rows'], case['n'], case['k']
        tiles = round(case['tiles'] * (n // 128) * (k // 128)) if case['tiles'] else 0
        return dict(bytes=n * k * 9 // 16 + tiles * 128 * 72 + 2 * r * (n + k) + 4 * k * case['prescale'] + 2 * n * case['bias'],
                    flops=2 * r * (n * k + tiles * 128 * 128))
    elt = 1 if case.get('fp8') else 2
    if op == 'attend':
        total = sum(_lengths(case))
        return dict(bytes=2 * total * case['hk'] * case['dim'] * elt + 4 * case['batch'] * case['hq'] * (case['dim'] + 1),
                    flops=4 * total * case['hq'] * case['dim'])
    if op == 'norm':
        rows = case['batch'] * case['tokens']
        return dict(bytes=8 * rows * case['hidden'] + 2 * case['hidden'] * (1 + case['batch'] * (1 + 2 * case['modulate'])),
                    flops=12 * rows * case['hidden'])
    row, lens = 2 * case['hk'] * case['dim'] * elt, _lengths(case)
    if op == 'append':
        return dict(bytes=case['batch'] * case['each'] * case['hk'] * case['dim'] * 2 * (2 + elt) + 12 * case['batch'], flops=0)
    if op == 'fork':
        part = sum(n % case['page'] for n in lens)
        return dict(bytes=2 * row * part + 16 * sum(_pages(n, case['page']) for n in lens), flops=0)
    # the pages that lie behind the live count move, about half of the live ones
    live = sum(_pages(n, case['page']) for n, gone in zip(lens, _moves(case)) if not gone)
    away = live * max(0, case['pages'] - live) // case['pages']
    return dict(bytes=2 * row * case['page'] * away + 4 * case['pages'] + 8 * live + 8, flops=0)


# ---- inputs ----------------------------------------------------------------------------------------------------------
def _gen(seed):
    return torch.Generator(device='cuda').manual_seed(seed)


def _e2m1_weights(n, k, g):
    """Codes and scales with the distribution that packing a normal weight gives: the group maximum near code 6."""
    codes = torch.randint(0, 256, (n, k // 2), generator=g, device='cuda', dtype=torch.uint8)
    scales = (torch.rand((n, k // 16), generator=g, device='cuda') * 200 + 40).to(torch.float8_e4m3fn)
    return codes, scales


def _pool(case, g, scale):
    shape = (case['pages'], case['hk'], case['page'], case['dim'])
    pool = torch.empty(shape, device='cuda', dtype=torch.bfloat16).normal_(generator=g)
    return (pool * scale).to(torch.float8_e4m3fn) if case['fp8'] else pool


def _cache(case, g, lens, room, pages):
    """A paged cache in use: page numbers in random order, -1 behind each sequence, reference counts. Table, lengths and
    reference counts are parts of one buffer, so that a pass can put them back in one copy."""
    s, page = len(lens), case['page']
    width = max(1, _pages(max(max(lens), case['longest']) + room, page))
    order = torch.randperm(pages, generator=g, device='cuda', dtype=torch.int64).int()
    need = torch.tensor([_pages(n, page) for n in lens], device='cuda')
    start = need.cumsum(0) - need
    col = torch.arange(width, device='cuda')[None]
    used = col < need[:, None]
    table = torch.where(used, order[(start[:, None] + col).clamp(max=pages - 1)], -1)
    small = torch.cat([table.flatten(), torch.tensor(lens, device='cuda', dtype=torch.int32),
                       torch.zeros(pages, device='cuda', dtype=torch.int32)])
    parts = (small[:s * width].view(s, width), small[s * width:s * width + s], small[s * width + s:])
    parts[2][table[used].long()] = 1
    return small, parts


def prepare(case, seed):
    g, op = _gen(seed), case['op']
    s = dict(case)
    randn = lambda *shape: torch.empty(shape, device='cuda', dtype=torch.float32).normal_(generator=g)  # noqa: E731
    if op == 'matvec':
        n, k = case['n'], case['k']
        s['x'] = randn(case['rows'], k).bfloat16()
        s['codes'], s['scales'] = _e2m1_weights(n, k, g)
        s['factor'] = torch.full((), 2e-5, device='cuda') * (1 + torch.rand((), device='cuda', generator=g))
        s['d'] = torch.rand(k, device='cuda', generator=g) + .5 if case['prescale'] else None
        s['b'] = randn(n).bfloat16() if case['bias'] else None
        s['bank'] = None
        if case['tiles']:
            nb, kb = n // 128, k // 128
            picked = torch.randperm(nb * kb, generator=g, device='cuda')[:round(case['tiles'] * nb * kb)].sort().values
            count = torch.zeros(nb, device='cuda', dtype=torch.int32).index_add_(0, picked // kb, torch.ones_like(picked, dtype=torch.int32))
            off = torch.cat([torch.zeros(1, device='cuda', dtype=torch.int32), count.cumsum(0).int()])
            wr, wrs = _e2m1_weights(len(picked) * 128, 128, g)
            s['bank'] = dict(wr=wr.view(-1, 128, 64), wrs=(wrs.float() / 8).to(torch.float8_e4m3fn).view(-1, 128, 8),
                             wi=(picked % kb).int(), off=off)
        return s
    if op == 'norm':
        b, t, h = case['batch'], case['tokens'], case['hidden']
        s['x'], s['y'] = randn(b, t, h).bfloat16(), randn(b, t, h).bfloat16()
        s['gate'] = (randn(b, h) * .3).bfloat16()
        s['weight'] = (1 + .1 * randn(h)).bfloat16()
        s['post_weight'] = (1 + .1 * randn(h)).bfloat16() if case['post'] else None
        s['shift'], s['scale'] = ((randn(b, h) * .1).bfloat16(), (randn(b, h) * .1).bfloat16()) if case['modulate'] else (None, None)
        s['residual_scale'] = .75 if case['post'] else 1.
        return s
    lens = _lengths(case)
    if op == 'attend':
        s['pages'] = sum(_pages(n, case['page']) for n in lens) + 3
        s['kp'], s['vp'] = _pool(s, g, 16.), _pool(s, g, 16.)
        s['small'], (s['table'], s['lengths'], _) = _cache(case, g, lens, 0, s['pages'])
        s['q'] = (randn(case['batch'], case['hq'], case['dim']) * 2).bfloat16()
        s['ks'], s['vs'] = (((1 + torch.rand(case['hk'], device='cuda', generator=g)) / 24 for _ in range(2)) if case['fp8'] else (None, None))
        return s
    s['kp'], s['vp'] = _pool(case, g, 16.), _pool(case, g, 16.)
    s['ks'], s['vs'] = ((torch.full((case['hk'],), 1 / 16, device='cuda'),) * 2 if case['fp8'] else (None, None))
    b = case['batch']
    if op == 'append':
        # every sequence gets between 1 and `each` new tokens
        r = random.Random(case['spread'] + 2)
        counts = [r.randint(1, case['each']) for _ in range(b)]
        counts[0] = case['each']
        s['cu'] = torch.tensor([0] + counts, device='cuda').cumsum(0).int() if case['each'] > 1 else None
        rows = sum(counts) if case['each'] > 1 else b
        s['k'], s['v'] = randn(rows, case['hk'], case['dim']).bfloat16(), randn(rows, case['hk'], case['dim']).bfloat16()
        s['slots'] = torch.randperm(b, generator=g, device='cuda').int()
        s['small'], parts = _cache(case, g, lens, case['each'], case['pages'])
    elif op == 'fork':
        s['parents'] = torch.randperm(b, generator=g, device='cuda').int()
        s['children'] = (torch.randperm(b, generator=g, device='cuda') + b).int()
        s['small'], parts = _cache(case, g, lens + [0] * b, 0, case['pages'])
    else:
        keep = [0 if gone else n for n, gone in zip(lens, _moves(case))]
        s['small'], parts = _cache(case, g, keep, 0, case['pages'])
    s['table'], s['lengths'], s['refs'] = parts
    s['before'] = s['small'].clone()
    return s


# ---- one pass --------------------------------------------------------------------------------------------------------
def run(s):
    return {'matvec': _matvec, 'attend': _attend, 'append': _append, 'fork': _fork, 'compact': _compact, 'norm': _norm}[s['op']](s)


def _decoded(codes, scales):
    """E2M1 codes (low nibble first) times the scale of their group of 16, in 32 bits; exact."""
    lut = torch.tensor(E2M1, device=codes.device)
    pair = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    return lut[pair].unflatten(-1, (-1, 16)).mul_(scales.float()[..., None]).flatten(-2)


def _matvec(s):
    bank = s['bank'] or {}
    if own:
        from thunderworld_b200 import ops
        return ops.fp4_matvec(s['x'], s['codes'], s['scales'], s['factor'], prescale=s['d'], bias=s['b'], **bank)
    w = _decoded(s['codes'], s['scales'])
    if bank:
        nb, kb = s['n'] // 128, s['k'] // 128
        block = torch.searchsorted(bank['off'][1:].contiguous(), torch.arange(len(bank['wi']), device='cuda', dtype=torch.int32), right=True)
        w.view(nb, 128, kb, 128)[block, :, bank['wi'].long()] += _decoded(bank['wr'], bank['wrs'])
    x = s['x'].float() if s['d'] is None else (s['x'].float() * s['d']).bfloat16().float()
    y = (x @ w.T) * s['factor']
    return (y if s['b'] is None else y + s['b'].float()).bfloat16()


def _attend(s):
    if own:
        from thunderworld_b200 import ops
        return ops.paged_attention(s['q'], s['kp'], s['vp'], s['table'], s['lengths'], k_scale=s['ks'], v_scale=s['vs'], return_lse=True)
    b, hq, hk, dim = s['batch'], s['hq'], s['hk'], s['dim']
    at = s['table'].clamp(min=0).long()
    k = s['kp'].view(torch.uint8)[at].view(s['kp'].dtype).float().transpose(1, 2).flatten(2, 3)      # [b, hk, t, dim]
    v = s['vp'].view(torch.uint8)[at].view(s['vp'].dtype).float().transpose(1, 2).flatten(2, 3)
    if s['ks'] is not None:
        k, v = k * s['ks'][:, None, None], v * s['vs'][:, None, None]
    q = s['q'].float().view(b, hk, hq // hk, dim)
    live = (torch.arange(k.shape[2], device='cuda') < s['lengths'][:, None])[:, None, None]
    scores = torch.where(live, (q @ k.transpose(2, 3)) * dim ** -.5, -math.inf)
    top = scores.amax(-1, keepdim=True)
    top = torch.where(top == -math.inf, 0., top)
    p = torch.exp(scores - top)
    total = p.sum(-1, keepdim=True)
    out = (p @ torch.where(live.transpose(2, 3), v, 0.)) / torch.where(total == 0, 1., total)
    return out.view(b, hq, dim).bfloat16(), (top + total.log()).view(b, hq)


def _stored(x, s, which):
    """Rows as the pool holds them."""
    pool = s['kp']
    return x if s[which] is None else (x.float() / s[which][:, None]).clamp(-448, 448).to(pool.dtype)


def _bytes(pool):
    return pool.view(torch.uint8) if pool.dtype == torch.float8_e4m3fn else pool


def _held(pool):
    """An 8-bit pool as the values that it stands for."""
    return pool.bfloat16() if pool.dtype == torch.float8_e4m3fn else pool


def _state(s):
    return dict(table=s['table'], lengths=s['lengths'], refs=s['refs'], k=_held(s['kp']), v=_held(s['vp']))


def _free_pages(refs):
    """Page numbers, the unused ones first, each kind in ascending order."""
    return torch.argsort((refs != 0).int(), stable=True).int()


def _append(s):
    # the small tables are put back first, so that a pass always starts from the same state
    s['small'].copy_(s['before'])
    if own:
        from thunderworld_b200 import ops
        ops.cache_append_(s['k'], s['v'], s['kp'], s['vp'], s['table'], s['lengths'], s['refs'], slots=s['slots'], cu=s['cu'],
                          k_scale=s['ks'], v_scale=s['vs'])
        return _state(s)
    rows, page = s['k'].shape[0], s['page']
    r = torch.arange(rows, device='cuda', dtype=torch.int32)
    cu = s['cu'] if s['cu'] is not None else torch.arange(rows + 1, device='cuda', dtype=torch.int32)
    i = torch.searchsorted(cu[1:].contiguous(), r, right=True)
    slot = s['slots'].long()[i]
    pos = (s['lengths'][slot] + r - cu[i]).long()
    new = pos % page == 0
    fresh = _free_pages(s['refs'])[(new.cumsum(0) - 1).clamp(min=0)]
    s['table'][slot[new], pos[new] // page] = fresh[new]
    s['refs'][fresh[new].long()] = 1
    at = s['table'][slot, pos // page].long()
    _bytes(s['kp'])[at, :, pos % page] = _bytes(_stored(s['k'], s, 'ks'))
    _bytes(s['vp'])[at, :, pos % page] = _bytes(_stored(s['v'], s, 'vs'))
    s['lengths'][s['slots'].long()] += cu[1:] - cu[:-1]
    return _state(s)


def _fork(s):
    s['small'].copy_(s['before'])
    if own:
        from thunderworld_b200 import ops
        ops.cache_fork_(s['kp'], s['vp'], s['table'], s['lengths'], s['refs'], s['parents'], s['children'])
        ops.cache_free_(s['table'], s['lengths'], s['refs'], s['parents'], s['page'])
        return _state(s)
    page, old, new = s['page'], s['parents'].long(), s['children'].long()
    n = s['lengths'][old].long()
    part, last = n % page, (n // page).clamp(max=s['table'].shape[1] - 1)
    torn = part > 0
    fresh = _free_pages(s['refs'])[(torn.cumsum(0) - 1).clamp(min=0)]
    rows = s['table'][old]
    col = torch.arange(rows.shape[1], device='cuda')[None]
    source = rows.gather(1, last[:, None])[:, 0].long()[torn]
    s['refs'].index_add_(0, rows.clamp(min=0).flatten().long(), (col < (n // page)[:, None]).int().flatten())
    rows[torn, last[torn]] = fresh[torn]
    s['refs'][fresh[torn].long()] = 1
    s['table'][new] = rows
    s['lengths'][new] = n.int()
    keep = (torch.arange(page, device='cuda')[None] < part[torn][:, None])[:, None, :, None]
    for pool in (_bytes(s['kp']), _bytes(s['vp'])):
        pool[fresh[torn].long()] = torch.where(keep, pool[source], pool[fresh[torn].long()])
    # the parents' pages lose a reference each
    rows = s['table'][old]
    held = col < -(-n // page)[:, None]
    s['refs'].index_add_(0, rows.clamp(min=0).flatten().long(), -held.int().flatten())
    s['table'][old] = -1
    s['lengths'][old] = 0
    return _state(s)


def _compact(s):
    s['small'].copy_(s['before'])
    if own:
        from thunderworld_b200 import ops
        live = ops.cache_compact_(s['kp'], s['vp'], s['table'], s['lengths'], s['refs'])
        return dict(_state(s), live=live)
    used = s['refs'] > 0
    live = used.sum().int()
    number = torch.arange(len(used), device='cuda', dtype=torch.int32)
    source, target = (used & (number >= live)).nonzero()[:, 0], (~used & (number < live)).nonzero()[:, 0]
    number[source] = target.int()
    for pool in (_bytes(s['kp']), _bytes(s['vp'])):
        pool[target] = pool[source]
    s['table'].copy_(torch.where(s['table'] >= 0, number[s['table'].clamp(min=0).long()], -1))
    s['refs'][target] = s['refs'][source]
    s['refs'][source] = 0
    return dict(_state(s), live=live)


def _norm(s):
    if own:
        from thunderworld_b200 import ops
        h, factor = ops.gate_residual_norm_(s['x'], s['y'], s['gate'], post_weight=s['post_weight'], residual_scale=s['residual_scale'],
                                            weight=s['weight'], shift=s['shift'], scale=s['scale'], eps=1e-6, want_factor=True)
        return s['x'], h, factor
    z = s['y'].float()
    if s['post_weight'] is not None:
        z = z * torch.rsqrt(z.square().mean(-1, keepdim=True) + 1e-6) * s['post_weight'].float()
    s['x'].copy_(s['x'].float() * s['residual_scale'] + s['gate'].float()[:, None] * z)
    h = s['x'].float()
    h = h * torch.rsqrt(h.square().mean(-1, keepdim=True) + 1e-6) * s['weight'].float()
    if s['scale'] is not None:
        h = h * (1 + s['scale'].float()[:, None]) + s['shift'].float()[:, None]
    h = h.bfloat16()
    top = h.abs().amax().float()
    return s['x'], h, torch.where(top > 0, top / 2688, 1.)


# ---- the definitions in 64 bits --------------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    return {'matvec': _exact_matvec, 'attend': _exact_attend, 'norm': _exact_norm}.get(case['op'], _exact_cache)(s)


def _value(codes, scales):
    """E2M1: sign, two exponent bits, one mantissa bit; exponent 0 holds 0 and 1/2."""
    c = torch.stack((codes.bitwise_and(15), codes.bitwise_right_shift(4)), codes.dim()).reshape(*codes.shape[:-1], -1).int()
    e, m = (c >> 1) & 3, (c & 1).double()
    size = torch.where(e == 0, m / 2, (1 + m / 2) * torch.pow(2., (e - 1).double()))
    return torch.where(c >= 8, -size, size) * scales.double().repeat_interleave(16, -1)


def _exact_matvec(s):
    x = s['x'] if s['d'] is None else (s['x'].float() * s['d'][None]).to(torch.bfloat16)
    x, bank = x.double(), s['bank']
    got = []
    for n0 in range(0, s['n'], 1024):
        got.append(x @ _value(s['codes'][n0:n0 + 1024], s['scales'][n0:n0 + 1024]).T)
    y = torch.cat(got, 1)
    if bank:
        off = bank['off'].tolist()
        for b in range(len(off) - 1):
            if off[b + 1] > off[b]:
                w = _value(bank['wr'][off[b]:off[b + 1]], bank['wrs'][off[b]:off[b + 1]])             # [tiles, 128, 128]
                part = x.view(len(x), -1, 128)[:, bank['wi'][off[b]:off[b + 1]].long()]               # [rows, tiles, 128]
                y[:, b * 128:(b + 1) * 128] += torch.einsum('rtk,tnk->rn', part, w)
    y = y * s['factor'].double()
    return y if s['b'] is None else y + s['b'].double()


def _exact_attend(s):
    b, hq, hk, dim, page = s['batch'], s['hq'], s['hk'], s['dim'], s['page']
    out = torch.zeros((b, hq, dim), device='cuda', dtype=torch.float64)
    lse = torch.full((b, hq), -math.inf, device='cuda', dtype=torch.float64)
    for i, n in enumerate(_lengths(s)):
        if not n:
            continue
        at = s['table'][i, :_pages(n, page)].long()
        k = s['kp'].view(torch.uint8)[at].view(s['kp'].dtype).double().permute(1, 0, 2, 3).reshape(hk, -1, dim)[:, :n]
        v = s['vp'].view(torch.uint8)[at].view(s['vp'].dtype).double().permute(1, 0, 2, 3).reshape(hk, -1, dim)[:, :n]
        if s['ks'] is not None:
            k, v = k * s['ks'].double().view(hk, 1, 1), v * s['vs'].double().view(hk, 1, 1)
        score = torch.einsum('hgd,htd->hgt', s['q'][i].double().view(hk, hq // hk, dim), k) / math.sqrt(dim)
        log = torch.logsumexp(score, -1)
        out[i] = torch.einsum('hgt,htd->hgd', torch.exp(score - log[..., None]), v).reshape(hq, dim)
        lse[i] = log.reshape(hq)
    return out, lse


def _exact_norm(s):
    z = s['y'].double()
    if s['post_weight'] is not None:
        z = z / torch.sqrt((z * z).mean(-1, keepdim=True) + 1e-6) * s['post_weight'].double()
    x = s['residual_scale'] * s['x'].double() + s['gate'].double().unsqueeze(1) * z
    h = x.to(torch.bfloat16).double()                                                          # the stream is held in bf16
    h = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * s['weight'].double()
    if s['scale'] is not None:
        h = (1 + s['scale'].double().unsqueeze(1)) * h + s['shift'].double().unsqueeze(1)
    top = float(h.to(torch.bfloat16).abs().max())
    return x, h, torch.tensor(top / 2688 if top > 0 else 1., dtype=torch.float64)


def _exact_cache(s):
    """The rows that a sequence of host-side steps leaves in the pools; tables and counts are whole numbers, compared as they are."""
    table, lens, refs = s['table'].tolist(), s['lengths'].tolist(), s['refs'].tolist()
    page, op = s['page'], s['op']
    k, v = _held(s['kp']).double(), _held(s['vp']).double()
    free = (p for p in range(len(refs)) if refs[p] == 0)
    if op == 'append':
        cu = s['cu'].tolist() if s['cu'] is not None else range(len(lens) + 1)
        new = [r if t is None else (r.float() / t[:, None]).clamp(-448, 448).to(torch.float8_e4m3fn)
               for r, t in ((s['k'], s['ks']), (s['v'], s['vs']))]
        at = []
        for i, slot in enumerate(s['slots'].tolist()):
            for j in range(cu[i + 1] - cu[i]):
                t = lens[slot] + j
                if t % page == 0:
                    table[slot][t // page] = next(free)
                at.append((table[slot][t // page], t % page))
        at = torch.tensor(at, device='cuda')
        k[at[:, 0], :, at[:, 1]], v[at[:, 0], :, at[:, 1]] = new[0].double(), new[1].double()
    elif op == 'fork':
        for old in s['parents'].tolist():
            part = lens[old] % page
            if part:
                a, b = table[old][lens[old] // page], next(free)
                k[b, :, :part], v[b, :, :part] = k[a, :, :part], v[a, :, :part]
    else:
        live = sum(r > 0 for r in refs)
        away = [p for p in range(live, len(refs)) if refs[p] > 0]
        to = [p for p in range(live) if refs[p] == 0]
        if away:
            k[to], v[to] = k[away], v[away]
    return dict(table=None, lengths=None, refs=None, k=k, v=v, **(dict(live=None) if op == 'compact' else {}))
