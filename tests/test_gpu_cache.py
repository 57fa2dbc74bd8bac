"""Pages of a key-value cache (`ops.cache_*_`, `PagedCache`) against a host model of the same rules: tables, lengths and counts have to be
equal, rows too (bf16 as they are; E4M3 as torch rounds them). What no rule writes stays as it was, to the byte."""
import pytest
import torch

gpu = pytest.mark.gpu


class Model:
    """The rules, in Python lists; pools as CPU byte tensors [pages, hk, page, bytes of a row]."""

    def __init__(self, cache):
        self.page = cache.page_size
        self.table, self.lengths, self.refs = cache.table.tolist(), cache.lengths.tolist(), cache.refs.tolist()
        self.fp8 = cache.k_pages.dtype == torch.float8_e4m3fn
        self.scales = [None if s is None else s.cpu() for s in (cache.k_scale, cache.v_scale)]
        self.pools = [p.contiguous().view(torch.uint8).cpu().clone() for p in (cache.k_pages, cache.v_pages)]

    def take(self):
        p = self.refs.index(0)
        self.refs[p] = 1
        return p

    def append(self, k, v, slots, cu):
        for i, s in enumerate(slots):
            for r in range(cu[i], cu[i + 1]):
                pos = self.lengths[s]
                if pos % self.page == 0:
                    self.table[s][pos // self.page] = self.take()
                for pool, x, scale in zip(self.pools, (k, v), self.scales):
                    x = x[r].cpu()
                    if self.fp8:
                        x = x.float() if scale is None else x.float() / scale[:, None]
                        x = x.clamp(-448, 448).to(torch.float8_e4m3fn)
                    pool[self.table[s][pos // self.page], :, pos % self.page] = x.contiguous().view(torch.uint8)
                self.lengths[s] += 1

    def fork(self, parents, children):
        before = list(self.lengths)                        # the parents are what they were before the call
        for p, c in zip(parents, children):
            n = before[p]
            for j in range(n // self.page):
                self.table[c][j] = self.table[p][j]
                self.refs[self.table[p][j]] += 1
            if n % self.page:
                new, old = self.take(), self.table[p][n // self.page]
                self.table[c][n // self.page] = new
                for pool in self.pools:
                    pool[new, :, :n % self.page] = pool[old, :, :n % self.page]
            self.lengths[c] = n

    def free(self, slots):
        for s in slots:
            for j in range(-(-self.lengths[s] // self.page)):
                self.refs[self.table[s][j]] -= 1
                self.table[s][j] = -1
            self.lengths[s] = 0

    def compact(self):
        live = sum(r > 0 for r in self.refs)
        away, to = [p for p in range(live, len(self.refs)) if self.refs[p] > 0], [p for p in range(live) if self.refs[p] == 0]
        number = dict(zip(away, to))
        for a, b in number.items():
            for pool in self.pools:
                pool[b] = pool[a]
            self.refs[b], self.refs[a] = self.refs[a], 0
        self.table = [[number.get(p, p) for p in row] for row in self.table]
        return live

    def same(self, cache):
        assert cache.table.tolist() == self.table and cache.lengths.tolist() == self.lengths and cache.refs.tolist() == self.refs
        for pool, mine in zip((cache.k_pages, cache.v_pages), self.pools):
            assert torch.equal(pool.contiguous().view(torch.uint8).cpu(), mine)


def i32(values):
    return torch.tensor(values, dtype=torch.int32, device='cuda')


def make(pages, page, hk, dim, fp8, sequences=12, tokens=200, scaled=True):
    from thunderworld_b200 import PagedCache
    s = [torch.rand(hk, device='cuda') + .25 for _ in range(2)] if fp8 and scaled else [None, None]
    cache = PagedCache(pages, page, hk, dim, sequences=sequences, max_tokens=tokens, dtype=torch.float8_e4m3fn if fp8 else torch.bfloat16, k_scale=s[0], v_scale=s[1])
    for pool in (cache.k_pages, cache.v_pages):            # what is stale is not zero
        pool.view(torch.uint8).copy_(torch.randint(0, 127, pool.view(torch.uint8).shape, device='cuda', dtype=torch.uint8))
    return cache


@gpu
@pytest.mark.parametrize('page,hk,dim,fp8', [(1, 1, 64, False), (4, 3, 64, True), (16, 2, 128, False), (16, 8, 128, True), (64, 1, 64, False)])
def test_a_cache_in_use(page, hk, dim, fp8):
    """Appends of every kind, forks, frees and compactions in turn, compared after each."""
    from thunderworld_b200 import ops
    g = torch.Generator().manual_seed(page * 10 + dim)
    draw = lambda n: int(torch.randint(0, n, (1,), generator=g))  # noqa: E731
    cache = make(12 * 200 // page + 7, page, hk, dim, fp8)
    model = Model(cache)
    for step in range(60):
        what = draw(10)
        if what < 5:
            slots = torch.randperm(12, generator=g)[:1 + draw(12)].tolist()
            one = draw(2)
            counts = [1 if one else draw(min(40, 201 - model.lengths[s])) for s in slots]
            slots, counts = zip(*[(s, n) for s, n in zip(slots, counts) if model.lengths[s] + n <= 200] or [(0, 0)])
            one = one and sum(counts) == len(slots)
            cu = [0]
            for n in counts:
                cu.append(cu[-1] + n)
            k, v = (torch.randn(cu[-1] + (0 if one else draw(3)), hk, dim, generator=g).mul(3).bfloat16().cuda() for _ in range(2)) if one else [
                t[:cu[-1] + 2] for t in torch.randn(2, cu[-1] + 2, hk, dim, generator=g).mul(200).bfloat16().cuda()]
            cache.append(k, v, i32(slots), None if one else i32(cu))
            model.append(k, v, slots, cu)
        elif what < 7:
            empty = [s for s in range(12) if model.lengths[s] == 0]
            children = [empty[i] for i in torch.randperm(len(empty), generator=g)[:draw(4)].tolist()]
            parents = [draw(12) for _ in children]
            if sum(r == 0 for r in model.refs) >= len(children):
                cache.fork(i32(parents), i32(children))
                model.fork(parents, children)
        elif what < 9:
            slots = torch.randperm(12, generator=g)[:draw(5)].tolist()
            cache.free(i32(slots + slots[:1]))             # the first one twice
            model.free(slots)
        else:
            assert int(cache.compact()) == model.compact()
        model.same(cache)
    assert ops.device_status() == 0
    cache.check()
    cache.free(i32(list(range(12))))
    assert not cache.refs.any() and (cache.table == -1).all() and int(cache.compact()) == 0


@gpu
@pytest.mark.parametrize('fp8', [False, True])
def test_default_slots_and_strided_rows(fp8):
    cache = make(30, 4, 2, 64, fp8, sequences=5, tokens=20, scaled=False)
    model = Model(cache)
    qkv = torch.randn(5, 8, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    for _ in range(6):
        k, v = qkv[:, 4:6], qkv[:, 6:8]                    # rows as they lie in a QKV projection
        cache.append(k, v)
        model.append(k, v, range(5), range(6))
        model.same(cache)
    odd = torch.randn(3, 2, 65, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()[..., 1:]
    cache.append(odd, odd, cu=i32([0, 2, 3]))
    model.append(odd, odd, range(2), [0, 2, 3])
    model.same(cache)


@gpu
def test_rounding_to_e4m3():
    """Ties, subnormals, saturation, infinities and NaN as torch rounds them."""
    cache = make(4, 16, 1, 64, True, sequences=1, tokens=64, scaled=False)
    values = torch.tensor([0., -0., 2. ** -10, 1.5 * 2. ** -9, 2. ** -9, 17., 19., 449., 464., 465., 1e30, -1e30, float('inf'), -float('inf'), float('nan'), 447.] * 4)
    x = values.bfloat16().view(1, 1, 64).cuda()
    cache.append(x, x)
    at = int(cache.table[0, 0])
    want = torch.where(values.bfloat16().isnan(), values.bfloat16().float(), values.bfloat16().float().clamp(-448, 448)).to(torch.float8_e4m3fn)
    got = cache.k_pages[at, 0, 0].cpu()
    assert torch.equal(got.float().nan_to_num(12345.), want.float().nan_to_num(12345.))
    number = ~want.float().isnan()                         # a NaN has no sign
    assert torch.equal(torch.signbit(got.float())[number], torch.signbit(want.float())[number])


@gpu
@pytest.mark.parametrize('what', ['pool', 'table', 'slot', 'twice', 'negative', 'cu', 'length'])
def test_an_append_that_cannot_be_done_changes_nothing(what):
    from thunderworld_b200 import ops
    cache = make(9, 4, 1, 64, False, sequences=4, tokens=32)
    x = torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1]), i32([0, 6, 20]))       # 2 + 4 pages
    if what == 'length':
        cache.lengths[1] = -7
    model = Model(cache)
    slots, cu = dict(pool=([2, 3], [0, 8, 20]), table=([0, 1], [0, 1, 20]), slot=([2, 4], [0, 1, 2]), twice=([2, 2], [0, 1, 2]), negative=([2, -1], [0, 1, 2]),
                     cu=([2, 3], [0, 5, 21]), length=([1, 2], [0, 1, 2]))[what]
    cache.append(x, x, i32(slots), i32(cu))
    assert ops.device_status() == (12 if what in ('pool', 'table') else 11)
    with pytest.raises(RuntimeError, match='full' if what in ('pool', 'table') else 'outside'):
        cache.check()
    model.same(cache)
    ops.reset_device_status()
    cache.append(x[:2], x[:2], i32([2, 3]))                # and the cache goes on working
    model.append(x, x, [2, 3], [0, 1, 2])
    model.same(cache)
    cache.check()


@gpu
@pytest.mark.parametrize('what', ['pool', 'occupied', 'twice', 'slot', 'negative'])
def test_a_fork_that_cannot_be_done_changes_nothing(what):
    from thunderworld_b200 import ops
    cache = make(6, 4, 1, 64, False, sequences=6, tokens=32)
    x = torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1]), i32([0, 6, 16]))       # 2 + 3 pages, both torn: one is left
    model = Model(cache)
    parents, children = dict(pool=([0, 1], [2, 3]), occupied=([0], [1]), twice=([0, 5], [2, 2]), slot=([6], [2]), negative=([0], [-2]))[what]
    cache.fork(i32(parents), i32(children))
    assert ops.device_status() == (12 if what == 'pool' else 11)
    model.same(cache)
    ops.reset_device_status()
    cache.fork(i32([0, 5, 4]), i32([2, 4, 3]))             # one copy, and two of empty sequences
    model.fork([0], [2])
    model.same(cache)
    cache.check()


@gpu
def test_bad_frees_are_left_out():
    from thunderworld_b200 import ops
    cache = make(9, 4, 1, 64, False, sequences=4, tokens=32)
    x = torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1]), i32([0, 6, 20]))
    model = Model(cache)
    cache.free(i32([9, 0, -1]))
    assert ops.device_status() == 11
    ops.reset_device_status()
    model.free([0])
    model.same(cache)


@gpu
def test_large_tables():
    """More entries than the planning block has threads, and a pool that it scans in many passes."""
    cache = make(30000, 2, 1, 64, False, sequences=3000, tokens=64)
    model = Model(cache)
    g = torch.Generator().manual_seed(1)
    counts = torch.randint(0, 9, (3000,), generator=g).tolist()
    cu = [0]
    for n in counts:
        cu.append(cu[-1] + n)
    slots = torch.randperm(3000, generator=g).tolist()
    x = torch.randn(cu[-1], 1, 64, generator=g).bfloat16().cuda()
    # the same by prefix sums: the model's list search would take minutes
    cache.append(x, x, i32(slots), i32(cu))
    page = 0
    for i, s in enumerate(slots):
        need = -(-counts[i] // 2)
        model.table[s][:need] = range(page, page + need)
        page += need
        model.lengths[s] = counts[i]
    for p in range(page):
        model.refs[p] = 1
    assert cache.table.tolist() == model.table and cache.lengths.tolist() == model.lengths and cache.refs.tolist() == model.refs
    cache.free(i32(slots[::2]))
    live = int((cache.refs > 0).sum())
    before = {s: cache.k_pages[cache.table[s, :-(-n // 2)].long()].clone() for s, n in zip(slots[1:40:2], counts[1:40:2]) if n}
    assert int(cache.compact()) == live and (cache.refs[:live] == 1).all() and not cache.refs[live:].any()
    for s, rows in before.items():
        assert torch.equal(cache.k_pages[cache.table[s, :len(rows)].long()], rows)
    held = cache.table[cache.table >= 0].sort().values
    assert torch.equal(held, torch.arange(live, device='cuda', dtype=torch.int32))


@gpu
def test_pool_past_32_bits():
    """Pages that lie more than 2^32 elements into the pool are written, copied and moved."""
    from thunderworld_b200 import ops
    pages, hk, page, dim = 70000, 8, 64, 128
    kp, vp = (torch.zeros((pages, hk, page, dim), device='cuda', dtype=torch.bfloat16) for _ in range(2))
    refs = torch.ones(pages, device='cuda', dtype=torch.int32)
    refs[[5, 66000, 69000, 69999]] = 0
    table, lengths = torch.full((3, 4), -1, device='cuda', dtype=torch.int32), torch.zeros(3, device='cuda', dtype=torch.int32)
    x = torch.randn(100, hk, dim, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    ops.cache_append_(x, x, kp, vp, table, lengths, refs, slots=i32([1]), cu=i32([0, 100]))
    assert table[1].tolist() == [5, 66000, -1, -1]
    assert torch.equal(kp[66000, :, :36], x[64:].transpose(0, 1)) and torch.equal(vp[5], x[:64].transpose(0, 1))
    ops.cache_fork_(kp, vp, table, lengths, refs, i32([1]), i32([2]))
    assert table[2].tolist() == [5, 69000, -1, -1] and torch.equal(vp[69000, :, :36], x[64:].transpose(0, 1))
    refs[6:60000] = 0
    assert int(ops.cache_compact_(kp, vp, table, lengths, refs)) == int((refs > 0).sum()) < 60000
    a, b = table[1, 1].item(), table[2, 1].item()
    assert max(a, b) < 60000 and torch.equal(kp[a, :, :36], x[64:].transpose(0, 1)) and torch.equal(vp[b, :, :36], x[64:].transpose(0, 1))
    assert ops.device_status() == 0


@gpu
def test_a_captured_step_allocates():
    """Append and attend in a graph: every replay takes the pages that it needs."""
    cache, eager = make(64, 4, 2, 64, False, sequences=3, tokens=60), None
    eager = make(64, 4, 2, 64, False, sequences=3, tokens=60)
    x = torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    q = torch.randn(3, 8, 64, generator=torch.Generator().manual_seed(2)).bfloat16().cuda()
    slots = i32([2, 0, 1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.append(x, x, slots)
        out = cache.attend(q, slots)
    for step in range(30):
        x.copy_(torch.randn(3, 2, 64, generator=torch.Generator().manual_seed(step)).bfloat16())
        graph.replay()
        eager.append(x, x, slots)
        assert torch.equal(out, eager.attend(q, slots))
        assert torch.equal(cache.table, eager.table) and torch.equal(cache.lengths, eager.lengths) and torch.equal(cache.refs, eager.refs)


@gpu
def test_refusals():
    from thunderworld_b200 import PagedCache, ops
    c = make(6, 4, 2, 64, False)
    pools, tables = (c.k_pages, c.v_pages), (c.table, c.lengths, c.refs)
    x = torch.zeros(2, 2, 64, device='cuda', dtype=torch.bfloat16)
    s = i32([0, 1])
    for call, match in ((lambda: ops.cache_append_(x, x[:1], *pools, *tables, slots=s), 'alike'), (lambda: ops.cache_append_(x.float(), x, *pools, *tables), 'BF16'),
                        (lambda: ops.cache_append_(x[:, :1], x[:, :1], *pools, *tables), 'BF16'), (lambda: ops.cache_append_(x, x, *pools, *tables, slots=s[:1]), 'one row'),
                        (lambda: ops.cache_append_(x, x, *pools, *tables, slots=s, cu=s), 'one row'), (lambda: ops.cache_append_(x, x, *pools, *tables, slots=s.long()), 'slots'),
                        (lambda: ops.cache_append_(x.repeat(7, 1, 1), x.repeat(7, 1, 1), *pools, *tables), 'more entries'),
                        (lambda: ops.cache_append_(x, x, *pools, *tables, k_scale=torch.ones(2, device='cuda')), 'float8'),
                        (lambda: ops.cache_append_(x, x, *pools, c.table, c.lengths, c.refs[:3]), 'refs'), (lambda: ops.cache_append_(x, x, *pools, c.table.t(), c.lengths, c.refs), 'table'),
                        (lambda: ops.cache_append_(x, x, c.k_pages[:1].expand(6, 2, 4, 64), c.v_pages, *tables), 'expanded'),
                        (lambda: ops.cache_append_(x, x, *pools, c.table[:1].expand(12, -1), c.lengths, c.refs), 'overlap'),
                        (lambda: ops.cache_append_(c.k_pages[0, :, :2].transpose(0, 1), x, *pools, *tables), 'lie in the pages'),
                        (lambda: ops.cache_append_(x, c.k_pages[5, :, 2:].transpose(0, 1), *pools, *tables), 'lie in the pages'),
                        (lambda: ops.cache_append_(x, x, c.k_pages, c.k_pages, *tables), 'same memory'), (lambda: ops.cache_compact_(c.k_pages, c.k_pages, *tables), 'same memory'),
                        (lambda: ops.cache_fork_(*pools, *tables, s, s[:1]), 'one child'), (lambda: ops.cache_fork_(*pools, *tables, s.float(), s), 'parents'),
                        (lambda: ops.cache_free_(*tables, s.long(), 4), 'slots'), (lambda: ops.cache_free_(*tables, s, 3), 'power of two'),
                        (lambda: ops.cache_compact_(*pools, c.table, c.lengths[:3], c.refs), 'lengths'),
                        (lambda: PagedCache(4, 3, 1, sequences=1, max_tokens=8), 'power of two'), (lambda: PagedCache(4, 4, 1, 96, sequences=1, max_tokens=8), '64 or 128'),
                        (lambda: PagedCache(0, 4, 1, sequences=1, max_tokens=8), 'positive'), (lambda: PagedCache(4, 4, 1, sequences=1, max_tokens=8, dtype=torch.float16), 'bfloat16'),
                        (lambda: PagedCache(4, 4, 1, sequences=1, max_tokens=8, device='cpu'), 'CUDA')):
        with pytest.raises(ValueError, match=match):
            call()
    with pytest.raises(RuntimeError, match='inference'):
        ops.cache_append_(x.clone().requires_grad_(), x, *pools, *tables, slots=s)
    before = [t.clone() for t in tables]
    c.append(x[:0], x[:0], s[:0])                          # nothing to do is nothing done
    c.fork(s[:0], s[:0])
    c.free(s[:0])
    assert all(torch.equal(a, b) for a, b in zip(before, tables))


@gpu
def test_pools_of_one_buffer():
    """Keys and values as the halves of one tensor are two pools, not one."""
    from thunderworld_b200 import ops
    both = torch.zeros(6, 2, 2, 4, 64, device='cuda', dtype=torch.bfloat16)
    c = make(6, 4, 2, 64, False)
    k, v = torch.randn(2, 3, 2, 64, device='cuda').bfloat16()
    ops.cache_append_(k, v, both[:, 0], both[:, 1], c.table, c.lengths, c.refs, slots=i32([0]), cu=i32([0, 3]))
    page = int(c.table[0, 0])
    assert torch.equal(both[page, 0, :, :3], k.transpose(0, 1)) and torch.equal(both[page, 1, :, :3], v.transpose(0, 1))


@gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float8_e4m3fn])
def test_a_new_cache_takes_no_more_than_its_pages(dtype):
    from thunderworld_b200 import PagedCache
    c = PagedCache(4096, 64, 8, 128, sequences=4, max_tokens=1024, dtype=dtype)
    assert c.k_pages.shape == (4096, 8, 64, 128) and c.k_pages.dtype is dtype and not c.v_pages.float().any()
    del c
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    c = PagedCache(4096, 64, 8, 128, sequences=4, max_tokens=1024, dtype=dtype)
    pages = 2 * c.k_pages.numel() * c.k_pages.element_size()
    assert torch.cuda.max_memory_allocated() - before < 1.01 * pages + 2 ** 20


def test_refusals_without_a_gpu():
    import ctypes
    from thunderworld_b200 import _lib
    lib, ref = _lib.load(), ctypes.byref
    ok = dict(k_pages=256, v_pages=256, table=256, lengths=256, refs=256, k_stride_page=4096, k_stride_head=2048, v_stride_page=4096, v_stride_head=2048,
              table_stride=4, sequences=3, max_pages=4, pages=8, hk=2, page=16, dim=128)
    rows = dict(k=256, v=256, k_stride_row=256, k_stride_head=128, v_stride_row=256, v_stride_head=128, batch=2, rows=2)
    assert lib.tw_cache_append(None, None, None, None) == 1 and lib.tw_cache_fork(None, None, None, 1, None, None) == 1
    assert lib.tw_cache_free(None, None, 1, None) == 1 and lib.tw_cache_compact(None, None, None, None) == 1
    for bad, status in ((dict(table=None), 1), (dict(pages=0), 1), (dict(hk=0), 1), (dict(page=12), 2), (dict(dim=96), 2), (dict(sequences=65537), 9),
                        (dict(max_pages=1 << 27), 9), (dict(k_pages=264), 3), (dict(v_stride_page=4092), 3)):
        c = _lib.Cache(**(ok | bad))
        assert lib.tw_cache_append(ref(c), ref(_lib.AppendArgs(**rows)), 256, None) == status, bad
        assert lib.tw_cache_fork(ref(c), 256, 256, 1, 256, None) == status and lib.tw_cache_compact(ref(c), None, 256, None) == status
    c = _lib.Cache(**ok)
    for bad, status in ((dict(k=None), 1), (dict(batch=0), 1), (dict(rows=3), 1), (dict(batch=4, rows=4), 1), (dict(k=264), 3), (dict(v_stride_row=250), 3),
                        (dict(batch=65537, rows=65537, slots=256), 9)):
        assert lib.tw_cache_append(ref(c), ref(_lib.AppendArgs(**(rows | bad))), 256, None) == status, bad
    assert lib.tw_cache_append(ref(c), ref(_lib.AppendArgs(**rows)), None, None) == 1 and lib.tw_cache_append(ref(c), ref(_lib.AppendArgs(**rows)), 264, None) == 3
    assert lib.tw_cache_fork(ref(c), None, 256, 1, 256, None) == 1 and lib.tw_cache_fork(ref(c), 256, 256, 0, 256, None) == 1
    assert lib.tw_cache_free(ref(c), 256, 0, None) == 1 and lib.tw_cache_compact(ref(c), None, None, None) == 1
    assert lib.tw_cache_append_workspace(0, 1) == 0 and lib.tw_cache_fork_workspace(0) == 0 and lib.tw_cache_compact_workspace(0) == 0


@gpu
@pytest.mark.parametrize('entry', [-1, -2 ** 31, 9, 2 ** 31 - 1])
def test_a_bad_entry_of_the_last_page_leaves_an_append_undone(entry):
    """The page that the next row belongs to is not in the pool: no length, page or row changes, for the sequences beside it neither."""
    from thunderworld_b200 import ops
    cache = make(9, 4, 1, 64, False, sequences=4, tokens=32)
    x = torch.randn(20, 1, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1]), i32([0, 6, 14]))       # 2 pages, the second torn; 2 full pages
    cache.table[0, 1] = entry
    model = Model(cache)
    cache.append(x, x, i32([0, 2]), i32([0, 1, 8]))
    assert ops.device_status() == 11
    model.same(cache)
    ops.reset_device_status()
    cache.append(x, x, i32([0, 1, 2]), i32([0, 0, 3, 8]))  # no row for that sequence, which is then not looked at
    model.append(x, x, [1, 2], [0, 3, 8])
    model.same(cache)
    cache.check()
    cache.table[1, 1] = entry                              # a full page that no new row lies in
    model.table[1][1] = entry
    cache.append(x, x, i32([1]), i32([0, 1]))
    model.append(x, x, [1], [0, 1])
    model.same(cache)
    cache.check()


@gpu
@pytest.mark.parametrize('entry', [-1, -2 ** 31, 40, 2 ** 31 - 1])
@pytest.mark.parametrize('at', [0, 3, 6])
@pytest.mark.parametrize('count', [1, 2, 5])
def test_a_bad_entry_of_a_parent_leaves_a_fork_undone(entry, at, count):
    """A full page (0, 3) or the torn last one (6) of one of the parents is not in the pool: no child is made, no count raised."""
    from thunderworld_b200 import ops
    cache = make(40, 4, 2, 64, False, sequences=12, tokens=64)
    x = torch.randn(40, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1]), i32([0, 27, 36]))      # 7 and 3 pages, both with a torn one
    good = int(cache.table[0, at])
    cache.table[0, at] = entry
    model = Model(cache)
    cache.fork(i32(([1] * (count - 1) + [0])), i32(range(2, 2 + count)))
    assert ops.device_status() == 11
    model.same(cache)
    ops.reset_device_status()
    cache.table[0, at] = model.table[0][at] = good
    cache.table[0, 7] = entry                              # behind the sequence's pages: nobody's
    model.table[0][7] = entry
    cache.fork(i32([1, 0]), i32([3, 2]))
    model.fork([1, 0], [3, 2])
    model.same(cache)
    cache.check()


@gpu
def test_forks_of_more_sequences_than_threads():
    from thunderworld_b200 import ops
    cache = make(3000, 2, 1, 64, False, sequences=2700, tokens=20)
    x = torch.randn(1300 * 3, 1, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x[:3900], x[:3900], i32(range(1300)), i32(range(0, 3901, 3)))
    good, before = int(cache.table[1290, 0]), [t.clone() for t in (cache.table, cache.lengths, cache.refs)]
    cache.table[1290, 0] = 3000
    cache.fork(i32(range(100, 1300)), i32(range(1300, 2500)))
    assert ops.device_status() == 11
    ops.reset_device_status()
    cache.table[1290, 0] = good
    assert all(torch.equal(a, b) for a, b in zip(before, (cache.table, cache.lengths, cache.refs)))
    cache.fork(i32(range(100, 500)), i32(range(1300, 1700)))
    assert ops.device_status() == 0 and torch.equal(cache.table[1300:1700, 0], cache.table[100:500, 0])
    assert cache.table[1300:1700, 1].tolist() == list(range(2600, 3000)) and (cache.lengths[1300:1700] == 3).all()


@gpu
@pytest.mark.parametrize('entry', [-1, 40, 2 ** 31 - 1])
def test_compact_leaves_a_bad_entry_as_it_is(entry):
    """And reports it; the good ones' pages move, and are found, all the same."""
    from thunderworld_b200 import ops
    cache = make(40, 4, 2, 64, False, sequences=6, tokens=64)
    x = torch.randn(60, 2, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    cache.append(x, x, i32([0, 1, 2]), i32([0, 20, 39, 60]))
    cache.free(i32([0]))
    cache.table[1, 2] = entry
    model = Model(cache)
    assert int(cache.compact()) == model.compact()
    assert ops.device_status() == 11
    ops.reset_device_status()
    model.same(cache)


@gpu
def test_offsets_that_hold_nothing_are_refused():
    """cu has one offset at least: an empty one is a mistake, not a call with nothing to do."""
    cache = make(6, 4, 2, 64, False)
    x = torch.zeros(2, 2, 64, device='cuda', dtype=torch.bfloat16)
    for slots in (None, i32([])):
        with pytest.raises(ValueError, match='one offset more'):
            cache.append(x, x, slots, i32([]))
    cache.append(x, x, None, i32([0]))
    cache.append(x, x, i32([]), i32([2]))
    assert not cache.lengths.any()
