"""The token operators called by several threads at once: on one stream, where the calls' launches must not mix, and on streams of their
own. Each thread has its own inputs and cache; what it gets has to be, bit for bit, what a call alone gives."""
import threading
import pytest
import torch

gpu = pytest.mark.gpu


def together(bodies):
    """Runs the bodies in threads of their own; raises what any of them raised."""
    wrong, start = [], threading.Barrier(len(bodies))

    def go(body):
        try:
            start.wait()
            body()
        except BaseException as e:                         # noqa: B036  (handed to the caller)
            wrong.append(e)
    threads = [threading.Thread(target=go, args=(b,)) for b in bodies]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    if wrong:
        raise wrong[0]
    torch.cuda.synchronize()


@gpu
@pytest.mark.parametrize('own_streams', [False, True])
def test_attention_of_several_threads(own_streams):
    """Batches of different sizes, so that the calls' borders and parts lie at different places of a scratch."""
    from thunderworld_b200 import ops
    cases = []
    for i, (lens, hq) in enumerate((([3000], 32), ([700, 1, 2500], 8), ([90] * 40, 4), ([5000, 4000], 16))):
        g = torch.Generator().manual_seed(i)
        pages = [-(-n // 16) for n in lens]
        kp, vp = torch.randn(2, sum(pages), 4, 16, 128, generator=g).bfloat16().cuda()
        order, table = torch.randperm(sum(pages), generator=g).tolist(), torch.full((len(lens), max(pages)), -1, dtype=torch.int32)
        for b, n in enumerate(pages):
            table[b, :n] = torch.tensor([order.pop() for _ in range(n)])
        q = torch.randn(len(lens), hq, 128, generator=g).bfloat16().cuda()
        args = q, kp, vp, table.cuda(), torch.tensor(lens, dtype=torch.int32, device='cuda')
        cases.append((args, ops.paged_attention(*args, return_lse=True), torch.cuda.Stream() if own_streams else torch.cuda.current_stream()))
    torch.cuda.synchronize()
    got = [[] for _ in cases]

    def body(i):
        args, _, stream = cases[i]
        with torch.cuda.stream(stream):
            for _ in range(200):
                got[i].append(ops.paged_attention(*args, return_lse=True))
    together([lambda i=i: body(i) for i in range(len(cases))])
    for (_, want, _), results in zip(cases, got):
        assert all(torch.equal(out, want[0]) and torch.equal(lse, want[1]) for out, lse in results)
    assert ops.device_status() == 0


@gpu
def test_caches_of_several_threads():
    """Append, fork, free and compact on a cache per thread, one stream: tables, counts and rows as one thread leaves them."""
    from thunderworld_b200 import PagedCache, ops
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device='cuda')  # noqa: E731

    def make(i):
        return PagedCache(400, 4, 2, 64, sequences=8 + i, max_tokens=200)

    def use(cache, i):
        n = 3 + i
        slots, spare = i32(list(range(n))), i32([n, n + 1])
        g = torch.Generator().manual_seed(i)
        x = torch.randn(40, n, 2, 64, generator=g).bfloat16().cuda()
        for t in range(40):
            cache.append(x[t], x[t], slots)
            if t % 7 == 3:
                cache.fork(slots[:2], spare)
                cache.free(spare[:1])
                cache.compact()
                cache.free(spare)
    want = [make(i) for i in range(4)]
    for i, cache in enumerate(want):
        use(cache, i)
    caches = [make(i) for i in range(4)]
    torch.cuda.synchronize()
    together([lambda i=i: use(caches[i], i) for i in range(4)])
    for a, b in zip(caches, want):
        for name in ('table', 'lengths', 'refs', 'k_pages', 'v_pages'):
            assert torch.equal(getattr(a, name), getattr(b, name)), name
    assert ops.device_status() == 0
