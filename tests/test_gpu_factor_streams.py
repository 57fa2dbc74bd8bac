"""Tensor factors (max|y| / 2688 of the pointwise producers) of calls that run side by side: on two streams, and
as two captured graphs replayed on two streams. Each call has the maximum of its own tensor, whatever the other's is."""
import pytest
import torch

gpu = pytest.mark.gpu


def producers(i):
    """Calls of one kind of producer with inputs of their own; the second's are eight times the first's."""
    from thunderworld_b200 import ops
    g = torch.Generator().manual_seed(i)
    a, b = (torch.randn(1500, 2048, generator=g) * 8 ** i).bfloat16().cuda(), torch.randn(1500, 2048, generator=g).bfloat16().cuda()
    w = (torch.randn(2048, generator=g).abs() * 8 ** i).bfloat16().cuda()
    return dict(relu2=lambda: ops.activate_with_factor(a), mul=lambda: ops.activate_with_factor(a, b),
                gelu=lambda: ops.activate_with_factor(a, mode='gelu_tanh'), norm=lambda: ops.rms_norm(b, w, want_factor=True))


@gpu
@pytest.mark.parametrize('kind', ['relu2', 'mul', 'gelu', 'norm'])
def test_two_streams(kind):
    calls = [producers(i)[kind] for i in range(2)]
    want = [call() for call in calls]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for _ in range(50):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got.append((i, calls[i]()))
    torch.cuda.synchronize()
    for i, (y, factor) in got:
        assert torch.equal(y, want[i][0]) and torch.equal(factor, want[i][1])


@gpu
@pytest.mark.parametrize('kind', ['gelu', 'norm'])
def test_two_graphs(kind):
    calls = [producers(i)[kind] for i in range(2)]
    want = [call() for call in calls]
    made = []
    for call in calls:
        graph = torch.cuda.CUDAGraph()
        torch.cuda.synchronize()
        with torch.cuda.graph(graph):
            out = [call() for _ in range(8)]
        made.append((graph, out, torch.cuda.Stream()))
    torch.cuda.synchronize()
    for _ in range(10):
        for graph, _, stream in made:
            with torch.cuda.stream(stream):
                graph.replay()
    torch.cuda.synchronize()
    for (_, out, _), (y, factor) in zip(made, want):
        assert all(torch.equal(a, y) and torch.equal(f, factor) for a, f in out)
