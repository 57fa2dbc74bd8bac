"""The operators of a token at a time together, as a layer uses them: norm, QKV product, rotary embedding, cache append, attention over
the cache, output product, gated residual with the next norm, FFN, residual; several sequences, some of them forked and released on
the way, eager and as a replayed graph.

Tolerance: the reference is the layer in 64 bits without any rounding, over the whole history. A step rounds to bf16 twelve times
(norm, qkv, q and k norm and rotation in three, rows in the cache, attention, product, residual, norm, up, activation, down,
residual), each at most 2^-8 of its value; the norms and softmax carry a relative error on about as it is (scores are of the order of
one here, so an error of theirs is that of the probabilities): under 12 * 2^-8 = 0.047 of the output's norm in the worst case."""
import pytest
import torch

gpu = pytest.mark.gpu
HEADS, KV, DIM, HIDDEN, FFN = 4, 2, 128, 512, 1024


class Layer:
    def __init__(self, seed=0):
        from thunderworld_b200 import FP4Linear
        g = torch.Generator().manual_seed(seed)
        w = lambda n, k: (torch.randn(n, k, generator=g) * k ** -.5).bfloat16().cuda()  # noqa: E731
        self.qkv, self.out, self.up, self.down = (FP4Linear.from_float(w(n, k)) for n, k in (
            ((HEADS + 2 * KV) * DIM, HIDDEN), (HIDDEN, HEADS * DIM), (FFN, HIDDEN), (HIDDEN, FFN)))
        self.gate = (torch.rand(2, HIDDEN, generator=g) + .5).bfloat16().cuda()
        self.weights = (1 + .1 * torch.randn(2, HIDDEN, generator=g)).bfloat16().cuda()

    def dense(self, layer):
        lut = torch.tensor([0., .5, 1., 1.5, 2., 3., 4., 6., -0., -.5, -1., -1.5, -2., -3., -4., -6.], dtype=torch.float64, device='cuda')
        c = layer.weight_codes
        values = lut[torch.stack([c & 15, c >> 4], -1).flatten(-2).long()] * layer.weight_scales.double().repeat_interleave(16, -1)
        return values * layer.weight_global_scale.double()

    def step(self, x, cache, slots, cos, sin):
        """x [batch, 1, HIDDEN] in place; cos / sin [batch, DIM]: row b's position."""
        from thunderworld_b200 import ops
        b = x.shape[0]
        y = ops.rms_norm(x, self.weights[0])
        qkv = self.qkv.matvec(y).view(b, HEADS + 2 * KV, DIM)
        q = ops.rope_heads(qkv[:, :HEADS], cos, sin, norm=True)
        k = ops.rope_heads(qkv[:, HEADS:HEADS + KV], cos, sin, norm=True)
        cache.append(k, qkv[:, HEADS + KV:], slots)
        a = self.out.matvec(cache.attend(q, slots).view(b, 1, HEADS * DIM))
        y = ops.gate_residual_norm_(x, a, self.gate[:1].expand(b, -1).contiguous(), weight=self.weights[1])
        u, _ = ops.activate_with_factor(self.up.matvec(y), mode='gelu_tanh')
        ops.gate_residual_(x, self.gate[1:].expand(b, -1).contiguous(), self.down.matvec(u))
        return x

    def reference(self, history):
        """history [tokens, HIDDEN] in 64 bits, one sequence: the layer's outputs."""
        norm = lambda t: t / (t.square().mean(-1, keepdim=True) + 1e-6).sqrt()  # noqa: E731
        x = history
        cos, sin = (t.double() for t in tables(len(x)))
        qkv = (norm(x) * self.weights[0].double()) @ self.dense(self.qkv).T
        qkv = qkv.view(len(x), HEADS + 2 * KV, DIM)

        def rope(t):
            t = norm(t)
            return t * cos[:, None] + torch.cat([-t[..., DIM // 2:], t[..., :DIM // 2]], -1) * sin[:, None]
        q, k, v = rope(qkv[:, :HEADS]), rope(qkv[:, HEADS:HEADS + KV]), qkv[:, HEADS + KV:]
        score = torch.einsum('qhgd,khd->hgqk', q.view(len(x), KV, HEADS // KV, DIM), k) * DIM ** -.5
        score = score.masked_fill(torch.ones(len(x), len(x), dtype=torch.bool, device='cuda').triu(1), float('-inf'))
        a = torch.einsum('hgqk,khd->qhgd', score.softmax(-1), v).reshape(len(x), -1) @ self.dense(self.out).T
        x = x + self.gate[0].double() * a
        u = torch.nn.functional.gelu((norm(x) * self.weights[1].double()) @ self.dense(self.up).T, approximate='tanh')
        return x + self.gate[1].double() * (u @ self.dense(self.down).T)


def tables(tokens):
    from thunderworld_b200.cosmos.dit import rope_tables
    return rope_tables(tokens, 'cuda')


@gpu
def test_a_layer_token_by_token():
    from thunderworld_b200 import PagedCache, ops
    layer, tokens, batch = Layer(), 40, 3
    cos, sin = tables(tokens)
    cache = PagedCache(60, 4, KV, DIM, sequences=8, max_tokens=64)
    g = torch.Generator().manual_seed(1)
    inputs = torch.randn(batch, tokens, HIDDEN, generator=g).bfloat16().cuda()
    slots = [5, 0, 2]
    wants = [layer.reference(inputs[b].double()) for b in range(batch)]
    for t in range(tokens):
        if t == 17:                                       # sequence 0 goes on as a copy of itself, in another slot
            cache.fork(torch.tensor([5], dtype=torch.int32, device='cuda'), torch.tensor([7], dtype=torch.int32, device='cuda'))
            cache.free(torch.tensor([5], dtype=torch.int32, device='cuda'))
            slots[0] = 7
        if t == 23:
            cache.compact()
        s = torch.tensor(slots, dtype=torch.int32, device='cuda')
        row = lambda m: m[t:t + 1].expand(batch, -1).contiguous()  # noqa: E731
        x = layer.step(inputs[:, t:t + 1].clone(), cache, s, row(cos), row(sin))
        for b in range(batch):
            want = wants[b][t]
            assert (x[b, 0].double() - want).norm() <= 12 * 2. ** -8 * want.norm(), (t, b)
    cache.check()
    assert ops.device_status() == 0


@gpu
def test_the_step_as_a_graph():
    from thunderworld_b200 import PagedCache
    layer, batch = Layer(3), 5
    made = [PagedCache(40, 8, KV, DIM, sequences=5, max_tokens=64, dtype=dtype) for dtype in (torch.bfloat16,) * 2]
    cos, sin = tables(64)
    slots = torch.arange(5, dtype=torch.int32, device='cuda')
    x = torch.zeros(batch, 1, HIDDEN, device='cuda', dtype=torch.bfloat16)
    c, s = torch.zeros(batch, DIM, device='cuda'), torch.zeros(batch, DIM, device='cuda')
    layer.step(x.clone(), PagedCache(8, 8, KV, DIM, sequences=5, max_tokens=64), slots, c, s)          # every kernel has run once
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        layer.step(x, made[0], slots, c, s)
    g = torch.Generator().manual_seed(2)
    for t in range(20):
        inputs = torch.randn(batch, 1, HIDDEN, generator=g).bfloat16().cuda()
        x.copy_(inputs)
        c.copy_(cos[t].expand(batch, -1))
        s.copy_(sin[t].expand(batch, -1))
        graph.replay()
        want = layer.step(inputs.clone(), made[1], slots, c, s)
        assert torch.equal(x, want)
        assert torch.equal(made[0].table, made[1].table) and torch.equal(made[0].k_pages, made[1].k_pages)
