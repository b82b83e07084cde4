"""The products with an epilogue, the gated delta rule and the slot operators together, as a served layer uses them: a prompt by chunks,
its state forked, tokens decoded, slots freed and compacted between steps, and the same tokens without any of that."""
import pytest

from gpu_util import say

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

DEV = "cuda:0"
C, HK, HV, K, V, LAYERS = 256, 2, 4, 64, 64, 2


def _norm(x):
    return (x.float() * torch.rsqrt(x.float().square().mean(-1, keepdim=True) + 1e-6)).bfloat16()


class _Layer:
    def __init__(self, gen):
        from rwkv_next_amd.kernels import prepack_dense
        w = lambda k, n: prepack_dense((torch.randn(k, n, device=DEV, generator=gen) / k ** 0.5).bfloat16())  # noqa: E731
        self.qkv, self.step, self.write = w(C, 2 * HK * K + HV * V), w(C, HV), w(C, HV)
        self.out, self.up, self.down = w(HV * V, C), w(C, 2 * C), w(2 * C, C)
        self.bias = torch.randn(HV, device=DEV, generator=gen)

    def __call__(self, x, pool, slots, **kw):
        from rwkv_next_amd.kernels import dense_matmul, gated_delta_pool_
        n = _norm(x)
        f = dense_matmul(n, self.qkv)
        q, k, v = (f[..., :HK * K].unflatten(-1, (HK, K)), f[..., HK * K:2 * HK * K].unflatten(-1, (HK, K)),
                   f[..., 2 * HK * K:].unflatten(-1, (HV, V)))
        g = -dense_matmul(n, self.step, bias=self.bias, activation="sigmoid", out_dtype=torch.float32)
        beta = dense_matmul(n, self.write, activation="sigmoid", out_dtype=torch.float32)
        o = gated_delta_pool_(q, k, v, g, beta, pool, slots, qk_norm=True, **kw)
        x = dense_matmul(o.flatten(2), self.out, residual=x)
        return dense_matmul(dense_matmul(_norm(x), self.up, activation="relu2"), self.down, residual=x)


def _forward(layers, x, pools, slots, **kw):
    for i, layer in enumerate(layers):
        x = layer(x, pools[i], slots, **kw)
    return x


def test_a_served_layer():
    from rwkv_next_amd.kernels import SlotCaches
    gen = torch.Generator(device=DEV).manual_seed(0)
    layers = [_Layer(gen) for _ in range(LAYERS)]
    S = 10
    pools = torch.randn(LAYERS, S, HV, K, V, device=DEV, generator=gen)
    last = torch.zeros(S, C, device=DEV, dtype=torch.bfloat16)  # each sequence's last hidden state
    caches = SlotCaches(pools, (last, 0))
    prompts = [150, 7, 64]
    slots = torch.tensor([8, 3, 5], device=DEV)
    cu = torch.tensor([0] + prompts, device=DEV).cumsum(0).int()
    x = torch.randn(1, sum(prompts), C, device=DEV, generator=gen).bfloat16()
    say("prompts")
    caches.free_slots(slots)
    y = _forward(layers, x, pools, slots, cu_seqlens=cu)
    last[slots] = y[0, cu[1:].long() - 1]
    say("fork")
    caches.copy_slots(torch.tensor([8, 8, 3], device=DEV), torch.tensor([0, 9, 6], device=DEV))
    slots = torch.tensor([8, 0, 9, 3, 6, 5], device=DEV)
    alone = {int(s): (pools[:, s:s + 1].clone(), last[s].clone()) for s in slots}

    def step(where):
        h = last[where][:, None]
        z = _forward(layers, h, pools, where)
        last[where] = z[:, 0]
        return z[:, 0]

    got = [step(slots)]
    for s in (8, 0, 9):  # forks of one prompt agree, to the bit
        assert torch.equal(got[0][0], got[0][(slots == s).nonzero()[0, 0]])
    say("free and compact")
    names = slots.tolist()
    caches.free_slots(torch.tensor([0, 5], device=DEV))
    keep = torch.tensor([i for i, s in enumerate(names) if s not in (0, 5)], device=DEV)
    live = torch.zeros(S, dtype=torch.bool, device=DEV)
    live[slots[keep]] = True
    where, count = caches.compact_slots(live)
    assert int(count) == 4
    moved = where[slots[keep]]
    assert sorted(moved.tolist()) == [0, 1, 2, 3]
    got += [step(moved), step(moved)]
    say("the same alone")
    for i, s in enumerate(names):
        p, h = alone[s]
        for t in range(3 if s not in (0, 5) else 1):
            h = _forward(layers, h[None, None], p, torch.zeros(1, dtype=torch.int64, device=DEV))[0, 0]
            row = i if t == 0 else keep.tolist().index(i)
            assert torch.equal(h, got[t][row]), (s, t)


def test_a_captured_decode_step():
    gen = torch.Generator(device=DEV).manual_seed(1)
    layers = [_Layer(gen) for _ in range(LAYERS)]
    pools = torch.randn(LAYERS, 6, HV, K, V, device=DEV, generator=gen)
    slots = torch.tensor([5, 1, 2], device=DEV)
    x = torch.randn(3, 1, C, device=DEV, generator=gen).bfloat16()
    mine, start = pools.clone(), x.clone()
    _forward(layers, x, mine, slots)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        x.copy_(_forward(layers, x, mine, slots))
    mine.copy_(pools)
    x.copy_(start)
    want = start
    for t in range(4):
        g.replay()
        want = _forward(layers, want, pools, slots)
        torch.cuda.synchronize()
        assert torch.equal(x, want) and torch.equal(mine, pools), t
