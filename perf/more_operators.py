"""What the operators of a served layer with a recurrent state are measured on.

Three operators, each through the package's public entry points (`own` true) or in its plain form:

    dense   a product with 16-bit weights, with bias, activation and residual in its epilogue: a layer's projections, its
            channel mix, its low-rank parts
    delta   the gated delta rule over dense or ragged rows, states in a pool of slots: decode, verification and prefill
    slots   copies (forks) of a cache's slots, their compaction, their freeing, over all tensors of a model's cache

The widths 768, 2560, 4096, 10240 and 16384, heads of 64 and the vocabulary of 65536 are RWKV-7's; the others are generic.
"""
import math
import os
import random
import sys

import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infer-next_amd"))

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
CHUNK = 64  # tokens that the plain form of the delta rule takes at a time


# ----------------------------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user's decode step, a layer's output projection onto the residual stream: latency
        dict(name="dense_m1_4096x4096", op="dense", M=1, K=4096, N=4096, dtype="bf16", bias=False, act="none", residual=True),
        # a small odd batch through the narrow side of a low-rank part
        dict(name="dense_m23_2560x96_f16", op="dense", M=23, K=2560, N=96, dtype="f16", bias=True, act="tanh",
             residual=False),
        # the serving batch's channel mix: the squared ReLU, the largest weight of a layer
        dict(name="dense_m64_4096x16384", op="dense", M=64, K=4096, N=16384, dtype="bf16", bias=False, act="relu2",
             residual=False),
        # an odd prompt through the channel mix's way back
        dict(name="dense_m500_10240x2560_f16", op="dense", M=500, K=10240, N=2560, dtype="f16", bias=True, act="none",
             residual=True),
        # a long prompt's channel mix
        dict(name="dense_m4096_4096x16384", op="dense", M=4096, K=4096, N=16384, dtype="bf16", bias=False, act="relu2",
             residual=False),
        # one user's token
        dict(name="delta_b1", op="delta", rows=1, T=1, ragged=0, slots=4, Hk=16, Hv=32, K=128, V=128, norm=True),
        # the serving batch's tokens, slots in any order
        dict(name="delta_b64", op="delta", rows=64, T=1, ragged=0, slots=128, Hk=16, Hv=32, K=128, V=128, norm=True),
        # an odd prompt, few small heads, operands normalised before
        dict(name="delta_t500_h12", op="delta", rows=1, T=500, ragged=0, slots=4, Hk=12, Hv=12, K=64, V=64, norm=False),
        # a long prompt of one user
        dict(name="delta_t4096", op="delta", rows=1, T=4096, ragged=0, slots=4, Hk=16, Hv=32, K=128, V=128, norm=True),
        # a step of mixed work: eight prompts of up to 2048 tokens and 56 sequences of one token, one ragged call
        dict(name="delta_mixed", op="delta", rows=64, T=2048, ragged=8, slots=128, Hk=16, Hv=32, K=128, V=128, norm=True),
        # four prompts' states forked to 28 slots: states, token shifts and penalty counts of a small model
        dict(name="slots_fork", op="slots", do="copy", layers=12, slots=64, H=12, C=768, src=4, n=28),
        # a pool with holes after requests ended, a mid-size model
        dict(name="slots_compact", op="slots", do="compact", layers=32, slots=128, H=40, C=2560, src=70, n=17),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("dense", "dense", "delta", "delta", "slots"))
    if op == "dense":
        K = 32 * _log_int(rng, 1, 512)
        N = _log_int(rng, 16, 16384)
        M = min(_log_int(rng, 1, 4096), 4096 * 4096 * 16384 // (K * N))
        return dict(op=op, M=M, K=K, N=N, dtype=rng.choice(("bf16", "f16")), bias=rng.random() < 0.5,
                    act=rng.choice(("none", "relu", "relu2", "tanh", "sigmoid", "silu", "gelu")), residual=rng.random() < 0.5)
    if op == "delta":
        Hk, K, V = _log_int(rng, 1, 16), rng.choice((64, 128)), rng.choice((64, 128))
        Hv = Hk * rng.choice((1, 2, 4) if Hk <= 8 else (1, 2))
        kind = rng.choice(("decode", "verify", "prefill", "ragged"))
        if kind in ("decode", "verify"):
            rows, T, ragged = _log_int(rng, 1, 64), 1 if kind == "decode" else rng.randint(2, 8), 0
        elif kind == "prefill":
            T = _log_int(rng, 9, 4096)
            rows, ragged = rng.randint(1, max(1, min(4, 4096 // T))), 0
        else:
            rows, T, ragged = _log_int(rng, 2, 64), _log_int(rng, 9, 2048), rng.randint(1, 4)
            rows = max(rows, ragged)
        return dict(op=op, rows=rows, T=T, ragged=ragged, slots=rows + rng.randint(0, 32), Hk=Hk, Hv=Hv, K=K, V=V,
                    norm=rng.random() < 0.5)
    H = _log_int(rng, 1, 40)
    layers, slots = _log_int(rng, 1, 32), _log_int(rng, 8, 128)
    n = rng.randint(1, slots // 4)
    do = rng.choice(("copy", "compact", "free"))
    # compact: n slots move, src stay; copy: n destinations of src sources
    src = rng.randint(1, n) if do == "copy" else rng.randint(0, slots - 2 * n)
    return dict(op=op, do=do, layers=layers, slots=slots, H=H, C=64 * H + rng.choice((0, 0, 1)), src=src, n=n)


# ----------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ----------------------------------------------------------------------------------------------------------------
def _dense_inputs(case, gen, dev):
    M, K, N, t = case["M"], case["K"], case["N"], DTYPES[case["dtype"]]
    s = dict(a=torch.randn(M, K, device=dev, generator=gen).to(t),
             w=(torch.randn(K, N, device=dev, generator=gen) / math.sqrt(K)).to(t))
    if case["bias"]:
        s["bias"] = torch.randn(N, device=dev, generator=gen) * 0.5
    if case["residual"]:
        s["residual"] = torch.randn(M, N, device=dev, generator=gen).to(t)
    return s


def lengths(case):
    """Tokens of each row: all T, or `ragged` rows of up to T and the others of one, in mixed order."""
    if not case["ragged"]:
        return [case["T"]] * case["rows"]
    r = random.Random("%(rows)d %(T)d %(ragged)d" % case)
    lens = [r.randint(max(1, case["T"] // 8), case["T"]) for _ in range(case["ragged"])] + [1] * (case["rows"] - case["ragged"])
    r.shuffle(lens)
    return lens


def _delta_inputs(case, gen, dev):
    rows, T, Hk, Hv, K, V, S = (case[n] for n in ("rows", "T", "Hk", "Hv", "K", "V", "slots"))
    lens = lengths(case)
    B, T = (1, sum(lens)) if case["ragged"] else (rows, T)
    rand = lambda *n: torch.rand(*n, device=dev, generator=gen)  # noqa: E731
    randn = lambda *n: torch.randn(*n, device=dev, generator=gen)  # noqa: E731
    q, k = randn(B, T, Hk, K), randn(B, T, Hk, K)
    if not case["norm"]:  # the program has normalised them
        q, k = (x / x.square().sum(dim=-1, keepdim=True).sqrt() for x in (q, k))
    s = dict(q=q.bfloat16(), k=k.bfloat16(), v=randn(B, T, Hv, V).bfloat16())
    # decays of a trained layer: a rate for each head, a step for each token; writing strengths in (0, 1)
    s["g"] = -(1 + 15 * rand(Hv)) * torch.exp(rand(B, T, Hv) * (math.log(0.1) - math.log(0.001)) + math.log(0.001))
    s["beta"] = torch.sigmoid(randn(B, T, Hv))
    s["pool"] = randn(S, Hv, K, V) * 0.1
    s["slots"] = torch.randperm(S, device=dev, generator=gen)[:rows]
    if case["ragged"]:
        ends = torch.tensor([0] + lens, dtype=torch.int64).cumsum(0)
        s["cu"] = ends.to(device=dev, dtype=torch.int32)
        at = torch.arange(max(lens))[None, :] + ends[:-1, None]  # where the padded rows' tokens are; for the plain form
        s["pad"] = at.clamp_max(T - 1).to(dev)
        s["there"] = (torch.arange(max(lens))[None, :] < torch.tensor(lens)[:, None]).to(dev)
    return s


def _slots_inputs(case, gen, dev):
    L, S, H, C, n = (case[k] for k in ("layers", "slots", "H", "C", "n"))
    s = dict(states=torch.randn(L, S, H, 64, 64, device=dev, generator=gen),
             shifts=torch.randn(L, S, 2, C, device=dev, generator=gen).bfloat16(),
             counts=torch.randint(0, 4, (S, 65536), device=dev, dtype=torch.int32, generator=gen))
    order = torch.randperm(S, device=dev, generator=gen)
    if case["do"] == "copy":
        s["dst"] = order[:n].contiguous()
        s["src"] = order[n + torch.randint(0, case["src"], (n,), device=dev, generator=gen)]
    elif case["do"] == "free":
        s["dst"] = order[:n].contiguous()
    else:  # of the first k = src + n slots n are free, of those behind n are live
        k = case["src"] + n
        live = torch.arange(S, device=dev) < k
        live[torch.randperm(k, device=dev, generator=gen)[:n]] = False
        live[k + torch.randperm(S - k, device=dev, generator=gen)[:n]] = True
        s["live"] = live
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    inputs = {"dense": _dense_inputs, "delta": _delta_inputs, "slots": _slots_inputs}[case["op"]]
    s = dict(inputs(case, gen, dev), case=dict(case))
    if own:
        from rwkv_next_amd import kernels
        s["kernels"] = kernels
        if case["op"] == "dense":  # laid out once, when the weights are loaded
            s["weight"] = kernels.prepack_dense(s["w"])
        if case["op"] == "slots":
            s["caches"] = kernels.SlotCaches((s["states"], 1), (s["shifts"], 1), (s["counts"], 0))
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"dense": _dense_own, "delta": _delta_own, "slots": _slots_own}[op](state)
    return {"dense": _dense_plain, "delta": _delta_plain, "slots": _slots_plain}[op](state)


def _dense_own(s):
    return s["kernels"].dense_matmul(s["a"], s["weight"], bias=s.get("bias"), activation=s["case"]["act"],
                                     residual=s.get("residual"))


def _delta_own(s):
    o = s["kernels"].gated_delta_pool_(s["q"], s["k"], s["v"], s["g"], s["beta"], s["pool"], s["slots"],
                                       cu_seqlens=s.get("cu"), qk_norm=s["case"]["norm"])
    return o, s["pool"]


def _slots_own(s):
    out = [s["states"], s["shifts"], s["counts"]]
    if s["case"]["do"] == "copy":
        s["caches"].copy_slots(s["src"], s["dst"])
    elif s["case"]["do"] == "free":
        s["caches"].free_slots(s["dst"])
    else:
        out += s["caches"].compact_slots(s["live"])
    return out


def _dense_plain(s):
    x = s["a"].float() @ s["w"].float()
    if "bias" in s:
        x = x + s["bias"]
    act = s["case"]["act"]
    if act == "relu":
        x = x.clamp_min(0)
    elif act == "relu2":
        x = x.clamp_min(0).square()
    elif act == "tanh":
        x = torch.tanh(x)
    elif act == "sigmoid":
        x = torch.sigmoid(x)
    elif act == "silu":
        x = x * torch.sigmoid(x)
    elif act == "gelu":
        x = 0.5 * x * (1 + torch.erf(x * math.sqrt(0.5)))
    if "residual" in s:
        x = x + s["residual"].float()
    return x.to(s["a"].dtype)


def _delta_plain(s):
    case = s["case"]
    q, k, v, g, beta = s["q"].float(), s["k"].float(), s["v"].float(), s["g"], s["beta"]
    if "cu" in s:  # rows side by side, padded with tokens that neither decay nor write
        there = s["there"][..., None]
        q, k, v = (x[0][s["pad"]] for x in (q, k, v))
        g, beta = (x[0][s["pad"]] * there for x in (g, beta))
    if case["norm"]:
        q, k = (x * torch.rsqrt(x.square().sum(dim=-1, keepdim=True) + 1e-6) for x in (q, k))
    q = q * case["K"] ** -0.5
    head = torch.arange(case["Hv"], device=q.device) // (case["Hv"] // case["Hk"])
    q, k = q[:, :, head], k[:, :, head]
    q, k, v, g, beta = (x.transpose(1, 2) for x in (q, k, v, g, beta))  # (rows, heads, tokens, ..)
    steps = _delta_chunks if q.shape[2] > 8 else _delta_tokens
    o, state = steps(q, k, v, g, beta, s["pool"][s["slots"]])
    s["pool"][s["slots"]] = state
    o = o.transpose(1, 2).to(s["v"].dtype)
    if "cu" in s:
        o = o[s["there"]][None]
    return o, s["pool"]


def _delta_tokens(q, k, v, g, beta, S):
    o = []
    for t in range(q.shape[2]):
        S = S * torch.exp(g[:, :, t])[..., None, None]
        d = beta[:, :, t, None] * (v[:, :, t] - (S * k[:, :, t, :, None]).sum(dim=2))
        S = S + k[:, :, t, :, None] * d[:, :, None, :]
        o.append((S * q[:, :, t, :, None]).sum(dim=2))
    return torch.stack(o, dim=2), S


def _delta_chunks(q, k, v, g, beta, S):
    T, dev = q.shape[2], q.device
    more = -T % CHUNK
    pad = lambda x: torch.cat((x, x.new_zeros(*x.shape[:2], more, *x.shape[3:])), dim=2).unflatten(2, (-1, CHUNK))  # noqa: E731
    q, k, v, g, beta = (pad(x) for x in (q, k, v, g, beta))
    c = g.double().cumsum(dim=3)
    at = torch.arange(CHUNK, device=dev)
    before = at[:, None] >= at[None, :]
    decay = torch.exp(torch.where(before, c[..., :, None] - c[..., None, :], -torch.inf)).float()
    gamma, left = torch.exp(c).float()[..., None], torch.exp(c[..., -1:] - c).float()[..., None]
    attn = q @ k.transpose(-1, -2) * decay
    x = -((k @ k.transpose(-1, -2)) * decay * beta[..., None] * (at[:, None] > at[None, :])).double()
    inv = torch.eye(CHUNK, device=dev, dtype=torch.float64) + x
    for _ in range(5):  # the inverse of 1 - x, whose 64th power vanishes: (1 + x)(1 + x^2)(1 + x^4) ..
        x = x @ x
        inv = inv + inv @ x
    inv = inv.float()
    o = torch.empty_like(v)
    for i in range(q.shape[2]):
        r = beta[:, :, i, :, None] * (v[:, :, i] - gamma[:, :, i] * (k[:, :, i] @ S))
        d = inv[:, :, i] @ r
        o[:, :, i] = gamma[:, :, i] * (q[:, :, i] @ S) + attn[:, :, i] @ d
        S = gamma[:, :, i, -1:] * S + (k[:, :, i] * left[:, :, i]).transpose(-1, -2) @ d
    return o.flatten(2, 3)[:, :, :T], S


def _slots_plain(s):
    caches = ((s["states"], 1), (s["shifts"], 1), (s["counts"], 0))
    out = [t for t, _ in caches]
    if s["case"]["do"] == "free":
        for t, dim in caches:
            t.index_fill_(dim, s["dst"], 0)
        return out
    if s["case"]["do"] == "copy":
        src, dst = s["src"], s["dst"]
    else:
        live, at = s["live"], torch.arange(s["live"].numel(), device=s["live"].device)
        count = live.sum()
        dst, src = (~live & (at < count)).nonzero()[:, 0], (live & (at >= count)).nonzero()[:, 0]
        where = torch.where(live, at, -1)
        where[src] = dst
        out += [where, count.to(torch.int32).reshape(1)]
    for t, dim in caches:
        t.index_copy_(dim, dst, t.index_select(dim, src))
    return out


# ----------------------------------------------------------------------------------------------------------------
# what a pass has to do, and its results in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "dense":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": 2 * (K * N + M * K + M * N * (1 + case["residual"])) + 4 * N * case["bias"], "flops": 2 * M * K * N}
    if case["op"] == "delta":
        Hk, Hv, K, V = (case[n] for n in ("Hk", "Hv", "K", "V"))
        tokens = sum(lengths(case))
        return {"bytes": tokens * (4 * Hk * K + 4 * Hv * V + 8 * Hv) + 8 * case["rows"] * Hv * K * V,
                "flops": tokens * Hv * 7 * K * V}
    row = case["layers"] * (case["H"] * 64 * 64 * 4 + 2 * case["C"] * 2) + 65536 * 4
    rows = {"copy": case["n"] + min(case["src"], case["n"]), "free": case["n"], "compact": 2 * case["n"]}[case["do"]]
    return {"bytes": rows * row, "flops": 0}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"dense": _dense_exact, "delta": _delta_exact, "slots": _slots_exact}[case["op"]](case, s)


def _dense_exact(case, s):
    z = torch.mm(s["a"].double(), s["w"].double())
    if case["bias"]:
        z += s["bias"].double()
    f = {"none": lambda y: y, "relu": torch.relu, "relu2": lambda y: torch.relu(y) ** 2, "tanh": torch.tanh,
         "sigmoid": lambda y: 1 / (1 + torch.exp(-y)), "silu": lambda y: y / (1 + torch.exp(-y)),
         "gelu": lambda y: y * torch.special.erfc(-y / math.sqrt(2)) / 2}[case["act"]]
    z = f(z)
    return z + s["residual"].double() if case["residual"] else z


def _delta_exact(case, s):
    """Token by token, the rows that have a token t side by side."""
    lens = lengths(case)
    rows, share = case["rows"], case["Hv"] // case["Hk"]
    q, k, v, g, beta = (s[n].double().flatten(0, 1) for n in ("q", "k", "v", "g", "beta"))
    if case["norm"]:
        q = q / (q.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
        k = k / (k.pow(2).sum(-1, keepdim=True) + 1e-6).sqrt()
    q, k = q.repeat_interleave(share, dim=1) / math.sqrt(case["K"]), k.repeat_interleave(share, dim=1)
    order = sorted(range(rows), key=lambda n: -lens[n])
    starts = torch.tensor([sum(lens[:n]) for n in order], device=q.device)
    slots = s["slots"][torch.tensor(order, device=q.device)]
    pool = s["pool"].double()
    S, o = pool[slots], torch.zeros(v.shape, device=v.device, dtype=torch.float64)
    for t in range(lens[order[0]]):
        n = sum(x > t for x in lens)
        at, H = starts[:n] + t, S[:n]
        H *= g[at].exp()[..., None, None]
        seen = torch.matmul(k[at][..., None, :], H)
        H += k[at][..., :, None] * (beta[at][..., None, None] * (v[at][..., None, :] - seen))
        o[at] = torch.matmul(q[at][..., None, :], H)[..., 0, :]
    pool[slots] = S
    return o.view(s["v"].shape), pool


def _slots_exact(case, s):
    S, order = case["slots"], list(range(case["slots"]))  # which slot each one's contents come from, None: zeros
    if case["do"] == "copy":
        for a, b in zip(s["src"].tolist(), s["dst"].tolist()):
            order[b] = a
    elif case["do"] == "free":
        for b in s["dst"].tolist():
            order[b] = None
    else:
        live = s["live"].tolist()
        count = sum(live)
        holes = [i for i in range(count) if not live[i]]
        for i in range(count, S):
            if live[i]:
                order[holes.pop(0)] = i
    out = []
    for was in (s["states"].double(), s["shifts"].double()):
        new = was.clone()
        for i, a in enumerate(order):
            if a is None:
                new[:, i] = 0
            elif a != i:
                new[:, i] = was[:, a]
        out.append(new)
    return out + [None] * (3 if case["do"] == "compact" else 1)  # whole numbers
