"""What the operators between the last hidden state and the next token are measured on.

Three operators of a decode step's end, each through the package's public entry points (`own` true) or in its plain form:

    int4      a product of a few rows of activations with a 4-bit weight, one fp16 scale for each group of rows and column:
              the output head, or a layer's projections
    penalize  penalties for tokens that a sequence already holds, per-request biases and grammar masks, on the logits of
              one token per sequence or of a block of drafted tokens
    sample    the choice of the token: temperature, top-k, top-p, min-p, and a draw by given exponential noise

The vocabulary of 65536 and the widths 768, 2560 and 4096 are RWKV-7's; the others are generic.
"""
import math
import os
import sys

import numpy as np
import torch

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "rwkv-infer-next_amd"))

own = False

DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


# ----------------------------------------------------------------------------------------------------------------
# the cases
# ----------------------------------------------------------------------------------------------------------------
def listed():
    return [
        # one user's decode step, a square projection of the 7.2B shape: latency
        dict(name="int4_m1_4096x4096", op="int4", M=1, K=4096, N=4096, group=128, dtype="bf16", out="bf16"),
        # a small odd batch on the 2.9B shape's wide projection, fp16 activations, fine groups
        dict(name="int4_m5_2560x10240_f16", op="int4", M=5, K=2560, N=10240, group=64, dtype="f16", out="f16"),
        # the output head for one user: the largest weight of the model read for one row
        dict(name="int4_head_m1", op="int4", M=1, K=4096, N=65536, group=128, dtype="bf16", out="f32"),
        # the output head for the serving batch
        dict(name="int4_head_m64", op="int4", M=64, K=4096, N=65536, group=128, dtype="bf16", out="bf16"),
        # the output head over a block of drafted tokens of many sequences, of an odd size, on a vocabulary shard
        dict(name="int4_m203_2560x8191", op="int4", M=203, K=2560, N=8191, group=32, dtype="bf16", out="f32"),
        # one user's logits with every penalty
        dict(name="penalize_b1", op="penalize", B=1, T=1, V=65536, dtype="f32", slots=8, bias=4, masked=True),
        # the serving batch's logits as the head leaves them
        dict(name="penalize_b64", op="penalize", B=64, T=1, V=65536, dtype="bf16", slots=128, bias=32, masked=False),
        # speculative decoding under a grammar: five positions of each sequence, each sees the drafts before it
        dict(name="penalize_b64_t5", op="penalize", B=64, T=5, V=65536, dtype="f32", slots=128, bias=32, masked=True),
        # one user, the usual nucleus
        dict(name="sample_b1", op="sample", B=1, T=1, V=65536, dtype="f32", top_k=0, top_p=0.9, min_p=0.0, greedy=False,
             masked=False),
        # the serving batch, every filter, some requests greedy
        dict(name="sample_b64", op="sample", B=64, T=1, V=65536, dtype="f32", top_k=50, top_p=0.9, min_p=0.02, greedy=True,
             masked=False),
        # an odd vocabulary and no filter: every token may be drawn
        dict(name="sample_b23_v50001", op="sample", B=23, T=1, V=50001, dtype="bf16", top_k=0, top_p=1.0, min_p=0.0,
             greedy=False, masked=False),
        # the positions of a speculative step under a grammar, a wide nucleus
        dict(name="sample_b64_t5", op="sample", B=64, T=5, V=65536, dtype="bf16", top_k=0, top_p=0.95, min_p=0.0,
             greedy=True, masked=True),
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("int4", "penalize", "sample"))
    if op == "int4":
        group = rng.choice((32, 64, 128))
        K = rng.choice((768, 2560, 4096, 10240, 16384, group * _log_int(rng, 1, 8192 // group)))
        while K % group or K == 3 * 1024:
            K = group * _log_int(rng, 1, 8192 // group)
        N = rng.choice((_log_int(rng, 16, 65536), 16 * _log_int(rng, 1, 4096), 4096, 65536))
        N = min(N, 4096 * 65536 // K)
        N += N == 3 * 1024
        M = min(_log_int(rng, 1, 256), max(1, 64 * 4096 * 65536 // (K * N)))
        return dict(op=op, M=M, K=K, N=N, group=group, dtype=rng.choice(("bf16", "f16")),
                    out=rng.choice(("bf16", "f16", "f32")))
    B, T = _log_int(rng, 1, 64), rng.choice((1, 1, rng.randint(2, 5)))
    V = rng.choice((65536, _log_int(rng, 1000, 65536), _log_int(rng, 1000, 131072)))
    V = min(V, 64 * 65536 // B)
    V += V == 3 * 1024
    dtype = rng.choice(("f32", "bf16", "f16"))
    if op == "penalize":
        return dict(op=op, B=B, T=T, V=V, dtype=dtype, slots=B + rng.randint(0, 64), bias=rng.choice((0, 1, 32, 300)),
                    masked=rng.random() < 0.5)
    return dict(op=op, B=B, T=T, V=V, dtype=dtype, top_k=rng.choice((0, 0, 1, 40, 50, 500)),
                top_p=rng.choice((1.0, 0.5, 0.9, 0.95)), min_p=rng.choice((0.0, 0.0, 0.02, 0.1)),
                greedy=rng.random() < 0.3, masked=rng.random() < 0.3)


# ----------------------------------------------------------------------------------------------------------------
# what a program has in hand
# ----------------------------------------------------------------------------------------------------------------
def _int4_inputs(case, gen, dev):
    K, N, G = case["K"], case["N"], case["K"] // case["group"]
    return dict(
        a=torch.randn(case["M"], K, device=dev, generator=gen).to(DTYPES[case["dtype"]]),
        # two codes to a byte, rows 2j (low) and 2j + 1, and scales that make weights of a trained layer's size
        codes=torch.randint(0, 256, (K // 2, N), device=dev, dtype=torch.uint8, generator=gen),
        scales=((torch.rand(G, N, device=dev, generator=gen) + 0.5) * (0.25 / math.sqrt(K))).half())


def _logits(case, gen, dev):
    """Logits of a language model: a broad bulk, and a few dozen tokens that stand out of it."""
    B, T, V = case["B"], case["T"], case["V"]
    x = torch.randn(B, T, V, device=dev, generator=gen) * 2
    at = torch.randint(0, V, (B, T, 48), device=dev, generator=gen)
    up = 14 - 1.5 * torch.rand(B, T, 48, device=dev, generator=gen).log().neg().clamp_max(6.0)
    up = up + torch.rand(B, T, 48, device=dev, generator=gen)
    return x.scatter_reduce_(2, at, up, "amax")  # the same whatever the order of equal places


def _penalize_inputs(case, gen, dev):
    B, T, V, S, P = case["B"], case["T"], case["V"], case["slots"], case["bias"]
    s = dict(logits=_logits(case, gen, dev).to(DTYPES[case["dtype"]]))
    # a sequence holds some hundred different tokens, some many times
    counts = torch.zeros(S, V, device=dev, dtype=torch.int32)
    held = (torch.rand(S, 600, device=dev, generator=gen).square() * (V - 1)).long()
    s["counts"] = counts.scatter_add_(1, held, torch.ones_like(held, dtype=torch.int32))
    s["slots"] = torch.randperm(S, device=dev, generator=gen)[:B]
    s["repetition"] = 1 + torch.rand(B, device=dev, generator=gen) * 0.3
    s["presence"] = torch.rand(B, device=dev, generator=gen) * 0.5
    s["frequency"] = torch.rand(B, device=dev, generator=gen) * 0.5
    if T > 1:
        s["drafts"] = (torch.rand(B, T - 1, device=dev, generator=gen).square() * (V - 1)).long()
    if P:  # distinct ids, the end of some rows unused (-1)
        ids = torch.rand(B, V, device=dev, generator=gen).topk(P, dim=1).indices
        ids[torch.rand(B, P, device=dev, generator=gen) < 0.25] = -1
        s["bias_ids"], s["bias_values"] = ids, torch.randn(B, P, device=dev, generator=gen) * 3
    if case["masked"]:
        words = (V + 31) // 32
        m = torch.randint(-2 ** 31, 2 ** 31, (2, B, T, words), device=dev, generator=gen)
        s["mask"] = (m[0] | m[1]).to(torch.int32)
    return s


def _sample_inputs(case, gen, dev):
    B, T, V = case["B"], case["T"], case["V"]
    x = _logits(case, gen, dev)
    if case["masked"]:  # tokens that a grammar does not allow
        x.masked_fill_(torch.rand(B, T, V, device=dev, generator=gen) < 0.6, float("-inf"))
    s = dict(logits=x.to(DTYPES[case["dtype"]]))
    s["noise"] = torch.empty(B, T, V, device=dev).exponential_(generator=gen)
    s["temperature"] = 0.6 + torch.rand(B, device=dev, generator=gen)
    if case["greedy"]:
        s["temperature"][torch.rand(B, device=dev, generator=gen) < 0.25] = 0.0
    # requests differ: half of them ask for the case's filter, the others for one near it
    near = torch.randint(0, 2, (B,), device=dev, generator=gen)
    s["top_k"] = torch.full((B,), case["top_k"], device=dev, dtype=torch.int32) + (near * (case["top_k"] > 1)).int()
    s["top_p"] = torch.full((B,), case["top_p"], device=dev) - near * (0.05 if case["top_p"] < 1 else 0.0)
    s["min_p"] = torch.full((B,), case["min_p"], device=dev) * (1 + near)
    return s


def prepare(case, seed):
    dev = torch.device("cuda")
    gen = torch.Generator(device=dev).manual_seed(seed)
    inputs = {"int4": _int4_inputs, "penalize": _penalize_inputs, "sample": _sample_inputs}[case["op"]]
    s = dict(inputs(case, gen, dev), case=dict(case))
    if own:
        from rwkv_next_amd import kernels
        s["kernels"] = kernels
        if case["op"] == "int4":  # laid out once, when the weights are loaded
            s["weight"] = kernels.prepack_int4(s["codes"], s["scales"], case["group"])
    return s


# ----------------------------------------------------------------------------------------------------------------
# one pass
# ----------------------------------------------------------------------------------------------------------------
def run(state):
    op = state["case"]["op"]
    if own:
        return {"int4": _int4_own, "penalize": _penalize_own, "sample": _sample_own}[op](state)
    return {"int4": _int4_plain, "penalize": _penalize_plain, "sample": _sample_plain}[op](state)


def _int4_own(s):
    return s["kernels"].int4_matmul(s["a"], s["weight"], out_dtype=DTYPES[s["case"]["out"]])


def _penalize_own(s):
    return s["kernels"].penalize_logits(
        s["logits"], counts=s["counts"], slots=s["slots"], repetition=s["repetition"], presence=s["presence"],
        frequency=s["frequency"], drafts=s.get("drafts"), bias_ids=s.get("bias_ids"),
        bias_values=s.get("bias_values"), mask=s.get("mask"))


def _sample_own(s):
    return s["kernels"].sample_logits(s["logits"], s["noise"], temperature=s["temperature"], top_k=s["top_k"],
                                      top_p=s["top_p"], min_p=s["min_p"])


def _int4_plain(s):
    case = s["case"]
    K, N, g = case["K"], case["N"], case["group"]
    q = torch.stack((s["codes"] & 15, s["codes"] >> 4), dim=1).view(K // g, g, N).float() - 8
    w = (q * s["scales"].float()[:, None, :]).view(K, N)
    return (s["a"].float() @ w).to(DTYPES[case["out"]])


def _penalize_plain(s):
    x = s["logits"].float()
    B, T, V = x.shape
    c = s["counts"][s["slots"]].float()[:, None, :].expand(B, T, V)
    if "drafts" in s:  # position t has the drafts before it
        seen = torch.arange(T - 1, device=x.device)[None, :] < torch.arange(T, device=x.device)[:, None]
        at = s["drafts"][:, None, :].expand(B, T, T - 1)
        c = c + torch.zeros_like(x).scatter_add_(2, at, seen.float()[None].expand(B, T, T - 1))
    rep, pres, freq = (s[n][:, None, None] for n in ("repetition", "presence", "frequency"))
    x = torch.where(c > 0, torch.where(x > 0, x / rep, x * rep) - (freq * c + pres), x)
    if "bias_ids" in s:
        used = s["bias_ids"] >= 0
        bias = torch.zeros(B, V, device=x.device)
        x = x + bias.scatter_add_(1, s["bias_ids"].clamp_min(0), s["bias_values"] * used)[:, None, :]
    if "mask" in s:
        bits = (s["mask"][..., None] >> torch.arange(32, device=x.device, dtype=torch.int32)) & 1
        x = torch.where(bits.view(B, T, -1)[..., :V] != 0, x, float("-inf"))
    return x.to(s["logits"].dtype)


def _sample_plain(s):
    x = s["logits"].float()
    V = x.shape[-1]
    temperature, top_k, top_p, min_p = (s[n][:, None, None] for n in ("temperature", "top_k", "top_p", "min_p"))
    greedy = temperature <= 0
    d = (x.amax(dim=2, keepdim=True) - x) * (1 / torch.where(greedy, 1.0, temperature))
    w = torch.exp(-d)
    total = w.sum(dim=2, keepdim=True)
    ds, order = d.sort(dim=2, stable=True)  # most likely first, equal ones by their index
    ws = torch.exp(-ds)
    place = torch.arange(V, device=x.device)
    ws = torch.where((place < top_k) | (top_k <= 0), ws, 0.0)
    before = ws.cumsum(dim=2) - ws
    keep = ((before < top_p * ws.sum(dim=2, keepdim=True)) | (top_p >= 1)) & (ws >= min_p) & (ws > 0)
    keep = (keep & ~greedy) | (place == 0)
    score = torch.where(keep, ws / s["noise"].gather(2, order), -1.0)
    best = score.argmax(dim=2, keepdim=True)
    logprob = -ds.gather(2, best) - total.log()
    return order.gather(2, best)[..., 0], logprob[..., 0]


# ----------------------------------------------------------------------------------------------------------------
# what a pass has to do, and its results in 64 bits
# ----------------------------------------------------------------------------------------------------------------
def work(case):
    size = {n: t.itemsize for n, t in DTYPES.items()}
    if case["op"] == "int4":
        M, K, N = case["M"], case["K"], case["N"]
        return {"bytes": K * N // 2 + 2 * (K // case["group"]) * N + 2 * M * K + size[case["out"]] * M * N,
                "flops": 2 * M * K * N}
    B, T, V, e = case["B"], case["T"], case["V"], size[case["dtype"]]
    if case["op"] == "penalize":
        return {"bytes": 2 * B * T * V * e + 4 * B * V + (B * T * ((V + 31) // 32) * 4 if case["masked"] else 0)
                + 12 * B * case["bias"], "flops": 8 * B * T * V}
    # of the noise only what belongs to tokens that may be drawn: all of it where nothing is filtered
    every = case["top_k"] == 0 and case["top_p"] >= 1 and case["min_p"] == 0
    return {"bytes": B * T * V * (e + (4 if every else 0)) + 12 * B * T, "flops": 5 * B * T * V}


def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return {"int4": _int4_exact, "penalize": _penalize_exact, "sample": _sample_exact}[case["op"]](case, s)


def _int4_exact(case, s):
    K, N, g = case["K"], case["N"], case["group"]
    a, y = s["a"].double(), torch.empty(case["M"], N, device=s["a"].device, dtype=torch.float64)
    rows = torch.arange(K, device=a.device)
    for n0 in range(0, N, 4096):
        byte = s["codes"][:, n0:n0 + 4096][rows // 2].int()
        u = torch.where((rows % 2 == 0)[:, None], byte % 16, byte // 16)
        y[:, n0:n0 + 4096] = a @ ((u - 8).double() * s["scales"][:, n0:n0 + 4096][rows // g].double())
    return y


def _penalize_exact(case, s):
    B, T, V = case["B"], case["T"], case["V"]
    x = s["logits"].double().cpu().numpy().copy()
    h = {n: s[n].cpu().numpy() for n in s if isinstance(s[n], torch.Tensor) and n != "logits"}
    for b in range(B):
        rep, pres, freq = (float(h[n][b]) for n in ("repetition", "presence", "frequency"))
        c = h["counts"][h["slots"][b]].astype(np.float64)
        for t in range(T):
            if t:
                c[h["drafts"][b, t - 1]] += 1
            row, at = x[b, t], np.flatnonzero(c)
            v = row[at]
            row[at] = np.where(v > 0, v / rep, v * rep) - freq * c[at] - pres
            if "bias_ids" in h:
                ok = h["bias_ids"][b] >= 0
                np.add.at(row, h["bias_ids"][b][ok], h["bias_values"][b][ok].astype(np.float64))
            if "mask" in h:
                bits = np.unpackbits(h["mask"][b, t].view(np.uint8), bitorder="little")[:V]
                row[bits == 0] = -np.inf
    return torch.from_numpy(x)


def _sample_exact(case, s):
    B, T = case["B"], case["T"]
    x = s["logits"].double().cpu().numpy()
    h = {n: s[n].cpu().numpy() for n in ("noise", "temperature", "top_k", "top_p", "min_p")}
    token, logprob = np.zeros((B, T), np.int64), np.zeros((B, T))
    for b in range(B):
        temp, k, top_p, min_p = (float(h[n][b]) for n in ("temperature", "top_k", "top_p", "min_p"))
        for t in range(T):
            z = x[b, t] / (temp if temp > 0 else 1.0)
            z = z - z.max()
            w = np.exp(z)
            if temp > 0:
                kept = np.lexsort((np.arange(z.size), -z))[:int(k) if k > 0 else None]
                run_up = np.cumsum(w[kept])
                if top_p < 1:
                    kept = kept[:1 + int(np.searchsorted(run_up, top_p * run_up[-1], side="left"))]
                kept = np.sort(kept[w[kept] >= min(min_p, 1.0)])
                token[b, t] = kept[np.argmax(w[kept] / h["noise"][b, t, kept].astype(np.float64))]
            else:
                token[b, t] = int(np.argmax(x[b, t]))
            logprob[b, t] = z[token[b, t]] - math.log(w.sum())
    return torch.from_numpy(token), torch.from_numpy(logprob)
