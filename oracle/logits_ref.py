"""CPU oracle of the logit operators (include/logits.h) -- TEST INFRASTRUCTURE ONLY.

Plain numpy in 64 bits, row by row, from the definitions:
  * penalize_ref -- penalties for repeated tokens, biases, grammar masks;
  * choices_ref  -- which tokens a row's draw may give when weights are off by a relative `slack`, and its log-probabilities.
"""
from __future__ import annotations

import numpy as np


def penalize_ref(x, counts=None, slots=None, repetition=1.0, presence=0.0, frequency=0.0, drafts=None, bias_ids=None,
                 bias_values=None, mask=None, mask_rows=None):
    """x (B, T, V); arguments as rwkv_next_amd.kernels.penalize_logits takes them, in numpy.  mask (B, T, words) uint32, or a
    table with mask_rows (B, T).  Returns float64."""
    x = np.array(x, np.float64)
    B, T, V = x.shape
    rep, pres, freq = (np.broadcast_to(np.asarray(v, np.float64), (B,)) for v in (repetition, presence, frequency))
    for b in range(B):
        c = np.zeros(V)
        if counts is not None:
            s = b if slots is None else int(slots[b])
            if 0 <= s < counts.shape[0]:
                c = counts[s].astype(np.float64)
        for t in range(T):
            if t and drafts is not None and 0 <= drafts[b, t - 1] < V:
                c[drafts[b, t - 1]] += 1
            for v in np.flatnonzero(c > 0):
                y = x[b, t, v]
                x[b, t, v] = (y / rep[b] if y > 0 else y * rep[b]) - (freq[b] * c[v] + pres[b])
            if bias_ids is not None:
                for i, v in zip(bias_ids[b], bias_values[b]):
                    if 0 <= i < V:
                        x[b, t, i] += float(v)
            if mask is not None:
                row = mask[b, t] if mask_rows is None else (mask[mask_rows[b, t]] if 0 <= mask_rows[b, t] < len(mask)
                                                            else None)
                if row is not None:
                    bits = np.unpackbits(np.ascontiguousarray(row).view(np.uint8), bitorder="little")[:V]
                    x[b, t, bits == 0] = -np.inf
    return x


def choices_ref(x, noise, temperature, top_k, top_p, min_p, slack):
    """One row x (V,): (the tokens that a draw may give when each weight, and so each sum, is off by up to `slack` relatively; a
    float64 array of every token's log-probability).  No tokens where nothing can be chosen."""
    x = np.array(x, np.float64)
    x[np.isnan(x)] = -np.inf
    V = x.size
    if not np.any(x > -np.inf):
        return set(), np.full(V, -np.inf)
    x = np.minimum(x, np.finfo(np.float32).max)
    greedy = noise is None or not temperature > 0
    d = (x.max() - x) / (1.0 if greedy else temperature)
    w = np.exp(-d)
    logprob = -d - np.log(w.sum())
    if greedy:
        return {int(np.argmax(x))}, logprob
    order = np.lexsort((np.arange(V), d))
    order = order[d[order] < np.inf]
    if top_k > 0:
        # places whose d differ by less than the slack may change: every token as near as the last one counts as a candidate
        sure = order[:top_k]
        if len(order) > top_k:
            edge = d[order[top_k - 1]]
            near = np.abs(d[order] - edge) <= slack * max(1.0, edge)
            ties = d[order] == edge
            if not np.array_equal(near, ties):  # not equal values, whose order is exact, but near ones
                maybe, sure = order[(np.arange(len(order)) < top_k) | near], order[:top_k][~near[:top_k]]
            else:
                maybe = sure
        else:
            maybe = sure
    else:
        sure = maybe = order
    def prefix(tokens, p):
        if top_p >= 1 or len(tokens) == 0:
            return tokens
        sums = np.cumsum(w[tokens])
        return tokens[:1 + int(np.searchsorted(sums, p * sums[-1], side="left"))]
    few = prefix(sure, top_p * (1 - slack))
    many = prefix(maybe, top_p * (1 + slack))
    few = few[w[few] >= min(min_p, 1.0) * (1 + slack)]
    many = many[w[many] >= min(min_p, 1.0) * (1 - slack)]
    top = int(order[0])
    few, many = set(few.tolist()) | {top}, set(many.tolist()) | {top}
    # noise that is no number draws nothing, and without any the most likely token is taken
    e = np.asarray(noise, np.float64)
    with np.errstate(divide="ignore", invalid="ignore"):
        score = np.where(np.isnan(e), -1.0, w / e)
    best = max((score[i] for i in few), default=-1.0)
    if best < 0:
        return {top}, logprob
    return {i for i in many if score[i] >= best * (1 - 4 * slack)}, logprob
