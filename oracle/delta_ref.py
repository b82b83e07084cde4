"""The gated delta rule and the product with an epilogue in 64 bits, from their definitions (test infrastructure only)."""
import math

import numpy as np
from scipy.special import erfc


def gated_delta_ref(q, k, v, g, beta, state=None, scale=None, qk_norm=False, keep=None):
    """One row: q, k (T, Hk, K), v (T, Hv, V), g, beta (T, Hv), state (Hv, K, V) or None, the first `keep` tokens.
    Returns (o (T, Hv, V), the states after 0 .. T tokens (T + 1, Hv, K, V))."""
    q, k, v, g, beta = (np.asarray(x, np.float64) for x in (q, k, v, g, beta))
    (T, Hk, K), (Hv, V) = q.shape, v.shape[1:]
    if qk_norm:
        q = q / np.sqrt((q * q).sum(-1, keepdims=True) + 1e-6)
        k = k / np.sqrt((k * k).sum(-1, keepdims=True) + 1e-6)
    scale = K ** -0.5 if scale is None else scale
    q, k = (np.repeat(x, Hv // Hk, axis=1) for x in (q, k))
    S = np.zeros((Hv, K, V)) if state is None else np.asarray(state, np.float64).copy()
    o, states = np.zeros((T, Hv, V)), [S.copy()]
    for t in range(T if keep is None else max(0, min(T, keep))):
        S = S * np.exp(g[t])[:, None, None]
        d = beta[t][:, None] * (v[t] - np.einsum("hk,hkv->hv", k[t], S))
        S = S + k[t][:, :, None] * d[:, None, :]
        o[t] = scale * np.einsum("hk,hkv->hv", q[t], S)
        states.append(S.copy())
    return o, np.stack(states)


ACTIVATIONS = {
    None: lambda x: x, "none": lambda x: x, "relu": lambda x: np.maximum(x, 0), "relu2": lambda x: np.maximum(x, 0) ** 2,
    "tanh": np.tanh, "sigmoid": lambda x: 1 / (1 + np.exp(-x)), "silu": lambda x: x / (1 + np.exp(-x)),
    "gelu": lambda x: x * erfc(-x / math.sqrt(2)) / 2}


def dense_ref(a, w, bias=None, activation=None, residual=None):
    """(act(a @ w + bias) + residual, a @ w + bias)"""
    x = np.asarray(a, np.float64) @ np.asarray(w, np.float64)
    if bias is not None:
        x = x + np.asarray(bias, np.float64)
    y = ACTIVATIONS[activation](x)
    return (y if residual is None else y + np.asarray(residual, np.float64)), x
