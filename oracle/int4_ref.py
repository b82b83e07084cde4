"""CPU oracle for the 4-bit weight format and product (include/w4a16.h) -- TEST INFRASTRUCTURE ONLY.

Plain numpy: pack_codes / unpack_codes (two codes u = q + 8 to a byte), dequantize_ref and int4_matmul_ref in 64 bits, and the
kernel's order of the same bits, restated from its definition (packed_ref, packed_scales_ref).
"""
from __future__ import annotations

import numpy as np


def pack_codes(u):
    """u uint8 (K, N) in [0, 15] -> (K/2, N): row 2j in the low bits, row 2j + 1 in the high ones."""
    u = np.asarray(u, np.uint8)
    return u[0::2] | (u[1::2] << 4)


def unpack_codes(codes):
    u = np.empty((2 * codes.shape[0], codes.shape[1]), np.uint8)
    u[0::2], u[1::2] = codes & 15, codes >> 4
    return u


def dequantize_ref(codes, scales, group_k):
    q = unpack_codes(codes).astype(np.float64) - 8
    return q * np.asarray(scales, np.float16).astype(np.float64)[np.arange(q.shape[0]) // group_k]


def int4_matmul_ref(a, codes, scales, group_k):
    return np.asarray(a, np.float64) @ dequantize_ref(codes, scales, group_k)


def packed_ref(codes):
    """Words (strip, chunk, lane, step): lane l has column l % 16 of the strip, and of step k of the chunk the rows
    32 k + 8 (l // 16) + 0..7: row 2j in bits 4j.., row 2j + 1 in bits 16 + 4j..; code 8 past the weight."""
    u = unpack_codes(codes)
    K, N = u.shape
    S, C = -(-N // 16), -(-K // 128)
    full = np.full((C * 128, S * 16), 8, np.uint32)
    full[:K, :N] = u
    t = full.reshape(C, 4, 4, 4, 2, S, 16)      # chunk, step, lane // 16, j, odd, strip, column
    w = np.zeros((C, 4, 4, S, 16), np.uint32)
    for j in range(4):
        w |= t[:, :, :, j, 0] << np.uint32(4 * j)
        w |= t[:, :, :, j, 1] << np.uint32(16 + 4 * j)
    return np.ascontiguousarray(w.transpose(3, 0, 2, 4, 1)).reshape(S, C, 64, 4)


def packed_scales_ref(scales, K, group_k):
    """(strip, chunk, column, part): one scale where a group holds whole chunks of 128 rows, two or four of its parts else."""
    parts = 1 if group_k % 128 == 0 else 2 if group_k % 64 == 0 else 4
    N = scales.shape[1]
    S, C = -(-N // 16), -(-K // 128)
    out = np.zeros((S, C, 16, parts), np.float16)
    for c in range(C):
        for j in range(parts):
            row = 128 * c + j * (128 // parts)
            if row < K:
                line = np.zeros(S * 16, np.float16)
                line[:N] = scales[row // group_k]
                out[:, c, :, j] = line.reshape(S, 16)
    return out
