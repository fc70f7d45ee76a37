"""CPU oracle of the decode step's attention operators (test infrastructure
only: imported by tests/, never by the package): per-head RMSNorm and rotation,
the quantised cache's format, and attention over it, from their formulas in
64 bits (the quantiser in the single IEEE fp32 operations that define it).
"""
from __future__ import annotations

import numpy as np

BLOCK = 16


# ---- per-head RMSNorm and rotation ----
def qknorm_rope(x, w, table, positions, eps, interleaved):
    """fp64 [T, H, D] of x [T, H, D], w [D] or None, table [P, R], positions [T]."""
    y = np.asarray(x, np.float64)
    if w is not None:
        y = y / np.sqrt(np.mean(y * y, axis=-1, keepdims=True) + eps) * np.asarray(w, np.float64)
    R = table.shape[1]
    cs = np.asarray(table, np.float64)[positions]
    c, s = cs[:, None, :R // 2], cs[:, None, R // 2:]
    i = np.arange(R // 2)
    a, b = (2 * i, 2 * i + 1) if interleaved else (i, i + R // 2)
    out = y.copy()
    out[..., a] = y[..., a] * c - y[..., b] * s
    out[..., b] = y[..., b] * c + y[..., a] * s
    return out


# ---- the cache ----
def row_bytes(dim, bits):
    return dim * bits // 8


def place(row, j, b):
    """Byte offset of byte b of token j's row inside its 16-row part."""
    chunk = b >> 4
    if row >= 128:
        chunk = chunk ^ (j & 7)
    elif row == 64:
        j, chunk = j ^ ((j >> 1) & 1), chunk ^ ((j >> 2 & 1) << 1)
    else:
        j = j ^ ((j >> 2) & 1)
    return j * row + chunk * 16 + (b & 15)


def quantise(x, bits):
    """x [..., D] -> (q int8, s fp16) with single fp32 operations."""
    top = np.float32(127 if bits == 8 else 7)
    x = np.asarray(x, np.float32)
    amax = np.max(np.where(np.isnan(x), np.float32(0), np.abs(x)), axis=-1)
    with np.errstate(over="ignore"):
        s = np.minimum(amax / top, np.float32(65504)).astype(np.float16)
    s32 = s.astype(np.float32)
    with np.errstate(divide="ignore"):
        inv = np.where(s32 == 0, np.float32(0), np.float32(1) / s32)[..., None]
    with np.errstate(invalid="ignore"):
        y = np.where(np.isnan(x), np.float32(0), x * inv)
        y = np.where(np.isnan(y), np.float32(0), y)  # inf * 0
    return np.clip(np.rint(y), -top, top).astype(np.int8), s


def dequantise(q, s):
    """fp32 values that (q, s) stand for (the product rounds once)."""
    return q.astype(np.float32) * s.astype(np.float32)[..., None]


def pack_rows(q, bits):
    """int8 [..., D] -> uint8 [..., row]."""
    u = q.view(np.uint8)
    if bits == 8:
        return u
    return (u[..., 0::2] & 15) | ((u[..., 1::2] & 15) << 4)


def write(pages, page_size, slots, k, v, bits):
    """Writes tokens into pages (uint8 [P, H, page/16, block bytes]) in place."""
    row = row_bytes(k.shape[-1], bits)
    b = np.arange(row)
    for t, slot in enumerate(slots):
        if slot < 0:
            continue
        page, off = divmod(int(slot), page_size)
        blk, j = divmod(off, BLOCK)
        for part, x in enumerate((k, v)):
            q, s = quantise(x[t], bits)
            pages[page, :, blk, part * BLOCK * row + place(row, j, b)] = pack_rows(q, bits).T
            at = 2 * BLOCK * row + 2 * (part * BLOCK + j)
            pages[page, :, blk, at:at + 2] = s.reshape(-1, 1).view(np.uint8)


# ---- attention ----
def attention(q, k, v, length, scale, window=0, prefix=0):
    """fp64 (out, lse, bound parts) of q [n, Hq, D] over k, v [prefix + length, H, D].

    Row i sees the prefix and its own tokens up to length - n + i (the last
    `window` of them).  Also returns sum_j p_j |v_j| per output element and
    max_j scale sum_d |q_d k_jd| per row, from which tolerances follow."""
    n, Hq, D = q.shape
    H = k.shape[1]
    G = Hq // H
    q = np.asarray(q, np.float64).reshape(n, H, G, D)
    k, v = np.asarray(k, np.float64), np.asarray(v, np.float64)
    out, pv = np.zeros((n, H, G, D)), np.zeros((n, H, G, D))
    lse, mag = np.full((n, H, G), -np.inf), np.zeros((n, H, G))
    for i in range(n):
        end = prefix + max(0, length - n + i + 1)
        lo = max(prefix, prefix + length - n + i + 1 - window) if window else 0
        if end <= lo:
            continue
        s = np.einsum("hgd,nhd->hgn", q[i], k[lo:end]) * scale
        mag[i] = np.max(np.einsum("hgd,nhd->hgn", np.abs(q[i]), np.abs(k[lo:end])), -1) * abs(scale)
        m = s.max(-1, keepdims=True)
        p = np.exp(s - m)
        z = p.sum(-1, keepdims=True)
        lse[i] = (np.log(z) + m)[..., 0]
        p /= z
        out[i] = np.einsum("hgn,nhd->hgd", p, v[lo:end])
        pv[i] = np.einsum("hgn,nhd->hgd", p, np.abs(v[lo:end]))
    shape = (n, Hq, D)
    return out.reshape(shape), lse.reshape(n, Hq), pv.reshape(shape), mag.reshape(n, Hq)


def attention_tolerance(out, pv, mag, vmax, tokens, dim, out_bits):
    """Largest error that the kernel's roundings allow, per output element.

    out_bits: significand bits of the output type (11 or 8).
      * the output rounds once: 2^-out_bits |o|
      * a weight rounds to fp16: 2^-11 p |v|, or below fp16's normal range by
        2^-25 of the largest weight: tokens 2^-25 max|v|
      * a score is dim / 16 tensor-core steps of fp32 sums, each losing at most
        2^-22 of sum |q k|, and a handful of fp32 operations (4 more steps); a
        relative error of a weight moves o by twice itself times sum p |v|
      * the fp32 sums over tokens: 16 tokens a step
    """
    ds = (dim / 16 + 4) * 2.0 ** -22 * (mag[..., None] + 1)
    steps = (tokens / 16 + 64) * 2.0 ** -23
    return (2.0 ** -out_bits * np.abs(out) + 2.0 ** -11 * pv + tokens * 2.0 ** -25 * vmax
            + 2 * (ds + steps) * pv + 1e-30)


def lse_tolerance(lse, mag, tokens, dim):
    """The scores' error, the approximate 2^x and log2 (2^-21 each) and the fp32 sums."""
    with np.errstate(invalid="ignore"):
        rel = np.where(np.isfinite(lse), np.abs(lse), 0)
    return ((dim / 16 + 4) * 2.0 ** -22 * (mag + 1) + 2.0 ** -20 + rel * 2.0 ** -22
            + (tokens / 16 + 64) * 2.0 ** -23)
