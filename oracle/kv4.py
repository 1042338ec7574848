"""Oracle of the 4-bit ring KV cache, its attention and the head norm with
rotation, in 64 bits.  Test infrastructure only.

Parity unpinned: the reference has neither a quantised cache nor an attention
kernel; the quantiser restates the format's definition (``include/qx_b200.h``),
the attention is the plain softmax formula.
"""

from __future__ import annotations

import numpy as np

__all__ = ["kv4_values", "attention64", "head_norm_rope64"]

F16_MAX = 65504.0


def kv4_values(x: np.ndarray, group: int) -> np.ndarray:
    """What fp16 ``x`` ``[..., D]`` becomes in the cache (float64, each value a
    fp16 number): per group s = the smallest fp16 number of 7 significant bits
    >= (max(x, 0) - min(x, 0)) / 15, z = rint(-min(x, 0) / s), c = rint(x / s) + z
    within 0..15 and with |s (c - z)| <= 65504; a group with a NaN or an infinity
    is NaN."""
    g = x.astype(np.float64).reshape(x.shape[:-1] + (x.shape[-1] // group, group))
    fine = np.isfinite(g).all(-1, keepdims=True)
    g = np.where(fine, g, 0.0)
    lo = np.minimum(g.min(-1, keepdims=True), 0.0)
    hi = np.maximum(g.max(-1, keepdims=True), 0.0)
    least = (hi - lo) / 15
    # unit of a 7-bit number of that size, none below 2^-20 (fp16's subnormals without their four low bits)
    _, e = np.frexp(least)
    unit = np.ldexp(1.0, np.maximum(e - 7, -20))
    s = np.ceil(least / unit) * unit
    some = np.where(s > 0, s, 1.0)
    z = np.rint(-lo / some)
    k = np.clip(np.rint(g / some) + z, 0, 15) - z
    k = np.where(np.abs(k * s) > F16_MAX, k - np.sign(k), k)
    return np.where(fine, k * s, np.nan).reshape(x.shape)


def attention64(q, k, v, seen, scale: float | None = None):
    """``q`` ``[n, Hq, D]``, ``k`` / ``v`` ``[L, Hkv, D]``, ``seen`` bool ``[n, L]``.
    Returns the output ``[n, Hq, D]``, and per element the sum of weight times
    |v| and per (row, head) the largest sum of |q| |k| over the seen keys: what
    the tolerances are made of.  Hidden keys do not enter, whatever they hold; a
    row that sees none is zero."""
    n, hq, d = q.shape
    rep = hq // k.shape[1]
    scale = 1.0 / np.sqrt(d) if scale is None else scale
    out, weight, size = np.zeros((n, hq, d)), np.zeros((n, hq, d)), np.zeros((n, hq))
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    groups = {}
    for r in range(n):  # rows that see the same keys are done together
        groups.setdefault(seen[r].tobytes(), []).append(r)
    with np.errstate(invalid="ignore", over="ignore"):
        for rows in groups.values():
            at = np.flatnonzero(seen[rows[0]])
            if at.size == 0:
                continue
            for h in range(hq):
                kk, vv, qq = k[at, h // rep], v[at, h // rep], q[rows, h]
                s = qq @ kk.T * scale
                p = np.exp(s - s.max(-1, keepdims=True))
                p /= p.sum(-1, keepdims=True)
                out[rows, h] = p @ vv
                weight[rows, h] = p @ np.abs(vv)
                size[rows, h] = (np.abs(qq) @ np.abs(kk).T).max(-1) * scale
    return out, weight, size


def head_norm_rope64(qkv, q_heads: int, kv_heads: int, q_norm, k_norm, eps: float, cos, sin):
    """``qkv`` ``[B, T, (Hq + 2 Hkv) D]``, ``cos`` / ``sin`` ``[T, D]`` or ``[B, T, D]``:
    (q, k, v) in 64 bits, no rounding in between."""
    d = q_norm.shape[0]
    B, T = qkv.shape[:2]
    x = qkv.astype(np.float64).reshape(B, T, -1, d)
    w = np.concatenate([np.tile(q_norm, (q_heads, 1)), np.tile(k_norm, (kv_heads, 1))]).astype(np.float64)
    y = x[:, :, :q_heads + kv_heads]
    y = y / np.sqrt((y ** 2).mean(-1, keepdims=True) + eps) * w
    rot = np.concatenate([-y[..., d // 2:], y[..., :d // 2]], -1)
    cos, sin = (np.broadcast_to(t.astype(np.float64), (B, T, d))[:, :, None] for t in (cos, sin))
    y = y * cos + rot * sin
    return y[:, :, :q_heads], y[:, :, q_heads:], x[:, :, q_heads + kv_heads:]
