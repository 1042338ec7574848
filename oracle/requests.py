"""What each request of a served batch brings of its own, in 64 bits and more:
low-rank adapters beside a shared projection, and sampling from logits by given
random numbers.  Definitions of this library (the reference merges one adapter into
a linear and leaves sampling to HF); plain loops, no shared code with the kernels."""

import numpy as np


def multi_lora_ref(y, x, lora_A, lora_B, adapters, scales, splits=None):
    """(out, bound): ``y + scales[a] (x A[a]) B[a]`` in 64 bits, and ``sum |terms|`` of
    every output, the number its rounding errors are relative to.  ``y`` ``[B, (T,) N]``."""
    y, x, lora_A, lora_B = (np.asarray(t, np.float64) for t in (y, x, lora_A, lora_B))
    n, r, N = lora_B.shape
    splits = [N] if splits is None else list(splits)
    out, bound = y.copy(), np.abs(y)
    for b, a in enumerate(adapters):
        if not 0 <= a < n:
            continue
        at = 0
        for j, width in enumerate(splits):
            A, B = lora_A[a][:, j * r:(j + 1) * r], lora_B[a][:, at:at + width]
            s = float(scales[a])
            out[b][..., at:at + width] += s * (x[b] @ A @ B)
            bound[b][..., at:at + width] += abs(s) * (np.abs(x[b]) @ np.abs(A) @ np.abs(B))
            at += width
    return out, bound


def sample_ref(logits, u, temperature, top_k, top_p, min_p):
    """(tokens int64, logprobs float64) of fp16 ``logits`` ``[B, V]``; the settings are
    ``[B]`` as the library holds them (fp32, ``top_k`` int64)."""
    tokens, logprobs = [], []
    for row, uu, t, k, p, m in zip(np.asarray(logits), u, temperature, top_k, top_p, min_p):
        l = row.astype(np.longdouble)
        alive = np.flatnonzero(~(np.isnan(l) | np.isneginf(l)))
        if alive.size == 0:
            tokens.append(-1)
            logprobs.append(-np.inf)
            continue
        order = alive[np.lexsort((alive, -l[alive]))]
        l = l[order]
        greedy = not t > 0
        with np.errstate(all="ignore"):
            away = np.where(l == l[0], 0, l - l[0])
            w = np.where(l == l[0], 1, np.where(np.isneginf(away), 0, np.exp(away / np.longdouble(1 if greedy else t))))
        if greedy:
            w = w[:1]
        elif k > 0:
            w = w[: int(k)]
        if not greedy and p < 1:
            running = np.cumsum(w)
            want = np.longdouble(max(float(p), 0.0)) * running[-1]
            w = w[: 1 + int(np.searchsorted(running, want, side="left"))] if want > 0 else w[:1]
        if not greedy and m > 0:
            w = w[w >= min(np.longdouble(m), 1)]
        running = np.cumsum(w)
        want = np.longdouble(uu) * running[-1] if uu > 0 else np.longdouble(0)
        at = int(np.searchsorted(running, want, side="right"))
        at = min(at, int(np.flatnonzero(w > 0)[-1]))
        tokens.append(int(order[at]))
        logprobs.append(float(np.log(w[at]) - np.log(running[-1])))
    return np.array(tokens), np.array(logprobs)
