"""Attention over the 4-bit ring where keys or values are NaN or infinite, against the
softmax formula in 64 bits over the keys a row sees: NaN and infinities exactly where the
formula has them, every other element within a finite bound.

Bound of an element, from the roundings, per (row, head) and over the finite values
alone: the result once to fp16 (2^-11 of it, 2^-25 at fp16's end); every weight
once to fp16 (2^-11 of the sum of weight x |v|, and 2^-35 of the largest |v| a key for
its subnormals); a score's fp32 sum of D products, and the scale, D + 8 steps of at
most 2^-24 of the sum of |q| |k|, a weight by the factor exp of twice that; exp2's
2^-21; the fp32 sums over the keys of a row done again one key after the other, 2^-24
a key for the values' and for the weights'."""

import numpy as np
import pytest
import torch

from oracle import kv4_values, ring_positions
from qextract_infer_b200 import _lib
from tests._util import dev_tensor, to_np

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


@pytest.fixture(autouse=True)
def no_wait_ran_out(C):
    C.device_error()
    yield
    C.check_device_error("4-bit ring attention")


def _formula(q, k, v, seen):
    """``q`` ``[n, Hq, D]``, ``k`` / ``v`` ``[L, Hkv, D]``, ``seen`` ``[n, L]``: the output and its bound."""
    n, hq, d = q.shape
    rep, scale = hq // k.shape[1], 1 / np.sqrt(d)
    out, bound = np.zeros((n, hq, d)), np.zeros((n, hq, d))
    q, k, v = (t.astype(np.float64) for t in (q, k, v))
    with np.errstate(invalid="ignore", over="ignore"):
        for r in range(n):
            kr, vr = k[seen[r]], v[seen[r]]
            for h in range(hq):
                kk, vv, qq = kr[:, h // rep], vr[:, h // rep], q[r, h]
                s = kk @ qq * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[r, h] = w @ vv
                usable = np.isfinite(s)  # a score of minus infinity has weight 0 exactly
                size = (np.abs(kk[usable]) @ np.abs(qq)).max(initial=0.0) * scale
                mag = np.where(np.isfinite(vv), np.abs(vv), 0.0)
                sums = len(s) * 2.0 ** -23
                bound[r, h] = (np.abs(out[r, h]) * 2.0 ** -11 + 2.0 ** -25 + len(s) * 2.0 ** -35 * mag.max() +
                               np.nan_to_num(w) @ mag *
                               (2.0 ** -11 + np.expm1(2 * size * (d + 8) * 2.0 ** -24) + 2.0 ** -21 + sums))
    return out, bound


def _run(C, q, k, v, old, counts, S, W, group):
    """The op and the formula on a ring that holds, of ``old`` = (K, V) ``[B, positions, Hkv, D]``, what is not evicted."""
    B, n, Hq, D = q.shape
    Hkv = k.shape[2]
    codes, params = C.ring_q4_storage(B, Hkv, D, S, W, group)
    codes.fill_(0xFF)
    params.fill_(0x7E0F)  # free slots read as NaN
    refs = []
    for b, count in enumerate(counts):
        slots, pos = ring_positions(int(count), S, W)
        one = C.ring_q4_storage(1, Hkv, D, S, W, group)
        for lo, hi in ((0, min(count, S)), (max(S, count - W), count)):
            if hi > lo:
                C.ring_append_q4(*(dev_tensor(t[b:b + 1, lo:hi]) for t in old), *one, int(lo), S, W)
        at = torch.from_numpy(slots).cuda()
        codes[:, b, :, at], params[:, b, :, at] = one[0][:, 0, :, at], one[1][:, 0, :, at]
        kp = np.concatenate([pos, count + np.arange(n)])
        mine = count + np.arange(n)[:, None]
        seen = (kp <= mine) & ((kp < S) | (kp > mine - W))
        kk, vv = (np.concatenate([kv4_values(o[b, pos], group), x[b].astype(np.float64)]) for o, x in zip(old, (k, v)))
        refs.append(_formula(q[b], kk, vv, seen))
    arg = int(counts[0]) if B == 1 else dev_tensor(np.asarray(counts, np.int64))
    out = C.prefill_attention_q4(dev_tensor(q), dev_tensor(k), dev_tensor(v), codes, params, arg, S, W)
    return to_np(out).astype(np.float64), refs


def _same(got, ref, msg=""):
    out, bound = ref
    wrong = np.argwhere(np.isnan(got) != np.isnan(out))
    assert not len(wrong), f"{msg}: NaN where the formula has none, or the reverse: {len(wrong)}, first {wrong[0]}"
    inf = np.isinf(out)
    assert np.array_equal(got[inf], out[inf]) and not np.isinf(got[~inf]).any(), msg
    fine = np.isfinite(out)
    assert np.isfinite(bound[fine]).all()
    off = np.abs(got[fine] - out[fine]) - bound[fine]
    assert (off <= 0).all(), (msg, int((off > 0).sum()), np.argwhere(fine)[off.argmax()], off.max(), bound[fine][off.argmax()])


def _is_split(C, B, n, Hq, Hkv, D, S, W):
    return _lib.load().qx_prefill_attention_q4_workspace_size(B, n, Hq, Hkv, D, S, W) > 0


def _normal(rng, *shape):
    return rng.standard_normal(shape).astype(np.float16)


@pytest.mark.parametrize("D,group", [(128, 64), (128, 32), (64, 32)])
@pytest.mark.parametrize("n,W,count,ring_nan,chunk_nan", [
    (33, 4092, 5000, [1], []),            # a sink: alone in its split
    (33, 4092, 4096, [700, 800, 900, 1000], []),  # a token in each of the neighbouring tiles
    (20, 4092, 3, [], [0]),               # the chunk's first key: no row is without it
    (300, 4092, 0, [], [150]),            # rows from the 150th on
    (40, 60, 64, [4], [30]),              # evicted for all rows; the other seen by the last ten
])
def test_a_key_that_is_nan_makes_every_row_that_sees_it_nan(C, D, group, n, W, count, ring_nan, chunk_nan):
    """Whichever split its tile falls to."""
    rng = np.random.default_rng(n + count)
    S, Hq, Hkv = 4, 4, 2
    assert _is_split(C, 1, n, Hq, Hkv, D, S, W) == (W > 100)
    q, k, v = _normal(rng, 1, n, Hq, D), _normal(rng, 1, n, Hkv, D), _normal(rng, 1, n, Hkv, D)
    old = _normal(rng, 1, count, Hkv, D), _normal(rng, 1, count, Hkv, D)
    old[0][0, ring_nan, 1, 5] = np.nan
    k[0, chunk_nan, 1, 5] = np.nan
    out, refs = _run(C, q, k, v, old, [count], S, W, group)
    _same(out[0], refs[0])


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("B,n,Hq,Hkv,S,W,counts,split", [
    (2, 60, 6, 2, 4, 100, [30, 400], False),
    (1, 100, 2, 1, 0, 70, [72], False),          # the ring starts at slot 2, its tile goes on behind slot 69
    (10, 130, 8, 8, 3, 400, [0, 2, 3, 4, 100, 402, 403, 404, 700, 1999], False),  # enough row blocks to fill the GPU
    (2, 150, 4, 2, 4, 100, [30, 400], True),
    (1, 90, 7, 1, 0, 1000, [2500], True),
    (1, 33, 8, 2, 4, 4092, [5000], True),
])
def test_rows_that_hidden_values_reached_equal_the_formula(C, D, group, B, n, Hq, Hkv, S, W, counts, split):
    """Values of the chunk's later keys and of the ring's oldest tokens that are not finite share a tile with keys that a
    row sees: the row is done again over its own keys, where the tiles are split and where they are not."""
    assert _is_split(C, B, n, Hq, Hkv, D, S, W) == split
    rng = np.random.default_rng(n + D + group)
    q, k, v = _normal(rng, B, n, Hq, D), _normal(rng, B, n, Hkv, D), _normal(rng, B, n, Hkv, D)
    old = _normal(rng, B, max(counts), Hkv, D), _normal(rng, B, max(counts), Hkv, D)
    old[0][..., ::17] *= np.float16(4)
    k[:, n // 2, 0, 3] = np.inf
    v[:, n // 2, :, 7] = np.nan
    v[:, n - 1, :, 9] = -np.inf
    for b, count in enumerate(counts):
        first = count - W  # the oldest position held (the first row sees the one after it)
        if first >= S:
            old[1][b, first + 3, :, 5] = np.inf
            old[1][b, first + n // 3, 0, D - 1] = np.nan
        last = count - 1 - (count - 1 - (W - 1) - S) % W  # the position in the ring's last slot
        if max(S, first) <= last < first + n:  # not seen by all rows
            old[1][b, last, -1] = np.nan
    out, refs = _run(C, q, k, v, old, counts, S, W, group)
    for b in range(B):
        _same(out[b], refs[b], f"b={b} count={counts[b]}")
        assert np.isfinite(refs[b][0]).mean() > 0.125


@pytest.mark.parametrize("D,group,Hq,Hkv", [(128, 64, 8, 2), (64, 32, 5, 5), (128, 32, 18, 2)])
@pytest.mark.parametrize("B,W,counts,nan_at", [
    (1, 4092, [5000], [0, 3, 100, 4095]), (2, 1000, [900, 33], [32, 5]), (3, 12000, [12004, 129, 0], [128, 9000]),
    (1, 60, [40], [39]),
])
def test_decode_a_key_that_is_nan_makes_its_heads_nan(C, D, group, Hq, Hkv, B, W, counts, nan_at):
    """Alone in a step, a warp, a CTA or a piece; the other KV heads and sequences stay as the formula has them."""
    rng = np.random.default_rng(W + D)
    S = 4
    q = _normal(rng, B, Hq, D)
    k, v = _normal(rng, B, S + W, Hkv, D), _normal(rng, B, S + W, Hkv, D)
    k[0, nan_at, -1, 5] = np.nan
    codes, params = C.ring_q4_storage(B, Hkv, D, S, W, group)
    C.ring_append_q4(dev_tensor(k), dev_tensor(v), codes, params, 0, S, W)
    arg = counts[0] if B == 1 else dev_tensor(np.asarray(counts, np.int64))
    out = to_np(C.decode_attention_q4(dev_tensor(q), codes, params, arg, S, W)).astype(np.float64)
    for b, count in enumerate(counts):
        held = min(count, S + W)
        if held == 0:
            assert (out[b] == 0).all()
            continue
        kk, vv = kv4_values(k[b, :held], group), kv4_values(v[b, :held], group)
        ref, bound = _formula(q[b:b + 1], kk, vv, np.ones((1, held), bool))
        # codes and zero points are summed apart: each of the steps over the keys is off by 2^-22 x 2.1 max |v| more
        _same(out[b:b + 1], (ref, bound + (held / 16 + 16) * 2.0 ** -22 * 2.1 * np.abs(vv).max()), f"b={b}")
        assert np.isnan(ref[0, Hq - Hq // Hkv:]).all() == (b == 0)
