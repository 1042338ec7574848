"""Decode and prefill attention over the 4-bit ring against the softmax formula
in 64 bits on the values the cache stands for.

Tolerance of an element, from the roundings: the result once to fp16 (2^-11 of
it); every softmax weight once to fp16 (2^-11 of the sum of weight x |v|), its
subnormals after a scaling by 2^10 or more (2^-35 of the largest weight a key); scores
summed in fp32 over at most D/16 + 16 accumulations whose terms are at most
15 steps of a group by |q|, under 4 times the largest sum of |q| |k| (a value's
group reaches at least 7 steps on one side): each score is off by dS <= 4 size
(D/16 + 16) 2^-23, a weight by a factor exp(2 dS); exp2's 2^-22 and the fp32
sums over L / 16 steps of keys, 2^-23 each.  Decode sums s P c and s P z apart
before it subtracts them: with P at most 1 in all, terms of up to 15 s, and 15 s is
at most (1 + 2^-6) of the group's span, which is at most twice its largest |v|:
each of those fp32 steps is off by 2^-22 x 2.1 max |v| more."""

import numpy as np
import pytest
import torch

from oracle import attention64, kv4_values, ring_positions
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


def _check(got, ref, keys, D, msg="", apart=0.0):
    """``apart``: the largest |value| where the codes' sums are kept apart."""
    out, weight, size = ref
    got = got.astype(np.float64)
    assert got.shape == out.shape
    assert np.array_equal(np.isnan(got), np.isnan(out)), f"{msg}: NaN where the formula has none, or the reverse"
    ds = 4 * size[..., None] * (D / 16 + 16) * 2.0 ** -23
    vmax = np.nanmax(weight, initial=0.0)
    with np.errstate(invalid="ignore"):
        bound = (np.abs(out) * 2.0 ** -11 + 2.0 ** -25 + keys * 2.0 ** -35 * vmax +
                 (keys / 16 + 16) * 2.0 ** -22 * 2.1 * apart +
                 weight * (2.0 ** -11 + np.expm1(2 * ds) + 2.0 ** -20 + (keys / 16 + 16) * 2.0 ** -22))
        bad = np.abs(got - out) > bound
    assert not bad.any(), (msg, int(bad.sum()), np.argwhere(bad)[0], got[bad][0], out[bad][0], bound[bad][0])


def _ring(C, rng, B, H, D, group, S, W, counts, std=1.0):
    """A ring whose sequence b holds counts[b] tokens (only those the ring still
    has are written); slots past them hold the scale NaN.  Returns the storage and
    per sequence (K, V, positions) of the held tokens in 64 bits."""
    codes, params = C.ring_q4_storage(B, H, D, S, W, group)
    codes.fill_(0xFF)
    params.fill_(0x7E0F)
    seqs = []
    for b, n in enumerate(counts):
        slots, pos = ring_positions(int(n), S, W)
        k, v = ((rng.standard_normal((len(pos), H, D)) * std).astype(np.float16) for _ in range(2))
        k[..., ::17] *= np.float16(4)
        one = C.ring_q4_storage(1, H, D, S, W, group)
        tmp_k, tmp_v = dev_tensor(k[None]), dev_tensor(v[None])
        # written as a fresh ring in slot order, then placed: slot i holds the token of slots[i]
        order = np.argsort(slots)
        if len(pos):
            C.ring_append_q4(tmp_k[:, order].contiguous(), tmp_v[:, order].contiguous(), *one, 0, S, W)
            codes[:, b, :, :len(pos)] = one[0][:, 0, :, :len(pos)]
            params[:, b, :, :len(pos)] = one[1][:, 0, :, :len(pos)]
        seqs.append((kv4_values(k, group), kv4_values(v, group), pos))
    return codes, params, seqs


def _decode(C, B, Hq, Hkv, D, group, S, W, count, seed, scale=None, std=1.0, qstd=1.0):
    rng = np.random.default_rng(seed)
    counts = np.broadcast_to(count, (B,))
    codes, params, seqs = _ring(C, rng, B, Hkv, D, group, S, W, counts, std)
    q = (rng.standard_normal((B, Hq, D)) * qstd).astype(np.float16)
    arg = int(count) if np.ndim(count) == 0 else dev_tensor(np.asarray(count, np.int64))
    out = C.decode_attention_q4(dev_tensor(q), codes, params, arg, S, W, scale)
    for b in range(B):
        k, v, pos = seqs[b]
        ref = attention64(q[b][None], k, v, np.ones((1, len(pos)), bool), scale)
        _check(to_np(out)[b][None], ref, len(pos), D, f"b={b} count={counts[b]}", np.abs(v).max(initial=0.0))
    return q, codes, params, out


@pytest.mark.parametrize("count", [0, 1, 3, 31, 32, 33, 64, 65, 127, 128, 129, 1000, 4095, 4096, 4097, 9000])
def test_decode_lengths(C, count):
    _decode(C, 1, 32, 8, 128, 64, 4, 4092, count, seed=count)


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (8, 8), (15, 5), (14, 2), (8, 1), (9, 1), (32, 2)])
def test_decode_heads_and_groups(C, D, group, Hq, Hkv):
    _decode(C, 2, Hq, Hkv, D, group, 4, 300, 777, seed=Hq * 10 + D + group)


@pytest.mark.parametrize("B", [1, 3, 40])
def test_decode_batch_with_its_own_counts(C, B):
    rng = np.random.default_rng(B)
    counts = rng.integers(0, 2500, B)
    counts[B // 2] = 0
    _decode(C, B, 8, 2, 128, 64, 4, 996, counts, seed=B)


@pytest.mark.parametrize("B,Hq,Hkv,D,group,W,counts", [
    (6, 8, 2, 128, 64, 12000, [0, 13000, 1, 5000, 0, 129]), (4, 6, 3, 64, 32, 12000, 20000),
    (2, 18, 2, 128, 32, 12000, [12004, 77]), (3, 4, 1, 128, 128, 9000, [0, 0, 0]), (1, 9, 1, 64, 64, 12000, 300),
    (150, 2, 1, 64, 64, 2000, "mixed"), (300, 1, 1, 64, 32, 700, "mixed")])
def test_decode_runs(C, B, Hq, Hkv, D, group, W, counts):
    """Rings wide enough that the CTAs take runs over all pairs (more sequences than a
    block has threads, too) instead of a cluster a pair."""
    if counts == "mixed":
        rng = np.random.default_rng(B)
        counts = np.where(rng.random(B) < 0.3, 0, rng.integers(0, 2 * W, B))
    _decode(C, B, Hq, Hkv, D, group, 4, W, np.array(counts) if isinstance(counts, list) else counts, seed=B)


@pytest.mark.parametrize("count", [0, 500, 1500])
def test_decode_runs_that_end_with_pairs(C, count):
    """As many pairs as CTAs are resident: every pair is one CTA's."""
    B = 2 * torch.cuda.get_device_properties(0).multi_processor_count
    _decode(C, B, 1, 1, 128, 64, 0, 1000, count, seed=3)
    _decode(C, 3, 2, 1, 128, 64, 4, 5, count, seed=4)  # a CTA a pair: a ring of one unit


def test_decode_small_rings_scale_and_sizes(C):
    for S, W, count in [(0, 1, 5), (1, 1, 1), (4, 8, 12), (17, 8, 9), (2, 70, 200), (4, 60, 64)]:
        _decode(C, 1, 8, 2, 128, 64, S, W, count, seed=S * 100 + W)
    _decode(C, 1, 32, 8, 128, 64, 4, 1020, 900, seed=9, scale=0.05)
    _decode(C, 2, 8, 2, 64, 32, 4, 1020, 2000, seed=3, std=8.0)    # near one-hot
    _decode(C, 2, 8, 2, 128, 64, 4, 1020, 2000, seed=4, std=300.0, qstd=1e-4)  # tiny queries, large keys
    _decode(C, 2, 8, 2, 128, 128, 4, 1020, 2000, seed=5, std=1e-3, qstd=500.0)


def test_decode_long(C):
    """A wide ring: many splits; against the formula with the read-back values."""
    S, W, H, D = 4, 131068, 1, 128
    g = torch.Generator(device="cuda").manual_seed(2)
    codes, params = C.ring_q4_storage(1, H, D, S, W, 64)
    for at in range(0, S + W, 16384):
        k, v = (torch.randn(1, 16384, H, D, generator=g, device="cuda").half() for _ in range(2))
        C.ring_append_q4(k, v, codes, params, at, S, W)
    q = torch.randn(1, 4, D, generator=g, device="cuda").half()
    k, v = (to_np(t)[0] for t in C.ring_gather_q4(codes, params, S + W, S, W))
    out = C.decode_attention_q4(q, codes, params, S + W, S, W)
    ref = attention64(to_np(q), k, v, np.ones((1, S + W), bool))
    _check(to_np(out), ref, S + W, D, apart=np.abs(v.astype(np.float64)).max())
    counts = torch.full((1,), (1 << 40) + 5, dtype=torch.int64, device="cuda")  # the ring is full: every slot counts
    assert torch.equal(C.decode_attention_q4(q, codes, params, counts, S, W), out)


def test_decode_non_finite_values(C):
    rng = np.random.default_rng(8)
    B, Hq, Hkv, D, group, S, W, n = 3, 4, 2, 128, 64, 4, 60, 50
    k, v = (rng.standard_normal((B, n, Hkv, D)).astype(np.float16) for _ in range(2))
    k[0, 20, 1, 3] = np.nan   # every score of that token: rows of KV head 1 are NaN
    v[1, 30, 0, 70] = np.inf  # its group of 64 values only
    codes, params = C.ring_q4_storage(B, Hkv, D, S, W, group)
    C.ring_append_q4(dev_tensor(k), dev_tensor(v), codes, params, 0, S, W)
    q = rng.standard_normal((B, Hq, D)).astype(np.float16)
    q[2, 3, 5] = np.inf
    out = to_np(C.decode_attention_q4(dev_tensor(q), codes, params, n, S, W))
    nan = np.zeros((B, Hq, D), bool)
    nan[0, 2:] = True
    nan[1, :2, 64:] = True
    nan[2, 3] = True
    assert np.array_equal(np.isnan(out), nan)


@pytest.mark.parametrize("D,group,bad", [(128, 32, 40), (128, 64, 3), (64, 32, 63)])
def test_decode_a_group_that_reads_as_nan_leaves_the_others_exact(C, D, group, bad):
    """Small values next to a group whose scale is NaN keep their weights' bits."""
    rng = np.random.default_rng(D + group)
    n, S, W = 5, 4, 60
    k = rng.standard_normal((1, n, 1, D)).astype(np.float16)
    v = (rng.standard_normal((1, n, 1, D)) * 2.0 ** -9).astype(np.float16)
    v[0, 2, 0, bad] = np.nan
    codes, params = C.ring_q4_storage(1, 1, D, S, W, group)
    C.ring_append_q4(dev_tensor(k), dev_tensor(v), codes, params, 0, S, W)
    q = rng.standard_normal((1, 4, D)).astype(np.float16)
    out = to_np(C.decode_attention_q4(dev_tensor(q), codes, params, n, S, W))
    v64 = kv4_values(v, group)[0]
    ref = attention64(q, kv4_values(k, group)[0], v64, np.ones((1, n), bool))
    _check(out, ref, n, D, apart=np.nanmax(np.abs(v64)))


def test_decode_cache_object_streams_and_graph(C):
    """One captured step follows its count tensor and its cache; on another stream the same bits."""
    rng = np.random.default_rng(11)
    B, Hq, Hkv, D, S, W = 2, 8, 2, 128, 4, 124
    codes, params = C.ring_q4_storage(B, Hkv, D, S, W, 64)
    count = torch.zeros(B, dtype=torch.int64, device="cuda")
    q, k, v = (torch.zeros(B, h, D, dtype=torch.float16, device="cuda") for h in (Hq, Hkv, Hkv))

    def step():
        C.ring_append_q4(k.unsqueeze(1), v.unsqueeze(1), codes, params, count, S, W)
        return C.decode_attention_q4(q, codes, params, count + 1, S, W)

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = step()
        graphs.append((graph, out))
    cache = C.RingBufferKVCacheQ4(1, Hkv, D, S, W, batch=B)
    side = torch.cuda.Stream()
    for t in range(140):
        for x in (q, k, v):
            x.copy_(dev_tensor(rng.standard_normal(tuple(x.shape)).astype(np.float16)))
        count.fill_(t)
        graph, out = graphs[t % 2]
        graph.replay()
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            cache.append(k.unsqueeze(1), v.unsqueeze(1), 0)
            want = cache.decode_attention(q, 0)
        side.synchronize()
        assert torch.equal(out, want), t


def _prefill(C, B, n, Hq, Hkv, D, group, S, W, count, seed, scale=None, poison=False):
    rng = np.random.default_rng(seed)
    counts = np.broadcast_to(count, (B,))
    codes, params, seqs = _ring(C, rng, B, Hkv, D, group, S, W, counts)
    q = rng.standard_normal((B, n, Hq, D)).astype(np.float16)
    k, v = (rng.standard_normal((B, n, Hkv, D)).astype(np.float16) for _ in range(2))
    if poison:  # keys that the first rows must not see
        k[:, n // 2, 0, 3] = np.inf
        v[:, n // 2, :, 7] = np.nan
        v[:, n - 1, :, 9] = -np.inf
    arg = int(count) if np.ndim(count) == 0 else dev_tensor(np.asarray(count, np.int64))
    out = C.prefill_attention_q4(dev_tensor(q), dev_tensor(k), dev_tensor(v), codes, params, arg, S, W, scale)
    for b in range(B):
        ko, vo, pos = seqs[b]
        at = int(counts[b]) + np.arange(n)
        kp = np.concatenate([pos, at])
        seen = (kp[None] <= at[:, None]) & ((kp[None] < S) | (kp[None] > at[:, None] - W))
        ref = attention64(q[b], np.concatenate([ko, k[b].astype(np.float64)]),
                          np.concatenate([vo, v[b].astype(np.float64)]), seen, scale)
        _check(to_np(out)[b], ref, len(kp), D, f"b={b} count={counts[b]}")
    return out


@pytest.mark.parametrize("n", [1, 2, 31, 33, 63, 64, 65, 127, 128, 129, 300])
@pytest.mark.parametrize("count", [0, 100, 5000])
def test_prefill_lengths(C, n, count):
    _prefill(C, 1, n, 8, 2, 128, 64, 4, 252, count, seed=n + count)


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("Hq,Hkv", [(1, 1), (15, 5), (7, 1), (16, 1), (12, 4)])
def test_prefill_heads_and_groups(C, D, group, Hq, Hkv):
    _prefill(C, 2, 70, Hq, Hkv, D, group, 4, 140, 333, seed=Hq + D + group)


@pytest.mark.parametrize("S,W,count,n", [(0, 1, 0, 5), (0, 1, 7, 3), (4, 60, 2, 100), (17, 8, 5, 40), (17, 8, 30, 5),
                                         (4, 1000, 3, 200), (4, 100, 103, 1), (4, 100, 104, 257), (1, 64, 65, 64)])
def test_prefill_rings(C, S, W, count, n):
    _prefill(C, 1, n, 4, 2, 128, 64, S, W, count, seed=S + W + n)


def test_prefill_batch_with_its_own_counts(C):
    _prefill(C, 4, 90, 6, 2, 64, 32, 4, 200, np.array([0, 3, 170, 1 << 40]), seed=1)
    _prefill(C, 3, 33, 8, 2, 128, 64, 4, 3000, np.array([2900, 0, 7000]), seed=2, scale=0.2)


@pytest.mark.parametrize("D,group,n", [(128, 64, 150), (64, 32, 40)])
def test_prefill_hidden_values_do_not_reach_a_row(C, D, group, n):
    """NaN and infinities in a chunk's later keys and values, NaN scales in the ring's free slots."""
    _prefill(C, 2, n, 4, 2, D, group, 4, 100, np.array([30, 400]), seed=n, poison=True)


def test_prefill_evicted_values_do_not_reach_a_row(C):
    """A NaN token of the ring is seen by the first rows and evicted for the later ones."""
    S, W, n, D = 0, 64, 60, 128
    rng = np.random.default_rng(5)
    k, v = (rng.standard_normal((1, W, 1, D)).astype(np.float16) for _ in range(2))
    v[0, 20, 0, 3] = np.inf
    codes, params = C.ring_q4_storage(1, 1, D, S, W, 64)
    C.ring_append_q4(dev_tensor(k), dev_tensor(v), codes, params, 0, S, W)
    q, kn, vn = (dev_tensor(rng.standard_normal((1, n, h, D)).astype(np.float16)) for h in (4, 1, 1))
    out = to_np(C.prefill_attention_q4(q, kn, vn, codes, params, W, S, W))[0]
    # position 20 is visible to row r (position 64 + r) iff 20 > 64 + r - 64
    assert np.isnan(out[:20, :, :64]).all() and np.isfinite(out[20:]).all() and np.isfinite(out[:, :, 64:]).all()


@pytest.mark.parametrize("n,W,count", [(700, 4092, 5000), (700, 4092, 100), (90, 4092, 4000)])
def test_prefill_a_visible_value_that_is_not_finite_costs_no_repair(C, n, W, count):
    """A NaN value that every row sees makes its column (its group, in the ring) NaN
    and nothing else, and no row is done again for it: within 20 times the time of
    the call without it (a repair of every row took hundreds)."""
    S, H, D = 4, 2, 128
    rng = np.random.default_rng(n)
    g = torch.Generator(device="cuda").manual_seed(n)

    def halves(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()

    q, k, v = halves(1, n, 8, D), halves(1, n, H, D), halves(1, n, H, D)
    ring = [C.ring_q4_storage(1, H, D, S, W, 64) for _ in range(2)]
    ko, vo = halves(1, count, H, D), halves(1, count, H, D)
    C.ring_append_q4(ko, vo, *ring[0], 0, S, W)
    vo[0, 1] = float("nan")  # a sink
    C.ring_append_q4(ko, vo, *ring[1], 0, S, W)
    times = []
    for codes, params in ring:
        for i in range(2):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            out = C.prefill_attention_q4(q, k, v, codes, params, count, S, W)
            b.record()
            b.synchronize()
        times.append(a.elapsed_time(b))
    assert out.isnan().all()
    assert times[1] < 20 * times[0] + 0.2, times
    v[0, 0, 1, 5] = float("inf")  # the chunk's first key: hidden from no row
    out = C.prefill_attention_q4(q, k, v, *ring[0], count, S, W)
    fine = out.isfinite()
    assert not fine[:, :, 4:, 5].any() and fine[:, :, :4].all() and fine[..., :5].all() and fine[..., 6:].all()


def test_prefill_free_slots_behind_a_nan(C):
    """The token in the ring's last slot is NaN and evicted for the later rows; the tile goes on behind it."""
    S, W, n, D = 0, 70, 100, 64
    rng = np.random.default_rng(6)
    count = 70
    k, v = (rng.standard_normal((1, count, 1, D)).astype(np.float16) for _ in range(2))
    v[0, 69] = np.nan
    codes, params = C.ring_q4_storage(1, 1, D, S, W, 32)
    C.ring_append_q4(dev_tensor(k), dev_tensor(v), codes, params, 0, S, W)
    # two more tokens put position 70 into slot 0: the ring then starts at slot 2
    x = dev_tensor(rng.standard_normal((1, 2, 1, D)).astype(np.float16))
    C.ring_append_q4(x, x, codes, params, count, S, W)
    q, kn, vn = (dev_tensor(rng.standard_normal((1, n, h, D)).astype(np.float16)) for h in (2, 1, 1))
    out = to_np(C.prefill_attention_q4(q, kn, vn, codes, params, count + 2, S, W))[0]
    # position 69 is visible to row r (position 72 + r) iff 69 > 72 + r - 70
    assert np.isnan(out[:67]).all() and np.isfinite(out[67:]).all()


@pytest.mark.parametrize("counted", [False, True])
def test_calls_at_once_and_captured(C, counted):
    """Split prefill and decode in runs, eager on two streams at once, then captured as two graphs that are replayed at
    once: the same bits as one call alone (each call has its own scratch)."""
    g = torch.Generator(device="cuda").manual_seed(8)

    def halves(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()

    B, Hq, H, D, S, W, n = 2, 8, 2, 128, 4, 9000, 37
    rings, args = [], []
    for i in range(2):
        ring = C.ring_q4_storage(B, H, D, S, W, 64)
        C.ring_append_q4(halves(B, 9004, H, D), halves(B, 9004, H, D), *ring, 0, S, W)
        rings.append(ring)
        args.append((halves(B, n, Hq, D), halves(B, n, H, D), halves(B, n, H, D), halves(B, Hq, D)))
    counts = [torch.tensor(c, device="cuda") for c in ([8000, 301], [12000, 9004])]

    def both(i):
        q, k, v, one = args[i]
        count = counts[i] if counted else (8000, 12000)[i]
        return (C.prefill_attention_q4(q, k, v, *rings[i], count, S, W), C.decode_attention_q4(one, *rings[i], count, S, W))

    want = [both(i) for i in range(2)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        got = []
        for i, st in enumerate(streams):
            with torch.cuda.stream(st):
                got.append(both(i))
        torch.cuda.synchronize()
        for a, b in zip(got, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    graphs, outs = [], []
    for i in range(2):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            outs.append(both(i))
    for _ in range(5):
        for o in outs:
            for t in o:
                t.zero_()
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])


def test_host_count_and_device_count_give_the_same_bits(C):
    for seed, (B, Hq, H, D, group, W, count) in enumerate([(1, 8, 2, 128, 64, 20000, 15000), (3, 6, 2, 64, 32, 9000, 30000),
                                                          (2, 18, 2, 128, 128, 500, 400), (140, 2, 1, 64, 64, 700, 600)]):
        codes, params, _ = _ring(C, np.random.default_rng(seed), 1, H, D, group, 4, W, [count])
        codes, params = (t.expand(2, B, *t.shape[2:]).contiguous() for t in (codes, params))
        g = torch.Generator(device="cuda").manual_seed(seed)
        q = torch.randn(B, Hq, D, generator=g, device="cuda").half()
        each = torch.full((B,), count, dtype=torch.int64, device="cuda")
        assert torch.equal(C.decode_attention_q4(q, codes, params, count, 4, W),
                           C.decode_attention_q4(q, codes, params, each, 4, W))
        q, k, v = (torch.randn(B, 21, h, D, generator=g, device="cuda").half() for h in (Hq, H, H))
        assert torch.equal(C.prefill_attention_q4(q, k, v, codes, params, count, 4, W),
                           C.prefill_attention_q4(q, k, v, codes, params, each, 4, W))


def test_prefill_equals_fp16_prefill_of_the_read_back(C):
    """Where the 4-bit ring's read-back is put into an fp16 ring, both attentions
    see the same numbers: equal up to the two kernels' fp32 order and weight rounding."""
    rng = np.random.default_rng(21)
    B, n, Hq, Hkv, D, S, W, count = 1, 257, 8, 2, 128, 4, 508, 700
    codes, params, seqs = _ring(C, rng, B, Hkv, D, 64, S, W, [count])
    kv = [torch.zeros(B, S + W, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2)]
    slots, _ = ring_positions(count, S, W)
    for t, r in zip(kv, C.ring_gather_q4(codes, params, count, S, W)):
        t[:, torch.from_numpy(slots).cuda()] = r
    q, k, v = (dev_tensor(rng.standard_normal((B, n, h, D)).astype(np.float16)) for h in (Hq, Hkv, Hkv))
    a = C.prefill_attention_q4(q, k, v, codes, params, count, S, W).float()
    b = C.prefill_attention(q, k, v, *kv, count, S, W).float()
    assert ((a - b).norm() / b.norm()).item() < 2.0 ** -10


def test_refusals(C):
    codes, params = C.ring_q4_storage(2, 3, 128, 4, 60, 64)
    q = torch.zeros(2, 6, 128, dtype=torch.float16, device="cuda")
    x = torch.zeros(2, 5, 3, 128, dtype=torch.float16, device="cuda")
    qn = torch.zeros(2, 5, 6, 128, dtype=torch.float16, device="cuda")
    for bad in (q.float(), q[:1], q[:, :4].contiguous(), q[..., :64].contiguous(), q.cpu(), q[:, ::2],
                torch.zeros(2, 51, 128, dtype=torch.float16, device="cuda")):
        with pytest.raises(RuntimeError):
            C.decode_attention_q4(bad, codes, params, 5, 4, 60)
    for count, S, W in ((-1, 4, 60), (5, 4, 61), (torch.zeros(1, dtype=torch.int64, device="cuda"), 4, 60)):
        with pytest.raises(RuntimeError):
            C.decode_attention_q4(q, codes, params, count, S, W)
        with pytest.raises(RuntimeError):
            C.prefill_attention_q4(qn, x, x, codes, params, count, S, W)
    for a in ((qn.float(), x, x), (qn, x[:, :4].contiguous(), x), (qn[:, :, :5].contiguous(), x, x), (qn, x, x.cpu()),
              (qn[0], x, x)):
        with pytest.raises(RuntimeError):
            C.prefill_attention_q4(*a, codes, params, 5, 4, 60)
    assert C.prefill_attention_q4(qn[:, :0].contiguous(), x[:, :0].contiguous(), x[:, :0].contiguous(), codes, params,
                                  5, 4, 60).shape == (2, 0, 6, 128)
    assert C.decode_attention_q4(q[:0].contiguous(), codes[:, :0].contiguous(), params[:, :0].contiguous(), 5, 4,
                                 60).shape == (0, 6, 128)
