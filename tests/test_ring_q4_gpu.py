"""The 4-bit ring: what is appended and read back, bit for bit, against the
quantiser's definition in 64 bits; its slots, counts and refusals."""

import numpy as np
import pytest
import torch

from oracle import kv4_values, ring_positions
from tests._util import dev_tensor, to_np

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


def _tokens(rng, *shape):
    """fp16 values with wide channels, values on a coarse grid (quotients that are
    ties), one-sided, tiny and large rows."""
    x = rng.standard_normal(shape).astype(np.float32)
    x[..., rng.random(shape[-1]) < 0.05] *= 8
    kind = rng.integers(0, 8, shape[:-1])[..., None]
    x = np.where(kind == 1, np.round(x * 4) / 4, x)
    x = np.where(kind == 2, np.abs(x), x)
    x = np.where(kind == 3, x * 1e-6, x)
    x = np.where(kind == 4, x * 9000, x)
    x = np.where(kind == 5, 0, x)
    return np.clip(x, -65504, 65504).astype(np.float16)


def _same(a, b):
    a = a.astype(np.float64)
    assert a.shape == b.shape
    assert np.array_equal(np.isnan(a), np.isnan(b))
    assert np.array_equal(np.nan_to_num(a), np.nan_to_num(b)), np.argwhere(np.nan_to_num(a) != np.nan_to_num(b))[:5]


@pytest.mark.parametrize("D,group", [(64, 32), (64, 64), (128, 32), (128, 64), (128, 128)])
@pytest.mark.parametrize("B,H,S,W,chunks", [
    (1, 8, 4, 60, [1]), (2, 3, 4, 60, [3, 1, 1, 90]), (1, 2, 0, 1, [1, 1, 5]), (3, 1, 17, 8, [2, 16, 1, 30]),
    (2, 5, 4, 100, [64, 64, 64, 1]),
])
def test_append_and_gather_equal_the_definition(C, D, group, B, H, S, W, chunks):
    rng = np.random.default_rng(D + group + W)
    T = sum(chunks)
    k, v = _tokens(rng, B, T, H, D), _tokens(rng, B, T, H, D)
    k64, v64 = kv4_values(k, group), kv4_values(v, group)
    codes, params = C.ring_q4_storage(B, H, D, S, W, group)
    done = 0
    for n in chunks:
        C.ring_append_q4(dev_tensor(k[:, done:done + n]), dev_tensor(v[:, done:done + n]), codes, params, done, S, W)
        done += n
        ko, vo = C.ring_gather_q4(codes, params, done, S, W)
        _, pos = ring_positions(done, S, W)
        _same(to_np(ko), k64[:, pos])
        _same(to_np(vo), v64[:, pos])
    err = np.abs(k64 - k.astype(np.float64)).reshape(B, T, H, -1, group)
    x = k.astype(np.float64).reshape(err.shape)
    s = (np.maximum(x.max(-1), 0) - np.minimum(x.min(-1), 0)) / 15 * (1 + 1 / 64) + 2.0 ** -20
    assert (err <= s[..., None] * np.where(np.abs(x) > 32000, 1.0, 0.5)).all()


def test_extreme_groups(C):
    x = np.zeros((1, 12, 1, 64), np.float16)
    x[0, 0, 0, :] = 65504
    x[0, 1, 0, :] = -65504
    x[0, 2, 0, ::2], x[0, 2, 0, 1::2] = 65504, -65504
    x[0, 3, 0, 5] = np.float16(2.0 ** -24)
    x[0, 4, 0, 6] = -np.float16(2.0 ** -14)
    x[0, 5, 0, 7] = np.nan
    x[0, 6, 0, 40] = np.inf
    x[0, 7, 0, 3] = -np.inf
    x[0, 8, 0, :] = -0.0
    x[0, 9, 0, :] = np.arange(64) / 8  # quotients of 15 steps and their halves
    x[0, 10, 0, 0], x[0, 10, 0, 1] = 60000, 1e-3
    x[0, 11, 0, :32] = 1.0
    codes, params = C.ring_q4_storage(1, 1, 64, 0, 12, 32)
    C.ring_append_q4(dev_tensor(x), dev_tensor(x[:, ::-1]), codes, params, 0, 0, 12)
    ko, vo = C.ring_gather_q4(codes, params, 12, 0, 12)
    want = kv4_values(x, 32)
    assert np.isnan(want[0, 5, 0, :32]).all() and np.isfinite(want[0, 5, 0, 32:]).all()
    assert np.abs(want[0, 2]).max() <= 65504
    _same(to_np(ko), want)
    _same(to_np(vo), want[:, ::-1])


def test_a_chunk_leaves_the_ring_as_single_tokens_do(C):
    """Storage bit for bit, other slots untouched, sequences with their own counts."""
    rng = np.random.default_rng(3)
    B, H, D, S, W, T = 3, 2, 128, 4, 50, 41
    k, v = (dev_tensor(_tokens(rng, B, T, H, D)) for _ in range(2))
    counts = torch.tensor([0, 30, 1000003], device="cuda")
    a, b = (C.ring_q4_storage(B, H, D, S, W, 64) for _ in range(2))
    for c, p in (a, b):
        c.fill_(0xA5)
        p.fill_(0x1234)
    C.ring_append_q4(k, v, *a, counts, S, W)
    for t in range(T):
        C.ring_append_q4(k[:, t:t + 1].contiguous(), v[:, t:t + 1].contiguous(), *b, counts + t, S, W)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    assert (a[1][:, 0, :, T:] == 0x1234).all() and (a[0][:, 0, :, T:] == 0xA5).all()  # first sequence: 41 tokens
    assert (a[1][:, :, :, S + W:] == 0x1234).all()
    one = C.ring_q4_storage(1, H, D, S, W, 64)
    C.ring_append_q4(k[2:].contiguous(), v[2:].contiguous(), *one, 1000003, S, W)
    used = torch.tensor([S + (1000003 + t - S) % W for t in range(T)], device="cuda")
    assert torch.equal(one[0][:, 0][:, :, used], a[0][:, 2][:, :, used])


def test_cache_objects(C):
    import qextract_infer_b200 as q
    rng = np.random.default_rng(1)
    k, v = _tokens(rng, 100, 8, 128), _tokens(rng, 100, 8, 128)
    cache = q.QExtractKVCache(2, 8, 128, sink_size=4, window_size=60, bits=4)
    for layer in range(2):
        cache.append(dev_tensor(k[:70]), dev_tensor(v[:70]), layer)
    for t in range(70, 100):
        for layer in range(2):
            cache.append(dev_tensor(k[t]), dev_tensor(v[t]), layer)
    assert cache.write_count == 100 and cache.valid_length == 64
    assert cache.memory_usage_bytes() == 2 * 2 * 8 * 64 * (64 + 2 * 2)
    _, pos = ring_positions(100, 4, 60)
    ko, vo = cache.get_kv(1)
    _same(to_np(ko), kv4_values(k[pos], 64))
    _same(to_np(vo), kv4_values(v[pos], 64))
    cache.reset()
    assert cache.valid_length == 0 and cache.get_kv(0)[0].shape == (0, 8, 128)
    with pytest.raises(RuntimeError, match="16 or 4 bits"):
        q.QExtractKVCache(2, 8, 128, bits=8)
    with pytest.raises(RuntimeError):
        q.QExtractKVCache(2, 8, 96, bits=4)
    batched = C.RingBufferKVCacheQ4(1, 2, 64, 4, 60, batch=3, group_size=32)
    x = dev_tensor(_tokens(rng, 3, 7, 2, 64))
    batched.append(x, x, 0)
    assert batched.get_kv(0)[0].shape == (3, 7, 2, 64) and batched.get_total_written() == 7


def test_refusals(C):
    codes, params = C.ring_q4_storage(2, 3, 128, 4, 60, 64)
    x = torch.zeros(2, 5, 3, 128, dtype=torch.float16, device="cuda")
    ok = dict(k=x, v=x, codes=codes, params=params, count=0, sink=4, window=60)
    for bad in (dict(k=x.float()), dict(k=x[:1]), dict(v=x[:, :4].contiguous()), dict(k=x.transpose(1, 2)),
                dict(codes=codes.int()), dict(codes=codes[:1].contiguous()), dict(params=params[..., :0].contiguous()),
                dict(params=params.half()), dict(window=61), dict(window=0), dict(sink=-1), dict(count=-1),
                dict(count=torch.zeros(2, dtype=torch.int32, device="cuda")), dict(count=torch.zeros(2, dtype=torch.int64)),
                dict(count=torch.zeros(3, dtype=torch.int64, device="cuda")), dict(k=x.cpu(), v=x.cpu())):
        a = {**ok, **bad}
        with pytest.raises(RuntimeError):
            C.ring_append_q4(a["k"], a["v"], a["codes"], a["params"], a["count"], a["sink"], a["window"])
    with pytest.raises(RuntimeError, match="number"):
        C.ring_gather_q4(codes, params, torch.zeros(2, dtype=torch.int64, device="cuda"), 4, 60)
    with pytest.raises(RuntimeError):
        C.ring_gather_q4(codes, params, -1, 4, 60)
    C.ring_append_q4(x[:, :0].contiguous(), x[:, :0].contiguous(), codes, params, 0, 4, 60)  # nothing to do
    with pytest.raises(RuntimeError):
        C.ring_q4_storage(1, 1, 96, 4, 60, 32)
    with pytest.raises(RuntimeError):
        C.ring_q4_storage(1, 1, 64, 4, 60, 128)
