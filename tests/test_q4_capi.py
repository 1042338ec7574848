"""Refusals of the 4-bit ring's entry points and of qx_qk_norm_rope at the C ABI
(before any launch: no GPU), and the quantiser's oracle on its own definition."""

import ctypes

import numpy as np
import pytest

from oracle import kv4_values
from qextract_infer_b200 import _lib

P = 4096  # a well-aligned address that is never read


def _append(lib, k_codes=P, new_k=P, batch=2, tokens=3, hkv=2, d=128, group=64, sink=4, window=60, count=0, counts=None):
    return lib.qx_ring_append_q4(k_codes, P, P, P, new_k, P, batch, tokens, hkv, d, group, sink, window, count, counts,
                                 None)


def _decode(lib, q=P, out=P, batch=2, hq=4, hkv=2, d=128, group=64, sink=4, window=60, count=0, counts=None, ws=None,
            nbytes=0):
    return lib.qx_decode_attention_q4(q, P, P, P, P, out, batch, hq, hkv, d, group, sink, window, count, counts,
                                      ctypes.c_float(0), ws, nbytes, None)


def _prefill(lib, q=P, batch=2, n=3, hq=4, hkv=2, d=128, group=64, sink=4, window=60, count=0, counts=None, ws=None,
             nbytes=0):
    return lib.qx_prefill_attention_q4(q, P, P, P, P, P, P, P, batch, n, hq, hkv, d, group, sink, window, count, counts,
                                       ctypes.c_float(0), ws, nbytes, None)


RING = [(dict(batch=-1), "bad sizes"), (dict(hkv=0), "kv"), (dict(d=96), "head_dim"), (dict(d=256), "head_dim"),
        (dict(group=16), "group"), (dict(d=64, group=128), "group"), (dict(sink=-1), "sink"), (dict(window=0), "window"),
        (dict(window=(1 << 31) - 8), "too large"), (dict(count=-1), "count"),
        (dict(count=1 << 62), "count")]


@pytest.mark.parametrize("call", [_append, _decode, _prefill])
@pytest.mark.parametrize("bad,msg", RING)
def test_ring_arguments(call, bad, msg):
    lib = _lib.load()
    assert call(lib, **bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()


@pytest.mark.parametrize("call,bad,msg", [
    (_append, dict(k_codes=None), "null"), (_append, dict(new_k=P + 8), "aligned"), (_append, dict(tokens=-1), "tokens"),
    (_decode, dict(hq=5), "heads"), (_decode, dict(hq=34), "heads"), (_decode, dict(q=None), "null"),
    (_decode, dict(out=P + 2), "aligned"), (_prefill, dict(hq=0), "heads"), (_prefill, dict(hq=66), "heads"),
    (_prefill, dict(n=-1), "n=-1"), (_prefill, dict(n=1 << 27), "too large"), (_prefill, dict(q=P + 4), "aligned"),
])
def test_other_arguments(call, bad, msg):
    lib = _lib.load()
    assert call(lib, **bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()


def test_nothing_to_do_and_workspace():
    lib = _lib.load()
    assert _append(lib, batch=0) == 0 and _append(lib, tokens=0) == 0
    assert _decode(lib, batch=0) == 0 and _prefill(lib, n=0) == 0 and _prefill(lib, batch=0) == 0
    assert lib.qx_ring_gather_q4(None, None, None, None, None, None, 2, 2, 128, 64, 4, 60, 0, None) == 0
    assert lib.qx_ring_gather_q4(P, P, P, P, P, P, 2, 2, 128, 64, 4, 60, -1, None) == -1
    assert lib.qx_ring_gather_q4(P, P, P, P, P, None, 2, 2, 128, 64, 4, 60, 5, None) == -1
    assert [lib.qx_ring_q4_slots(s, w) for s, w in ((4, 60), (4, 61), (0, 1), (4, 4092))] == [64, 128, 64, 4096]
    assert lib.qx_ring_q4_slots(-1, 5) < 0
    need = lib.qx_decode_attention_q4_workspace_size(1, 32, 8, 128, 4, 4092)
    if need:
        for ws, nbytes in ((None, need), (P, need - 1), (P + 4, need)):
            assert _decode(lib, batch=1, hq=32, hkv=8, window=4092, count=5, ws=ws, nbytes=nbytes) == -3
            assert "workspace" in _lib.last_error()
    assert lib.qx_decode_attention_q4_workspace_size(1, 30, 8, 128, 4, 4092) == 0


@pytest.mark.parametrize("bad,msg", [
    (dict(tokens=-1), "sizes"), (dict(hq=0), "sizes"), (dict(d=32), "head_dim"), (dict(tokens=1 << 31), "too large"),
    (dict(hq=70000), "heads"), (dict(rows=4), "rotation rows"), (dict(rows=0), "rotation rows"), (dict(qkv=None), "null"),
    (dict(cos=P + 4), "aligned")])
def test_qk_norm_rope_arguments(bad, msg):
    lib = _lib.load()

    def call(qkv=P, tokens=6, hq=4, hkv=2, d=128, cos=P, rows=3):
        return lib.qx_qk_norm_rope(qkv, tokens, hq, hkv, d, P, P, ctypes.c_float(1e-6), cos, P, rows, P, P, P, None)

    assert call(**bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()
    assert call(tokens=0) == 0


def test_python_ops_reject_cpu_tensors():
    import torch
    from qextract_infer_b200 import _C
    codes, params = torch.zeros(2, 1, 2, 64, 64, dtype=torch.uint8), torch.zeros(2, 1, 2, 64, 2, dtype=torch.int16)
    x = torch.zeros(1, 3, 2, 128, dtype=torch.float16)
    for call in (lambda: _C.ring_append_q4(x, x, codes, params, 0, 4, 60), lambda: _C.ring_gather_q4(codes, params, 3, 4, 60),
                 lambda: _C.decode_attention_q4(x[:, 0], codes, params, 3, 4, 60),
                 lambda: _C.prefill_attention_q4(x, x, x, codes, params, 3, 4, 60),
                 lambda: _C.qk_norm_rope(x.view(1, 3, 256), 1, 1, x[0, 0, 0], x[0, 0, 0], 1e-6, x[0, 0], x[0, 0])):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()


@pytest.mark.parametrize("group", [32, 64, 128])
def test_quantiser_definition(group):
    """The oracle's values are fp16 numbers, s is minimal among the 7-bit numbers, the error at most half a step."""
    rng = np.random.default_rng(group)
    x = (rng.standard_normal((400, 128)) * np.exp(rng.uniform(-12, 9, (400, 1)))).astype(np.float16)
    y = kv4_values(x, group)
    assert np.array_equal(y.astype(np.float16).astype(np.float64), y)
    table = np.arange(0x7C00, dtype=np.uint16)
    table = np.unique((table & 0xFFF0).view(np.float16).astype(np.float64))
    for row, out in zip(x.astype(np.float64).reshape(-1, group), y.reshape(-1, group)):
        span = max(row.max(), 0) - min(row.min(), 0)
        s = table[np.searchsorted(table, span / 15)]
        if s == 0:
            assert (out == 0).all()
            continue
        assert np.array_equal(np.rint(out / s) * s, out)
        assert len(np.unique(np.rint(out / s))) <= 16 and np.ptp(np.rint(out / s)) <= 15
        assert (np.abs(out - row) <= s / 2 + (np.abs(row) > 32000) * s / 2).all()
