"""Refusals of the adapters', the logits' and the sampler's entry points at the C ABI
(before any launch: no GPU) and in Python, and the sampler's oracle on cases done by hand."""

import ctypes

import numpy as np
import pytest

from oracle.requests import multi_lora_ref, sample_ref
from qextract_infer_b200 import _lib

P = 1 << 20  # well-aligned addresses far apart that are never read
Y, X, A, B, IDS, SCALES, OUT = (i << 32 for i in range(1, 8))


def _lora(lib, y=Y, x=X, a=A, b=B, ids=IDS, scales=SCALES, out=OUT, batch=2, tokens=3, k=64, n=64, rank=16, adapters=4,
          splits=None):
    arr = (ctypes.c_int * len(splits))(*splits) if splits else None
    return lib.qx_multi_lora_add(y, x, a, b, ids, scales, out, batch, tokens, k, n, rank, adapters, arr,
                                 len(splits) if splits else 0, None)


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=-1), "bad sizes"), (dict(tokens=-1), "bad sizes"), (dict(k=0), "bad sizes"), (dict(n=0), "bad sizes"),
    (dict(adapters=-1), "bad sizes"), (dict(k=60), "multiples of 8"), (dict(k=(1 << 30) + 8), "2^30"), (dict(n=60), "multiples of 8"),
    (dict(rank=4), "rank"), (dict(rank=12), "rank"), (dict(rank=264), "rank"), (dict(rank=72, splits=[16] * 4), "rank"),
    (dict(splits=[8] * 5), "column blocks"), (dict(splits=[32, 36]), "columns"), (dict(splits=[64, 0]), "columns"),
    (dict(splits=[32, 24]), "cover"), (dict(splits=[64, 8]), "exceed"), (dict(splits=[-64, 128]), "columns"),
    (dict(batch=1 << 14, tokens=1 << 20), "too many"), (dict(batch=32769), "32768"), (dict(y=None), "null"), (dict(x=None), "null"),
    (dict(a=None), "null"), (dict(b=None), "null"), (dict(ids=None), "null"), (dict(scales=None), "null"),
    (dict(out=None), "null"), (dict(y=Y + 8), "aligned"), (dict(x=X + 2), "aligned"), (dict(a=A + 8), "aligned"),
    (dict(b=B + 8), "aligned"), (dict(out=OUT + 8), "aligned"), (dict(ids=IDS + 4), "aligned"),
    (dict(scales=SCALES + 2), "aligned"), (dict(out=Y + 16), "overlap"), (dict(out=X), "overlap"),
    (dict(out=A + 16), "overlap"), (dict(out=B), "overlap"), (dict(out=Y - 16), "overlap")])
def test_multi_lora_arguments(bad, msg):
    lib = _lib.load()
    assert _lora(lib, **bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()


def test_nothing_to_do():
    lib = _lib.load()
    assert _lora(lib, batch=0) == 0 and _lora(lib, tokens=0) == 0 and _lora(lib, batch=0, y=None, out=None) == 0
    assert lib.qx_lm_head_logits(P, P, P, 0, 64, 8, None) == 0
    assert _sample(lib, batch=0) == 0


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=-1), "batch"), (dict(hidden=0), "hidden"), (dict(hidden=96), "hidden"), (dict(vocab=0), "vocab"),
    (dict(vocab=12), "vocab"), (dict(h=None), "null"), (dict(w=None), "null"), (dict(out=None), "null"),
    (dict(h=P + 8), "aligned"), (dict(w=P + 2), "aligned"), (dict(out=P + 2), "aligned")])
def test_logits_arguments(bad, msg):
    lib = _lib.load()

    def call(h=P, w=P, out=P, batch=2, hidden=128, vocab=64):
        return lib.qx_lm_head_logits(h, w, out, batch, hidden, vocab, None)

    assert call(**bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()


def _sample(lib, logits=P, u=P, t=None, k=None, p=None, m=None, tokens=P, logprobs=P, batch=2, vocab=100):
    f = ctypes.c_float
    return lib.qx_sample_logits(logits, u, t, k, p, m, f(1), 0, f(1), f(0), tokens, logprobs, batch, vocab, None)


@pytest.mark.parametrize("bad,msg", [
    (dict(batch=-1), "bad sizes"), (dict(vocab=0), "bad sizes"), (dict(vocab=524225), "524224"),
    (dict(batch=1 << 30), "too large"), (dict(logits=None), "null"), (dict(u=None), "null"), (dict(tokens=None), "null"),
    (dict(logprobs=None), "null"), (dict(logits=P + 1), "aligned"), (dict(u=P + 2), "aligned"), (dict(t=P + 2), "aligned"),
    (dict(k=P + 4), "aligned"), (dict(p=P + 1), "aligned"), (dict(m=P + 2), "aligned"), (dict(tokens=P + 4), "aligned"),
    (dict(logprobs=P + 2), "aligned")])
def test_sample_arguments(bad, msg):
    lib = _lib.load()
    assert _sample(lib, **bad) == -1
    assert msg in _lib.last_error(), _lib.last_error()


def test_python_ops_reject_cpu_tensors():
    import torch
    from qextract_infer_b200 import _C
    y, x = torch.zeros(2, 64, dtype=torch.float16), torch.zeros(2, 32, dtype=torch.float16)
    a, b = torch.zeros(3, 32, 8, dtype=torch.float16), torch.zeros(3, 8, 64, dtype=torch.float16)
    for call in (lambda: _C.multi_lora_add(y, x, a, b, torch.zeros(2, dtype=torch.int64), torch.zeros(3)),
                 lambda: _C.lm_head_logits(x, y), lambda: _C.sample_logits(y, torch.zeros(2)),
                 lambda: _C.w4a16_multi_lora_gemv(x, y, y, y, a, b, torch.zeros(2, dtype=torch.int64), torch.zeros(3))):
        with pytest.raises(RuntimeError, match="CUDA tensor"):
            call()
    with pytest.raises(RuntimeError, match=r"\[B, K\]"):
        _C.w4a16_multi_lora_gemv(x[0], y, y, y, a, b, torch.zeros(1, dtype=torch.int64), torch.zeros(3))


def test_multi_lora_oracle_by_hand():
    x = np.array([[1.0, 2.0], [3.0, 4.0], [5.0, 6.0]])
    A = np.array([[[1.0, 0.0], [0.0, 1.0]]])  # two blocks of rank 1
    B = np.array([[[10.0, 100.0]]])
    out, bound = multi_lora_ref(np.ones((3, 2)), x, A, B, [0, -1, 1], [2.0], splits=[1, 1])
    assert out.tolist() == [[21.0, 401.0], [1.0, 1.0], [1.0, 1.0]]
    assert bound.tolist() == [[21.0, 401.0], [1.0, 1.0], [1.0, 1.0]]


def test_sample_oracle_by_hand():
    ln2 = np.log(2.0)
    row = np.array([0.0, 1.0, 1.0, -np.inf, np.nan, 0.0], dtype=np.float16)  # order 1, 2, 0, 5

    def one(u, t=1.0, k=0, p=1.0, m=0.0, row=row):
        tok, lp = sample_ref(row[None], *([np.float64(v)] for v in (u, t)), [k], [p], [m])
        return int(tok[0]), float(lp[0])

    # weights at T = 1 / ln 2: 1, 1, 1/2, 1/2 (sum 3)
    t = 1 / ln2
    assert [one(u, t)[0] for u in (0.0, 0.32, 0.34, 0.66, 0.68, 0.82, 0.84, 0.9999)] == [1, 1, 2, 2, 0, 0, 5, 5]
    assert abs(one(0.7, t)[1] - np.log(1 / 6)) < 1e-12
    assert one(0.99, t, k=3)[0] == 0 and one(0.99, t, p=0.5)[0] == 2 and one(0.99, t, m=0.6)[0] == 2
    assert one(0.99, t, p=0.0)[0] == 1 and one(0.99, 0.0) == (1, 0.0)
    assert one(0.99, row=np.array([np.nan, -np.inf], dtype=np.float16)) == (-1, -np.inf)
    assert one(0.6, row=np.array([0.0, np.inf, np.inf], dtype=np.float16))[0] == 2
