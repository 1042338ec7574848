"""Greedy head: rows without a finite logit give an index inside the vocabulary (a decoder embeds it next)."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b", [1, 9, 32])
def test_rows_of_nan_and_infinities(b):
    from qextract_infer_b200 import _C
    h = torch.ones(b, 128, device="cuda").half()
    w = torch.randn(128, 1000, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda").half()
    plain = (h.float() @ w.float()).half()
    h[0, 5] = float("nan")
    val, idx = _C.lm_head_argmax(h, w, 300)
    assert idx[0].item() == 300 and (idx[1:] - 300).tolist() == plain[1:].argmax(1).tolist()
    w[:, :] = -60000.0  # sums below fp16's range: -inf everywhere
    val, idx = _C.lm_head_argmax(torch.ones(b, 128, device="cuda").half(), w, 300)
    assert idx.tolist() == [300] * b and (val == float("-inf")).all()
    w[:, 7] = float("nan")  # NaN is never the largest
    w[:, 900] = 1.0
    val, idx = _C.lm_head_argmax(torch.ones(b, 128, device="cuda").half(), w, 300)
    assert idx.tolist() == [1200] * b and (val == 128).all()
    w[:, 901] = 60000.0
    val, idx = _C.lm_head_argmax(torch.ones(b, 128, device="cuda").half(), w, 300)
    assert idx.tolist() == [1201] * b and (val == float("inf")).all()
