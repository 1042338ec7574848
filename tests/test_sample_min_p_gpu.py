"""Sampling with min_p close to 1 and high temperatures: the logits that a slice need not count are found from
temperature x ln(1 / min_p), whose factors may be tiny and huge.  Against the definition; tokens are equal."""

import numpy as np
import pytest
import torch

from oracle.requests import sample_ref

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("u", [0.0, 0.5, 1 - 2.0 ** -24])
@pytest.mark.parametrize("down", [1.004, 5.004, 8.004])
def test_min_p_near_one_at_high_temperatures(u, down):
    """the logits of a row are 8, 8 - 2^-7, ...; those within about `down` of 8 are heavy enough; its end lies between two
    of them, at least 0.003 from either: weights there are 0.003 / temperature > 2e-11 off min_p, which 64 bits tell"""
    from qextract_infer_b200 import _C
    steps = np.concatenate([np.arange(1, 40), np.arange(40, 600, 7)])
    min_p = (1 - steps * 2.0 ** -24).astype(np.float32)
    temperature = (down / -np.log(min_p.astype(np.float64))).astype(np.float32)
    b = len(steps)
    row = (8 - torch.arange(0, 3000) * 2.0 ** -7).half()
    logits = row[torch.randperm(3000, generator=torch.Generator().manual_seed(1))].expand(b, 3000).contiguous().cuda()
    uu = torch.full((b,), u)
    tok, lp = _C.sample_logits(logits, uu.cuda(), torch.from_numpy(temperature).cuda(), 0, 1.0, torch.from_numpy(min_p).cuda())
    want, want_lp = sample_ref(logits.cpu().numpy(), uu.numpy(), temperature, np.zeros(b, np.int64), np.ones(b, np.float32), min_p)
    assert tok.tolist() == want.tolist()
    # half a step of fp32, and the sum's integers: 3000 x 2^-44
    assert (np.abs(lp.cpu().numpy() - want_lp) <= np.abs(want_lp) * 2.0 ** -24 + 1e-9).all()
