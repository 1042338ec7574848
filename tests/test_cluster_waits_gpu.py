"""Messages within a cluster that do not come in time: the call ends, the device error word says so, tokens are -1 and an
addition's output is unwritten where it is not right, and the calls after it are as ever.  Waits are made to run
out by `qx_test_waits` (they give up without a look; nothing is dropped or overwritten)."""

import ctypes

import pytest
import torch

pytestmark = pytest.mark.gpu
TIMEOUT = 1


@pytest.fixture()
def lib():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _lib
    lib = _lib.load()
    assert error(lib) == 0
    yield lib
    assert lib.qx_test_waits(0, -1) == 0
    torch.cuda.synchronize()
    error(lib)


def error(lib):
    code = ctypes.c_uint(0)
    assert lib.qx_get_device_error(ctypes.byref(code), 1) == 0
    return code.value


def test_arguments(lib):
    assert lib.qx_test_waits(256, -1) < 0 and lib.qx_test_waits(1, 16) < 0 and lib.qx_test_waits(1, -2) < 0


@pytest.mark.parametrize("exchange", range(5))
@pytest.mark.parametrize("cta", [-1, 0, 1, 3])
@pytest.mark.parametrize("b,v", [(1, 20000), (12, 20000), (40, 3001)])  # 16, 8 and 4 CTAs a row
def test_sampling(lib, b, v, exchange, cta):
    from qextract_infer_b200 import _C
    g = torch.Generator(device="cuda").manual_seed(b)
    logits, u = (3 * torch.randn(b, v, generator=g, device="cuda")).half(), torch.rand(b, generator=g, device="cuda")
    limits = (0.9, 300, 0.9, 0.001)
    want = _C.sample_logits(logits, u, *limits)
    assert lib.qx_test_waits(1 << exchange, cta) == 0
    got = _C.sample_logits(logits, u, *limits)
    assert lib.qx_test_waits(0, -1) == 0
    torch.cuda.synchronize()
    assert error(lib) == TIMEOUT
    assert (got[0] == -1).all() and (got[1] == float("-inf")).all()
    again = _C.sample_logits(logits, u, *limits)
    assert torch.equal(again[0], want[0]) and torch.equal(again[1], want[1])
    assert error(lib) == 0


def test_sampling_without_that_exchange(lib):
    """no limits: nobody waits for the k-th token's border"""
    from qextract_infer_b200 import _C
    logits, u = torch.randn(9, 5000, generator=torch.Generator().manual_seed(1)).half().cuda(), torch.full((9,), 0.4, device="cuda")
    want = _C.sample_logits(logits, u)
    assert lib.qx_test_waits(1 << 2 | 1 << 3, -1) == 0
    got = _C.sample_logits(logits, u)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    assert error(lib) == 0


# few-token kernel (one exchange), and chunks of 32 and 64 rows (two), more than 64 ranks
@pytest.mark.parametrize("b,t,r,exchange", [(3, None, 16, 0), (20, None, 16, 0), (2, 40, 16, 0), (2, 40, 16, 1), (2, 700, 64, 0),
                                            (2, 700, 64, 1), (2, 130, 128, 0), (2, 130, 128, 1)])
@pytest.mark.parametrize("cta", [-1, 0, 5])
def test_adapters(lib, b, t, r, exchange, cta):
    from qextract_infer_b200 import _C
    g = torch.Generator(device="cuda").manual_seed(b)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda").half()
    lead = (b,) if t is None else (b, t)
    ids = torch.arange(b, device="cuda") % 3 - 1
    d = dict(y=normal(*lead, 1024), x=normal(*lead, 256), lora_A=normal(2, 256, r), lora_B=normal(2, r, 1024), adapters=ids,
             scales=torch.ones(2, device="cuda"))
    want = _C.multi_lora_add(**d)
    out = torch.full_like(want, 123.0)
    assert lib.qx_test_waits(1 << exchange, cta) == 0
    _C.multi_lora_add(**d, out=out)
    assert lib.qx_test_waits(0, -1) == 0
    torch.cuda.synchronize()
    assert error(lib) == TIMEOUT
    unwritten = out == 123.0
    assert torch.equal(out[~unwritten], want[~unwritten]) and torch.equal(out[ids < 0], want[ids < 0])
    one_ctas_part = cta >= 0 and (t is None or exchange == 1)  # else all of the cluster miss something
    share = unwritten[ids >= 0].float().mean().item()
    assert abs(share - (1 / 8 if one_ctas_part else 1)) < 0.01
    assert torch.equal(_C.multi_lora_add(**d, out=out), want)
    assert error(lib) == 0
