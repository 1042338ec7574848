"""Infinities in an adapter's B: a row's output is infinite or NaN where the definition says so, for
sequences of few tokens and for prompts alike (the latter hold x A as the sum of two fp16 numbers).

x and A are such that every x A is exact in 32 bits: its zeros and signs are those of the definition.
Tolerance of the finite outputs: that of the operator's other tests."""

import numpy as np
import pytest
import torch

from oracle.requests import multi_lora_ref

pytestmark = pytest.mark.gpu
INF, NAN = float("inf"), float("nan")


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


def whole(lo, hi, shape, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.randint(lo, hi + 1, shape, generator=g, device="cuda").half()


def check(C, d, splits):
    names = ("y", "x", "lora_A", "lora_B", "adapters", "scales")
    with np.errstate(invalid="ignore", over="ignore"):
        ref, _ = multi_lora_ref(*(d[n].cpu().numpy() for n in names), splits)
    finite_B = {**d, "lora_B": torch.where(d["lora_B"].isfinite(), d["lora_B"], 0)}
    with np.errstate(invalid="ignore", over="ignore"):
        _, bound = multi_lora_ref(*(finite_B[n].cpu().numpy() for n in names), splits)
    got = C.multi_lora_add(**d, splits=splits).cpu().numpy().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(ref))
    infinite = np.isinf(ref)
    assert infinite.any() and np.array_equal(got[infinite], ref[infinite])
    ok = np.isfinite(ref)
    assert ok.any()
    steps = d["x"].size(-1) + d["lora_B"].size(1) + 8
    allowed = np.abs(ref[ok]) * 2.0 ** -11 + 2.0 ** -25 + steps * 2.0 ** -23 * bound[ok]
    assert (np.abs(got[ok] - ref[ok]) <= allowed).all()
    return got


SHAPES = [(4, None), (3, 8), (3, 9), (2, 70), (3, 500)]  # few tokens, chunks of 32 rows, chunks of 64


@pytest.mark.parametrize("r,splits", [(8, (136, 64)), (16, (128, 128)), (24, (264,)), (64, (72, 200)), (80, (136,)), (128, (64, 96))])
@pytest.mark.parametrize("b,t", SHAPES)
def test_infinite_and_nan_values_of_b(C, b, t, r, splits):
    lead, parts = ((b,) if t is None else (b, t)), len(splits)
    d = dict(y=whole(-8, 8, (*lead, sum(splits)), 1), x=whole(-2, 2, (*lead, 72), 2),
             lora_A=whole(-3, 3, (3, 72, r * parts), 3) / 16, lora_B=whole(-6, 6, (3, r, sum(splits)), 4) / 8,
             adapters=torch.arange(b, device="cuda") % 2, scales=torch.tensor([0.75, 1.5, 1.0], device="cuda"))
    d["x"].view(b, -1, 72)[0, -1] = 0  # a row whose x A is zero: NaN beside the infinities
    clean = C.multi_lora_add(**d, splits=splits)
    B = d["lora_B"]
    at = [(0, 3), (1 % r, 5), (r - 1, 5), (r // 2, 33), (r - 1, sum(splits) - 1), (2, 63), (5, 64)]
    for i, (j, c) in enumerate(at):
        B[0, j, c] = INF if i % 2 else -INF
    B[1, 4, 10], B[1, 4, 11], B[1, 3, 11] = NAN, INF, -INF
    B[2, 0, 0] = INF  # of an adapter that nobody has
    got = check(C, d, splits)
    same = np.ones(got.shape, bool)  # columns without any keep their bits
    for i, a in enumerate(d["adapters"].tolist()):
        same[i][..., ~np.isfinite(B[a].cpu().numpy()).all(0)] = False
    assert np.array_equal(got[same], clean.cpu().numpy().astype(np.float64)[same])


@pytest.mark.parametrize("r", [16, 64, 80])
@pytest.mark.parametrize("b,t", SHAPES)
def test_small_low_rank_values_beside_large_ones(C, b, t, r):
    """x A of one rank 2^40 times that of another, whose B is infinite: the small one's sign counts"""
    lead = (b,) if t is None else (b, t)
    d = dict(y=whole(-8, 8, (*lead, 96), 1), x=whole(-2, 2, (*lead, 72), 2), lora_A=whole(-1, 1, (1, 72, r), 3) * 2.0 ** 15,
             lora_B=torch.zeros(1, r, 96, dtype=torch.float16, device="cuda"), adapters=torch.zeros(b, dtype=torch.int64, device="cuda"),
             scales=torch.ones(1, device="cuda"))
    d["lora_A"][0, :, 5] = whole(-2, 2, (72,), 4) * 2.0 ** -24
    d["lora_B"][0, 5, ::7], d["lora_B"][0, 5, 3::7] = INF, -INF
    check(C, d, (96,))


@pytest.mark.parametrize("r", [16, 64, 80])
@pytest.mark.parametrize("b,t", SHAPES)
def test_infinite_values_of_a_and_of_b(C, b, t, r):
    """rows that hold an infinity in x A beside finite values, both before infinities of B"""
    lead = (b,) if t is None else (b, t)
    d = dict(y=whole(-8, 8, (*lead, 96), 1), x=whole(1, 2, (*lead, 72), 2), lora_A=whole(-3, 3, (1, 72, r), 3) / 16,
             lora_B=whole(1, 6, (1, r, 96), 4) / 8, adapters=torch.zeros(b, dtype=torch.int64, device="cuda"),
             scales=torch.ones(1, device="cuda"))
    d["lora_A"][0, 7, 2], d["lora_A"][0, :, 9] = INF, 0.125  # x A: infinite at rank 2, positive at rank 9
    d["x"].view(b, -1, 72)[-1, 0, 7] = 0  # NaN at rank 2
    d["lora_B"][0, 9, ::5], d["lora_B"][0, 9, 2::5] = INF, -INF  # inf + inf, inf - inf
    d["lora_B"][0, 2, 1::5] = -INF
    d["lora_B"][0, 2, 3::5], d["lora_B"][0, 9, 3::5] = -1, -INF
    with np.errstate(invalid="ignore"):
        ref, _ = multi_lora_ref(*(d[n].cpu().numpy() for n in ("y", "x", "lora_A", "lora_B", "adapters", "scales")))
    got = C.multi_lora_add(**d).cpu().numpy().astype(np.float64)
    assert np.isinf(ref).any() and np.isnan(ref).any() and np.array_equal(got, ref, equal_nan=True)
