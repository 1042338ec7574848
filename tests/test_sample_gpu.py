"""Whole logits, and sampling from them, against 64 bits and more.

Tokens have to be equal.  The library sums weights as integers in units of 2^-43 of the
largest, the oracle in 64-bit mantissas: a border between two tokens lies at most V 2^-44
of the largest weight off, so a random ``u`` lands between the two borders with a
probability of about 1e-8 a row here.  Logprobs: half a step of fp32, and V 2^-44 of
the largest weight in the sum (below 1e-8 of it)."""

import numpy as np
import pytest
import torch

from oracle.requests import sample_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


def rows(value, b, dtype):
    return value if isinstance(value, torch.Tensor) else torch.full((b,), value, dtype=dtype, device="cuda")


def check(C, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    b = logits.size(0)
    tok, lp = C.sample_logits(logits, u, temperature, top_k, top_p, min_p)
    assert tok.shape == (b,) and tok.dtype == torch.int64 and lp.dtype == torch.float32
    settings = [rows(v, b, t) for v, t in ((temperature, torch.float32), (top_k, torch.int64), (top_p, torch.float32),
                                           (min_p, torch.float32))]
    want, want_lp = sample_ref(logits.cpu().numpy(), u.cpu().numpy(), *(s.cpu().numpy() for s in settings))
    assert tok.tolist() == want.tolist()
    got = lp.cpu().numpy().astype(np.float64)
    with np.errstate(invalid="ignore"):
        near = np.abs(got - want_lp) <= np.abs(want_lp) * 2.0 ** -24 + 1e-8
    assert (near | (got == want_lp)).all(), (got, want_lp)
    again = C.sample_logits(logits, u, *settings)  # numbers and tensors give the same bits
    assert torch.equal(again[0], tok) and torch.equal(again[1], lp)
    return tok, lp


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def heap(b, v, seed, wide=2.5):
    g = gen(seed)
    l = wide * torch.randn(b, v, generator=g, device="cuda")
    if v > 50:
        l.scatter_(1, torch.randint(0, v, (b, 9), generator=g, device="cuda"), 9 + 2 * torch.randn(b, 9, generator=g, device="cuda"))
    return l.half(), torch.rand(b, generator=g, device="cuda")


SETTINGS = [dict(), dict(temperature=0.0), dict(temperature=0.7, top_k=50, top_p=0.9, min_p=0.02), dict(top_k=1),
            dict(top_k=5), dict(top_p=0.5), dict(top_p=0.0), dict(min_p=0.1), dict(min_p=1.0), dict(temperature=2.0, top_p=0.99),
            dict(temperature=1e-3, top_p=0.9), dict(temperature=1e6, top_k=3), dict(temperature=1.5, top_k=700, min_p=1e-4),
            dict(temperature=0.9, top_k=1 << 40, top_p=0.999)]


@pytest.mark.parametrize("b,v", [(1, 1), (2, 2), (3, 7), (4, 100), (2, 1023), (3, 8193), (5, 32003), (1, 151936), (33, 4099)])
@pytest.mark.parametrize("setting", SETTINGS, ids=lambda s: ",".join(f"{k}={v}" for k, v in s.items()) or "all")
def test_against_the_definition(C, b, v, setting):
    logits, u = heap(b, v, seed=b * 1000 + v)
    check(C, logits, u, **setting)


@pytest.mark.parametrize("b,v", [(7, 300001), (1, 524224), (70, 20000), (9, 524223)])
def test_large(C, b, v):
    logits, u = heap(b, v, seed=v)
    check(C, logits, u, temperature=0.9, top_p=0.95)


def test_settings_of_each_row(C):
    b, v = 48, 5003
    logits, u = heap(b, v, seed=1)
    g = gen(2)
    pick = lambda values, t: torch.tensor(values, dtype=t, device="cuda")[torch.randint(0, len(values), (b,), generator=g, device="cuda")]
    for _ in range(4):
        check(C, logits, u, pick([0.0, 0.3, 1.0, 1.0, 4.0, -1.0], torch.float32), pick([0, 0, 1, 7, 300, -5, 10 ** 9], torch.int64),
              pick([1.0, 1.0, 0.9, 0.2, 0.0, 2.0, -1.0], torch.float32), pick([0.0, 0.0, 0.05, 0.5, 1.0, 7.0, -1.0], torch.float32))


@pytest.mark.parametrize("v", [8, 1000, 4096, 70000])
def test_equal_logits_borders_are_exact(C, v):
    """n equal weights: token floor(u n) of the first n, n the least with n >= p k"""
    for value in (0.0, -3.0, 65504.0, -65504.0, 2.0 ** -24):
        logits = torch.full((6, v), value, dtype=torch.float16, device="cuda")
        u = torch.tensor([0.0, 0.25, 0.5, 0.75, 1 - 2.0 ** -24, 0.125], device="cuda")
        for t in (1.0, 0.01, float("inf")):
            tok, lp = C.sample_logits(logits, u, t)
            assert tok.tolist() == [int(np.floor(float(x) * v)) for x in u]
            assert torch.allclose(lp, torch.full_like(lp, -np.log(v)), rtol=2.0 ** -23, atol=0)
        for k, p in ((v // 2, 0.5), (v, 0.25), (0, 0.75), (v // 2 + 1, 1.0), (3, 0.5)):
            kk = k or v
            n = kk if p >= 1 else int(np.ceil(p * kk))
            tok, _ = C.sample_logits(logits, u, 1.0, k, p)
            assert tok.tolist() == [int(np.floor(float(x) * n)) for x in u]


def test_equal_values_go_by_index(C):
    v = 20011
    logits = torch.full((1, v), -4.0, dtype=torch.float16, device="cuda")
    at = torch.randperm(v, generator=gen(5), device="cuda")[:300].sort().values
    logits[0, at] = 2.0
    logits[0, at[::2]] = 2.0
    for j in (0, 1, 150, 298, 299):
        u = torch.tensor([(j + 0.5) / 300], device="cuda")
        tok, _ = C.sample_logits(logits, u, 0.05, 300)
        assert tok.item() == at[j].item()
    assert C.sample_logits(logits, torch.tensor([0.9], device="cuda"), 0.0)[0].item() == at[0].item()
    logits.zero_()
    logits[0, 1::2] = -0.0  # the two zeros are one value
    assert C.sample_logits(logits, torch.tensor([0.5], device="cuda"))[0].item() == int(0.5 * v)


def test_masked_rows_infinities_and_nan(C):
    inf, nan = float("inf"), float("nan")
    v = 9001
    logits, u = heap(10, v, seed=3)
    logits[0] = -inf
    logits[1] = nan
    logits[2, ::2], logits[2, 1::2] = nan, -inf
    logits[3] = -inf
    logits[3, 8999] = -65504.0  # one token left
    logits[4, 5:] = -inf
    logits[5, ::3] = nan
    logits[6, [7, 70, 7000]] = inf
    logits[7] = inf
    logits[8] = -65504.0  # masked by the lowest value: all alike
    logits[9, 100:] = -65504.0
    tok, lp = C.sample_logits(logits, u)
    assert tok[:4].tolist() == [-1, -1, -1, 8999] and lp[:3].tolist() == [-inf] * 3 and lp[3].item() == 0.0
    for setting in SETTINGS:
        check(C, logits, u, **setting)
    tok, _ = C.sample_logits(logits, torch.full((10,), 0.999, device="cuda"))
    assert tok[6].item() == 7000 and tok[9].item() < 100


def test_random_numbers_outside_the_range(C):
    logits, _ = heap(8, 500, seed=6)
    u = torch.tensor([-1.0, float("nan"), -float("inf"), 0.0, 1.0, 2.0, float("inf"), 1 - 2.0 ** -24], device="cuda")
    same = logits[:1].expand(8, -1).contiguous()
    tok, _ = C.sample_logits(same, u, 1.0, 10)
    order = torch.sort(same[0].float(), descending=True, stable=True).indices
    assert tok[:4].tolist() == [order[0].item()] * 4 and tok[4:7].tolist() == [order[9].item()] * 3


def test_settings_that_are_no_limits(C):
    logits, u = heap(4, 3000, seed=12)
    nan, inf = float("nan"), float("inf")
    want = C.sample_logits(logits, u)
    for p, m in ((nan, 0.0), (1.0, nan), (inf, -inf), (1.5, -2.0)):
        for f in (lambda v: v, lambda v: torch.full((4,), v, device="cuda")):
            got = C.sample_logits(logits, u, 1.0, -7, f(p), f(m))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    greedy = C.sample_logits(logits, u, 0.0)
    for t in (nan, -1.0, -inf):
        got = C.sample_logits(logits, u, t, 50, 0.9, 0.1)
        assert torch.equal(got[0], greedy[0]) and torch.equal(got[1], greedy[1]) and (got[1] == 0).all()
    assert greedy[0].tolist() == logits.float().argmax(-1).tolist()


def test_frequencies(C):
    """evenly spaced random numbers meet each token in proportion to its weight, to within one number"""
    n = 4096
    logits = torch.tensor([[1.0, 0.0, -1.0, 2.0, 0.5]], dtype=torch.float16, device="cuda")
    u = (torch.arange(n, device="cuda") + 0.5) / n
    tok, _ = C.sample_logits(logits.expand(n, -1).contiguous(), u, 0.8)
    share = torch.bincount(tok, minlength=5).double().cpu() / n
    want = torch.softmax(logits[0].double().cpu() / 0.800000011920929, 0)
    assert (share - want).abs().max() <= 1.0 / n + 1e-9


def test_unaligned_rows_streams_and_captured_graph(C):
    flat, u = heap(1, 40000, seed=8)
    flat = flat[0]
    u = torch.rand(3, generator=gen(1), device="cuda")
    for shift in range(1, 9):  # a base that is aligned to nothing but its type
        check(C, flat[shift:shift + 3 * 12001].view(3, 12001), u, top_p=0.9)
    logits, u = heap(4, 20000, seed=9)
    want = C.sample_logits(logits, u, 0.8, 0, 0.9)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = C.sample_logits(logits, u, 0.8, 0, 0.9)
    s.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graph, t, k = torch.cuda.CUDAGraph(), torch.full((4,), 0.8, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda")
    held, hu = logits.clone(), u.clone()
    with torch.cuda.graph(graph):
        tok, lp = C.sample_logits(held, hu, t, k, 0.9)
    for i in range(4):
        hu.copy_(torch.rand(4, generator=gen(20 + i), device="cuda"))
        t.fill_(0.5 * i)
        k.fill_(i * 10)
        held.copy_(logits.roll(i * 31, 1))
        graph.replay()
        want = C.sample_logits(held, hu, t, k, 0.9)
        assert torch.equal(tok, want[0]) and torch.equal(lp, want[1])


def test_nothing_and_refusals(C):
    f = lambda *s: torch.zeros(*s, device="cuda")
    tok, lp = C.sample_logits(f(0, 5).half(), f(0))
    assert tok.shape == (0,) and lp.shape == (0,)
    l, u = f(2, 5).half(), f(2)
    for args, msg in [((l.float(), u), "float16"), ((l[0], u), r"\[B, V\]"), ((l.t(), u), "contiguous"), ((l, u.double()), "u must"),
                      ((l, f(3)), "u must"), ((l, u, u.double()), "temperature"), ((l, u, 1.0, u), "top_k"),
                      ((l, u, 1.0, 0, f(3)), "top_p"), ((l, u, 1.0, 0, 1.0, u.half()), "min_p"), ((l, u.cpu()), "CUDA"),
                      ((f(1, 524232).half(), f(1)), "524224"), ((f(2, 0).half(), u), "sizes")]:
        with pytest.raises(RuntimeError, match=msg):
            C.sample_logits(*args)
    for bad in (("hot",), (1.0, 0.5)):
        with pytest.raises(TypeError):
            C.sample_logits(l, u, *bad)


# ------------------------------------------------------------------- logits --
@pytest.mark.parametrize("b,h,v", [(1, 64, 8), (1, 4096, 151936), (3, 128, 520), (16, 512, 1000), (17, 192, 2056), (32, 256, 4096),
                                   (33, 64, 264), (70, 128, 1024)])
def test_logits(C, b, h, v):
    """half a step of fp16, and a step of fp32 (2^-23, towards zero) for each addition relative to the terms' magnitudes"""
    g = gen(b + v)
    x = torch.randn(b, h, generator=g, device="cuda").half()
    w = (torch.randn(h, v, generator=g, device="cuda") * 4 / h ** 0.5).half()
    got = C.lm_head_logits(x, w)
    assert got.shape == (b, v) and got.dtype == torch.float16
    for part in range(0, v, 16384):
        ww = w[:, part:part + 16384].double()
        ref, size = x.double() @ ww, x.double().abs() @ ww.abs()
        allowed = ref.abs() * 2.0 ** -11 + 2.0 ** -25 + h * 2.0 ** -23 * size
        assert ((got[:, part:part + 16384].double() - ref).abs() <= allowed).all()
    if b <= 32:  # the greedy head takes the maximum of these values
        val, idx = C.lm_head_argmax(x, w)
        assert torch.equal(val, got.float().amax(-1))
        assert torch.equal(idx, torch.sort(got.float(), dim=-1, descending=True, stable=True).indices[:, 0])


def test_logits_refusals(C):
    f = lambda *s: torch.zeros(*s, dtype=torch.float16, device="cuda")
    assert C.lm_head_logits(f(0, 64), f(64, 8)).shape == (0, 8)
    for args, msg in [((f(2, 64).float(), f(64, 8)), "float16"), ((f(64), f(64, 8)), r"\[B, H\]"), ((f(2, 64), f(128, 8)), r"\[H, V\]"),
                      ((f(2, 96), f(96, 8)), "hidden"), ((f(2, 64), f(64, 12)), "vocab"), ((f(2, 64), f(8, 64).t()), "contiguous")]:
        with pytest.raises(RuntimeError, match=msg):
            C.lm_head_logits(*args)


def test_a_run_as_a_served_batch_makes_it(C):
    """projection with adapters -> logits -> tokens, each step checked on the values that it got"""
    from tests.test_multi_lora_gpu import check as check_lora, inputs, quantised
    w = quantised(256, 256, 128, seed=1)
    d = inputs(12, None, 256, (256,), 16, 4, seed=6)
    base = C.w4a16_gemv(d["x"], *w)
    h = C.w4a16_multi_lora_gemv(d["x"], *w, d["lora_A"], d["lora_B"], d["adapters"], d["scales"])
    check_lora(h, {**d, "y": base}, (256,))
    head = (torch.randn(256, 5000, generator=gen(3), device="cuda") * 0.5).half()
    logits = C.lm_head_logits(h, head)
    assert torch.equal(logits.float().amax(-1), C.lm_head_argmax(h, head)[0])
    u = torch.rand(12, generator=gen(4), device="cuda")
    check(C, logits, u, temperature=torch.linspace(0, 2, 12, device="cuda"), top_k=40, top_p=0.95)


@pytest.mark.parametrize("b,v", [(1, 1000), (16, 40000), (40, 3001)])
@pytest.mark.parametrize("top_k", [0, 3, 200])
def test_subnormal_logits_many_alike(C, b, v, top_k):
    """logits of a few steps of 2^-24, zeros of both signs among them: all weights near one, the order by index counts"""
    g = torch.Generator(device="cuda").manual_seed(v + top_k)
    steps = torch.randint(-20, 21, (b, v), generator=g, device="cuda")
    logits = (steps * 2.0 ** -24).half()
    logits[steps == 0] = torch.where(torch.rand(int((steps == 0).sum()), generator=g, device="cuda") < 0.5, 0.0, -0.0).half()
    u = torch.rand(b, generator=g, device="cuda")
    check(C, logits, u, 1e-6, top_k)
    greedy = C.sample_logits(logits, u, 0.0)[0]
    assert torch.equal(greedy, logits.float().argmax(1))
