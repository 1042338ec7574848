"""Low-rank adapters of many requests beside a shared projection against 64 bits.

Tolerance of an output: half a step of fp16 (2^-11 of the value, 2^-25 below its
normal range) for the one rounding, and 2^-23 for each of the K + r + 8 fp32 additions
and products on a term's way, relative to the sum of the terms' magnitudes (the worst
case of a sum; rounding towards zero, as a matrix instruction may add, is a whole step
of 2^-23)."""

import numpy as np
import pytest
import torch

from oracle.requests import multi_lora_ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


def inputs(b, t, k, splits, r, n, seed=0, wide=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    normal = lambda *s: torch.randn(*s, generator=g, device="cuda")
    lead = (b,) if t is None else (b, t)
    return dict(y=normal(*lead, sum(splits)).half(), x=(wide * normal(*lead, k)).half(),
                lora_A=(normal(n, k, r * len(splits)) / k ** 0.5).half(), lora_B=(normal(n, r, sum(splits)) * 0.3).half(),
                adapters=torch.randint(-1, n + 1, (b,), generator=g, device="cuda"),
                scales=0.5 + torch.rand(n, generator=g, device="cuda"))


def check(out, d, splits):
    ref, bound = multi_lora_ref(*(d[n].cpu().numpy() for n in ("y", "x", "lora_A", "lora_B", "adapters", "scales")), splits)
    got = out.cpu().numpy().astype(np.float64)
    steps = d["x"].size(-1) + d["lora_B"].size(1) + 8
    allowed = np.abs(ref) * 2.0 ** -11 + 2.0 ** -25 + steps * 2.0 ** -23 * bound
    bad = ~(np.abs(got - ref) <= allowed)
    assert not bad.any(), (bad.sum(), np.argwhere(bad)[:3], got[bad][:3], ref[bad][:3])
    none = ((d["adapters"] < 0) | (d["adapters"] >= d["scales"].numel())).cpu()
    assert torch.equal(out.cpu()[none], d["y"].cpu()[none])


CASES = [  # b, t, k, splits, r, n
    (1, None, 64, (64,), 8, 1), (1, 1, 8, (8,), 8, 1), (3, None, 256, (256,), 16, 2), (7, 1, 520, (1000,), 24, 3),
    (32, None, 512, (512, 128, 128), 16, 40), (33, None, 328, (264, 264), 32, 2), (9, None, 1032, (40, 8, 16, 72), 64, 5),
    (5, 2, 136, (136,), 48, 2), (4, 3, 256, (512,), 16, 2), (2, 7, 400, (24, 1000), 8, 1), (64, 1, 64, (32,), 128, 3),
    (3, 8, 256, (256,), 16, 2), (2, 9, 256, (256,), 16, 3), (1, 64, 512, (512,), 16, 1), (3, 65, 264, (136, 72), 40, 2),
    (2, 130, 1024, (768,), 64, 2), (1, 301, 200, (1032,), 32, 1), (6, 33, 128, (96, 96, 96), 80, 2),
    (1, 513, 96, (2048,), 256, 1), (70, 17, 72, (88,), 8, 3), (2, 128, 4096, (520,), 8, 2), (200, None, 64, (64,), 16, 3),
    (1, None, 12288, (264,), 64, 1), (300, 1, 40, (16,), 8, 300)]


@pytest.mark.parametrize("case", CASES, ids=lambda c: "-".join(str(v) for v in c).replace(" ", ""))
def test_against_64_bits(C, case):
    b, t, k, splits, r, n = case
    d = inputs(*case, seed=b * 31 + k)
    y0 = d["y"].clone()
    out = C.multi_lora_add(**d, splits=splits)
    check(out, d, splits)
    assert torch.equal(d["y"], y0)
    if len(splits) == 1:
        assert torch.equal(C.multi_lora_add(**d), out)
    into = C.multi_lora_add(**{**d, "y": y0}, splits=splits, out=y0)  # in place: the same bits
    assert into.data_ptr() == y0.data_ptr() and torch.equal(y0, out)


@pytest.mark.parametrize("b,t", [(40, None), (5, 3), (3, 40), (2, 200)])
@pytest.mark.parametrize("ids", ["same", "none", "distinct", "far"])
def test_who_has_what(C, b, t, ids):
    d = inputs(b, t, 264, (72, 200), 16, 40, seed=b)
    d["adapters"] = {"same": torch.full((b,), 17), "none": torch.full((b,), -1), "distinct": torch.arange(b),
                     "far": torch.tensor([1 << 40, -(1 << 62), 39, 40, -1][:b] + [39 - i % 3 for i in range(b - 5)])}[ids].cuda()
    check(C.multi_lora_add(**d, splits=(72, 200)), d, (72, 200))


def test_a_row_does_not_depend_on_its_neighbours(C):
    """the same sequence alone and in batches, with the same and other adapters around it"""
    for t in (None, 20):
        d = inputs(24, t, 512, (512,), 16, 3, seed=5)
        d["adapters"] = torch.arange(24, device="cuda") % 3
        whole = C.multi_lora_add(**d)
        for i in (0, 7, 23):
            one = {n: v[i:i + 1].contiguous() if n in ("x", "y", "adapters") else v for n, v in d.items()}
            assert torch.equal(C.multi_lora_add(**one)[0], whole[i])


def test_no_adapters_at_all(C):
    d = inputs(3, None, 64, (64,), 8, 1)
    d.update(lora_A=d["lora_A"][:0], lora_B=d["lora_B"][:0], scales=d["scales"][:0])
    assert torch.equal(C.multi_lora_add(**d), d["y"])
    d = inputs(0, None, 64, (64,), 8, 1)
    assert C.multi_lora_add(**d).shape == (0, 64)
    d = inputs(2, 0, 64, (64,), 8, 1)
    assert C.multi_lora_add(**d).shape == (2, 0, 64)


@pytest.mark.parametrize("t", [None, 40])
def test_large_and_small_values(C, t):
    """x A beyond fp16's range, and far below it: the low-rank values keep 32-bit range and precision"""
    for wide, back in ((1e4, 2.0 ** -14), (2.0 ** -12, 1.0)):  # x stays finite (3e4 made it infinite, and the reference NaN)
        d = inputs(3, t, 512, (256,), 16, 2, seed=9, wide=wide)
        d["adapters"] = torch.tensor([0, 1, 0], device="cuda")
        if wide > 1:
            d["lora_A"] = d["lora_A"] * 30
            d["lora_B"] = (d["lora_B"].float() * back).half()
        else:
            d["lora_A"] = (d["lora_A"].float() * 2.0 ** -4).half()
            d["y"] = d["y"] * 0
        check(C.multi_lora_add(**d), d, (256,))


@pytest.mark.parametrize("t", [None, 70])
def test_infinities_and_nan_stay_in_their_rows(C, t):
    d = inputs(4, t, 256, (128, 128), 16, 2, seed=11)
    d["adapters"] = torch.tensor([0, 0, 1, -1], device="cuda")
    clean = C.multi_lora_add(**d, splits=(128, 128))
    x = d["x"].view(4, -1, 256)
    x[0, 0, 5], x[1, -1, 7], x[3, 0, 0] = float("inf"), float("nan"), float("nan")
    got = C.multi_lora_add(**d, splits=(128, 128)).view(4, -1, 256)
    ref, _ = multi_lora_ref(*(d[n].cpu().numpy() for n in ("y", "x", "lora_A", "lora_B", "adapters", "scales")), (128, 128))
    ref = torch.from_numpy(ref).view(4, -1, 256)
    assert torch.equal(got[0, 0].cpu().isnan(), ref[0, 0].isnan()) and got[1, -1].isnan().all()
    assert torch.equal(got[0, 0].cpu().double()[~ref[0, 0].isnan()], ref[0, 0][~ref[0, 0].isnan()])
    mask = torch.ones(got.shape[:2], dtype=torch.bool)
    mask[0, 0] = mask[1, -1] = False
    assert torch.equal(got.cpu()[mask], clean.view(4, -1, 256).cpu()[mask])


def test_rows_past_two_to_the_31(C):
    """element offsets beyond 32 bits: the last adapter of many, the last rows of a large batch"""
    k, n_out, r = 4096, 64, 64
    n = (1 << 31) // (k * r) + 2
    A = torch.zeros(n, k, r, dtype=torch.float16, device="cuda")
    d = inputs(4, None, k, (n_out,), r, 1, seed=3)
    A[-1] = d["lora_A"][0]
    B = torch.zeros(n, r, n_out, dtype=torch.float16, device="cuda")
    B[-1] = d["lora_B"][0]
    small = {**d, "adapters": torch.zeros(4, dtype=torch.int64, device="cuda")}
    want = C.multi_lora_add(**small)
    check(want, small, (n_out,))
    big = {**d, "lora_A": A, "lora_B": B, "adapters": torch.full((4,), n - 1, device="cuda"),
           "scales": d["scales"].expand(n).contiguous()}
    assert torch.equal(C.multi_lora_add(**big), want)
    del A, B, big
    t = 1 << 15
    b = (1 << 31) // (t * 4096) + 1
    y = torch.zeros(b, t, 4096, dtype=torch.float16, device="cuda")
    x = torch.zeros(b, t, 64, dtype=torch.float16, device="cuda")
    d = inputs(1, 5, 64, (4096,), 8, 1, seed=4)
    y[-1, -5:], x[-1, -5:] = d["y"][0], d["x"][0]
    ids = torch.full((b,), -1, device="cuda")
    ids[-1] = 0
    got = C.multi_lora_add(y, x, d["lora_A"], d["lora_B"], ids, d["scales"], out=y)[-1, -5:]
    d["adapters"] = torch.zeros(1, dtype=torch.int64, device="cuda")
    check(got[None], d, (4096,))


def test_other_stream_and_captured_graph(C):
    d = inputs(6, None, 256, (256,), 16, 3, seed=2)
    d["adapters"] = torch.tensor([0, 1, 2, -1, 0, 2], device="cuda")
    want = C.multi_lora_add(**d)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = C.multi_lora_add(**d)
    s.synchronize()
    assert torch.equal(got, want)
    graph, held = torch.cuda.CUDAGraph(), dict(d, adapters=d["adapters"].clone(), scales=d["scales"].clone())
    with torch.cuda.graph(graph):
        out = C.multi_lora_add(**held)
    for ids, f in (([0, 1, 2, -1, 0, 2], 1.0), ([2, -1, 2, 1, 1, 5], 0.5), ([-1] * 6, 1.0)):
        held["adapters"].copy_(torch.tensor(ids))
        held["scales"].copy_(d["scales"] * f)
        graph.replay()
        assert torch.equal(out, C.multi_lora_add(**{**d, "adapters": held["adapters"], "scales": held["scales"]}))


def test_two_streams_at_once(C):
    ds = [inputs(16, 3, 512, (512,), 16, 4, seed=s) for s in (1, 2)]
    want = [C.multi_lora_add(**d) for d in ds]
    streams = [torch.cuda.Stream() for _ in ds]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(C.multi_lora_add(**ds[i]))
    torch.cuda.synchronize()
    assert all(torch.equal(o, want[i]) for i in (0, 1) for o in got[i])


def quantised(k, n, group, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randint(-2 ** 31, 2 ** 31 - 1, (k // 8, n), generator=g, device="cuda", dtype=torch.int32),
            (torch.rand(k // group, n, generator=g, device="cuda") * 0.02 + 0.005).half(),
            torch.full((k // group, n // 8), 0x88888888 - 2 ** 32, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("b,t", [(1, None), (8, 1), (3, 20), (2, 130)])
def test_beside_the_quantised_projection(C, b, t):
    """the projection and the adapters in one call: the two calls' bits; one adapter for all: near the merged op"""
    k, splits = 512, (512, 256)
    w = quantised(k, sum(splits), 128, seed=8)
    d = inputs(b, t, k, splits, 16, 3, seed=b)
    y = C.w4a16_gemv(d["x"], *w)
    got = C.w4a16_multi_lora_gemv(d["x"], *w, d["lora_A"], d["lora_B"], d["adapters"], d["scales"], splits=splits)
    assert torch.equal(got, C.multi_lora_add(**{**d, "y": y}, splits=splits))
    check(got, {**d, "y": y}, splits)
    d = inputs(b, t, k, (768,), 16, 3, seed=b)
    d["adapters"].fill_(1)
    d["scales"].fill_(2.0)
    got = C.w4a16_multi_lora_gemv(d["x"], *w, d["lora_A"], d["lora_B"], d["adapters"], d["scales"])
    merged = C.w4a16_lora_gemv(d["x"], *w, d["lora_A"][1].contiguous(), d["lora_B"][1].contiguous(), 128, 32.0)
    base = C.w4a16_gemv(d["x"], *w)
    # the projection's own rounding here, one rounding of the sum there and here; both fp32 sums within 2^-12 of a step
    allowed = (base.float().abs() + 2 * merged.float().abs()) * 2.0 ** -11 * (1 + 2.0 ** -5) + 1e-3
    assert ((got.float() - merged.float()).abs() <= allowed).all()


def test_refusals(C):
    d = inputs(2, None, 64, (64,), 8, 3)
    for change, msg in [
            (dict(x=d["x"].float()), "float16"), (dict(y=d["y"].t().contiguous().t()), "contiguous"),
            (dict(x=d["x"][0]), r"\[B, K\]"), (dict(x=d["x"][:1]), r"\[B, K\]"), (dict(adapters=d["adapters"].int()), "int64"),
            (dict(adapters=d["adapters"][:1]), "int64"), (dict(scales=d["scales"].double()), "float32"),
            (dict(scales=d["scales"][:2]), "float32"), (dict(lora_A=d["lora_A"][:2]), "lora_A"),
            (dict(lora_A=d["lora_A"][:, :32].contiguous()), "lora_A"), (dict(lora_B=d["lora_B"][0]), "lora_A"),
            (dict(splits=(32, 32)), "lora_A"), (dict(splits=()), "splits"), (dict(splits=(32,)), "cover"),
            (dict(splits=("a",)), None), (dict(splits=8), "sequence"), (dict(out=d["y"][:1]), "like y"),
            (dict(out=d["y"].float()), "float16"), (dict(out=d["x"]), "overlap"), (dict(adapters=d["adapters"].cpu()), "CUDA"),
            (dict(lora_B=torch.zeros(3, 4, 64, dtype=torch.float16, device="cuda"),
                  lora_A=torch.zeros(3, 64, 4, dtype=torch.float16, device="cuda")), "rank")]:
        with pytest.raises((RuntimeError, TypeError), match=msg):
            C.multi_lora_add(**{**d, **change})


@pytest.mark.parametrize("r", [16, 32, 64])
@pytest.mark.parametrize("b,t", [(36, 32), (30, 20), (7, 9)])
def test_cold_y_behind_a_short_product(C, r, b, t):
    """short chunks with many blocks of columns, y and B not in L2: each block has to wait for its own copies"""
    splits = (1024, 6144)
    d = inputs(b, t, 64, splits, r, 5, seed=r + b)
    flush = torch.empty(1 << 26, dtype=torch.int64, device="cuda")
    for i in range(3):
        flush.fill_(i)
        check(C.multi_lora_add(**d, splits=splits), d, splits)


@pytest.mark.parametrize("b,t", [(1, 1), (7, 1), (300, 1), (600, 2), (9000, 1), (3, 40), (300, 12)])
def test_adapters_written_by_the_kernel_before(C, b, t):
    """a kernel that lets the next one in while it runs writes the ids: the ones that count are the new ones"""
    import ctypes
    from qextract_infer_b200 import _lib
    lib, splits = _lib.load(), (40, 24)
    d = inputs(b, t, 136, splits, 8, 11, seed=b + t)
    logits = [torch.randn(b, 13, generator=torch.Generator(device="cuda").manual_seed(i), device="cuda").half() for i in range(3)]
    want = []
    for l in logits:
        ids = C.sample_logits(l, torch.zeros(b, device="cuda"), 0.0)[0]
        assert torch.equal(ids, l.float().argmax(1))
        want.append(C.multi_lora_add(**{**d, "adapters": ids}, splits=splits))
    torch.cuda.synchronize()
    u, lp, ids = torch.zeros(b, device="cuda"), torch.empty(b, device="cuda"), torch.zeros(b, dtype=torch.int64, device="cuda")
    d["adapters"] = ids
    outs = [torch.empty_like(d["y"]) for _ in range(12)]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        st = torch.cuda.current_stream().cuda_stream
        for i, out in enumerate(outs):
            _lib.check(lib.qx_sample_logits(logits[i % 3].data_ptr(), u.data_ptr(), None, None, None, None, 0.0, 0, 1.0, 0.0,
                                            ids.data_ptr(), lp.data_ptr(), b, 13, ctypes.c_void_p(st)), "sample_logits")
            C.multi_lora_add(**d, splits=splits, out=out)
    for _ in range(3):
        for out in outs:
            out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(out, want[i % 3]) for i, out in enumerate(outs))
    C.check_device_error()


@pytest.mark.parametrize("r,splits", [(8, (264,)), (64, (136, 256)), (24, (40, 600, 72)), (128, (264,))])
@pytest.mark.parametrize("t", [1, 5, 9, 100])
def test_a_row_has_the_same_bits_in_any_batch(C, r, splits, t):
    """few and many rows a call: other chunks, other clusters a chunk, the same sums"""
    b = 24
    d = inputs(b, t, 520, splits, r, 3, seed=r + t)
    whole = C.multi_lora_add(**d, splits=splits)
    for i in (0, 11, 23):
        one = {n: v[i:i + 1].contiguous() if n in ("x", "y", "adapters") else v for n, v in d.items()}
        assert torch.equal(C.multi_lora_add(**one, splits=splits)[0], whole[i])
