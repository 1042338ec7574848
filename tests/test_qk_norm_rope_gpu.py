"""Head norm + rotation of a chunk in one pass (``qk_norm_rope``): bit for bit
the sequence it replaces, and against the formula in 64 bits."""

import numpy as np
import pytest
import torch

from oracle import head_norm_rope64

pytestmark = pytest.mark.gpu
EPS = 1e-6


@pytest.fixture(scope="module")
def C():
    assert torch.cuda.is_available(), "GPU test run without a GPU"
    from qextract_infer_b200 import _C
    return _C


def _inputs(B, T, hq, hkv, d, own_positions, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    qkv = (torch.randn(B, T, (hq + 2 * hkv) * d, generator=g, device="cuda") * 2).half()
    qn, kn = ((1 + 0.3 * torch.randn(d, generator=g, device="cuda")).half() for _ in range(2))
    first = torch.randint(0, 60000, (B if own_positions else 1,), generator=g, device="cuda")
    pos = first[:, None] + torch.arange(T, device="cuda")
    ang = pos.double()[..., None] * 1e6 ** (-torch.arange(0, d, 2, device="cuda").double() / d)
    cos = torch.cat([ang.cos(), ang.cos()], -1).float()
    sin = torch.cat([ang.sin(), ang.sin()], -1).float()
    if not own_positions:
        cos, sin = cos[0].contiguous(), sin[0].contiguous()
    return qkv, qn, kn, cos, sin


def _unfused(C, qkv, hq, hkv, qn, kn, cos, sin):
    """fused_rmsnorm over the heads, then x cos + rot(x) sin in fp32."""
    B, T, _ = qkv.shape
    d = qn.numel()
    q, k, v = qkv.view(B, T, -1, d).split([hq, hkv, hkv], 2)

    def rope(x):
        xf = x.float()
        rot = torch.cat([-xf[..., d // 2:], xf[..., :d // 2]], -1)
        return (xf * cos.unsqueeze(-2) + rot * sin.unsqueeze(-2)).half()

    return (rope(C.fused_rmsnorm(q.contiguous(), qn, EPS)), rope(C.fused_rmsnorm(k.contiguous(), kn, EPS)),
            v.contiguous())


@pytest.mark.parametrize("B,T,hq,hkv,d,own_positions", [
    (1, 1, 32, 8, 128, False), (1, 2048, 32, 8, 128, False), (2, 37, 4, 2, 128, True), (3, 333, 15, 5, 64, True),
    (32, 1, 32, 8, 128, False), (5, 1, 1, 1, 64, True), (1, 130, 7, 1, 256, False), (2, 300, 3, 3, 256, True),
])
def test_equals_the_unfused_sequence_and_the_formula(C, B, T, hq, hkv, d, own_positions):
    qkv, qn, kn, cos, sin = _inputs(B, T, hq, hkv, d, own_positions, seed=T + d)
    got = C.qk_norm_rope(qkv, hq, hkv, qn, kn, EPS, cos, sin)
    want = _unfused(C, qkv, hq, hkv, qn, kn, cos, sin)
    for a, b, n in zip(got, want, "qkv"):
        assert a.shape == b.shape and torch.equal(a, b), n
    ref = head_norm_rope64(*(t.cpu().numpy() if isinstance(t, torch.Tensor) else t
                             for t in (qkv, hq, hkv, qn, kn, EPS, cos, sin)))
    c, s = (np.abs(np.broadcast_to(t.cpu().numpy(), (B, T, d)))[:, :, None] for t in (cos, sin))
    for a, r, n in zip(got[:2], ref[:2], "qk"):
        # two fp16 roundings (2^-11 each): of the normed head, which enters as y cos and rot(y) sin with |y| at
        # most the pair's length, and of the result; fp32 in between (D terms of a sum of squares, under 2^-16)
        pair = np.sqrt(r ** 2 + np.concatenate([r[..., d // 2:], r[..., :d // 2]], -1) ** 2)
        bound = (2.0 ** -11 + 2.0 ** -15) * (np.abs(r) + pair * (c + s)) + 2.0 ** -23
        assert (np.abs(a.cpu().numpy().astype(np.float64) - r) <= bound).all(), n


def test_zero_heads_and_non_finite_values_stay_in_their_head(C):
    qkv, qn, kn, cos, sin = _inputs(1, 3, 4, 2, 128, False, seed=5)
    qkv.view(1, 3, 8, 128)[0, 0, 1] = 0
    qkv.view(1, 3, 8, 128)[0, 1, 2, 7] = float("inf")
    qkv.view(1, 3, 8, 128)[0, 2, 5, 9] = float("nan")
    q, k, v = C.qk_norm_rope(qkv, 4, 2, qn, kn, EPS, cos, sin)
    assert (q[0, 0, 1] == 0).all()
    assert q[0, 1, 2].isnan().any() and k[0, 2, 1].isnan().all()
    q[0, 1, 2], k[0, 2, 1] = 0, 0
    assert q.isfinite().all() and k.isfinite().all() and torch.equal(v, qkv.view(1, 3, 8, 128)[:, :, 6:])


def test_empty_and_refused(C):
    qkv, qn, kn, cos, sin = _inputs(2, 3, 4, 2, 128, False, seed=6)
    q, k, v = C.qk_norm_rope(qkv[:0].contiguous(), 4, 2, qn, kn, EPS, cos, sin)
    assert q.shape == (0, 3, 4, 128) and v.shape == (0, 3, 2, 128)
    q, _, _ = C.qk_norm_rope(qkv[:, :0].contiguous(), 4, 2, qn, kn, EPS, cos[:0], sin[:0])
    assert q.shape == (2, 0, 4, 128)
    for bad in (dict(qkv=qkv.float()), dict(qkv=qkv[:, :, :-128].contiguous()), dict(qkv=qkv[0]), dict(qkv=qkv[:, ::2]),
                dict(cos=cos.half()), dict(cos=cos[:2].contiguous()), dict(sin=sin[:, :64].contiguous()),
                dict(qn=qn[:64]), dict(kn=kn.cpu()), dict(hq=3)):
        a = {**dict(qkv=qkv, hq=4, hkv=2, qn=qn, kn=kn, cos=cos, sin=sin), **bad}
        with pytest.raises(RuntimeError):
            C.qk_norm_rope(a["qkv"], a["hq"], a["hkv"], a["qn"], a["kn"], EPS, a["cos"], a["sin"])
    with pytest.raises(RuntimeError):  # head_dim 32
        C.qk_norm_rope(qkv.view(2, 3, -1), 16, 8, qn[:32].contiguous(), kn[:32].contiguous(), EPS,
                       cos[:, :32].contiguous(), sin[:, :32].contiguous())


def test_on_another_stream_and_captured(C):
    qkv, qn, kn, cos, sin = _inputs(2, 37, 4, 2, 128, False, seed=7)
    want = C.qk_norm_rope(qkv, 4, 2, qn, kn, EPS, cos, sin)
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        got = C.qk_norm_rope(qkv, 4, 2, qn, kn, EPS, cos, sin)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    x = torch.zeros_like(qkv)
    with torch.cuda.graph(graph):
        got = C.qk_norm_rope(x, 4, 2, qn, kn, EPS, cos, sin)
    x.copy_(qkv)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
