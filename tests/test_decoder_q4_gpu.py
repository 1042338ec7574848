"""The decoder with its ring held in 4 bits (``kv_bits=4``) against its fp32 torch
restatement with the same quantisation: prompt chunks attend the ring's 4-bit
tokens and their own fp16 ones, decode steps 4-bit tokens only, their own among
them.  And the fp16 decoder's prefill, whose norms and rotation run in one
kernel, bit for bit against the separate ones.

Tolerance: 1e-2 of the largest value, as in the fp16 decoder's test, twice: keys
and values are off by fp16 roundings there (2^-11 of |x|), so against a step of
the quantiser (a fifteenth of a group's span, |x| about a quarter of it) about
2^-11 x 15/4 x 2 = 0.4 % of them land on the neighbouring code, which is one part
in 15 of a span off: in the 2-norm sqrt(0.004) / 4 = 1.6 % of the quantisation
error itself (7 % of the values), 0.1 % of the values."""

import pytest
import torch

from oracle import kv4_values
from tests.decoder_ref import RefDecoder
from tests.test_decoder_gpu import _close, _tiny_cfg

pytestmark = pytest.mark.gpu


class _Held(list):
    """(position, k, v) of a layer; what comes before ``fresh_from`` reads as the 4-bit ring holds it."""

    def __init__(self, group):
        super().__init__()
        self.group, self.fresh_from = group, 0

    def append(self, e):
        p, k, v = e
        q = [torch.from_numpy(kv4_values(t.half().cpu().numpy(), self.group)).to(t) for t in (k, v)]
        super().append((p, (k, v), q))

    def __iter__(self):
        for p, raw, q in super().__iter__():
            yield (p, *(raw if p >= self.fresh_from else q))


@pytest.mark.parametrize("kv_group", [32, 64, 128])
def test_prefill_and_decode_match_reference(kv_group):
    from qextract_infer_b200.tp_decoder import TPDecoder
    dev = torch.device("cuda", 0)
    cfg = _tiny_cfg()
    cfg.kv_bits, cfg.kv_group = 4, kv_group
    B, T, chunk = 2, 100, 64
    dec = TPDecoder(cfg, batch=B, device=dev, seed=7)
    ref = RefDecoder(dec)
    ref.kh = [_Held(kv_group) for _ in dec.layers]
    toks = torch.randint(0, cfg.vocab, (B, T), generator=torch.Generator().manual_seed(4)).to(dev)
    _, hid = dec.prefill(toks, chunk=chunk, return_hidden=True)
    for t in range(T):
        for kept in ref.kh:
            kept.fresh_from = t // chunk * chunk
        xr = ref.token(toks[:, t])
    _close(hid, xr, "prefill hidden", tol=2e-2)
    for step in range(6):
        for kept in ref.kh:
            kept.fresh_from = 1 << 30
        tok = torch.randint(0, cfg.vocab, (B,), generator=torch.Generator().manual_seed(50 + step)).to(dev)
        _, hid = dec.decode_step(tok, return_hidden=True)
        xr = ref.token(tok)
        _close(hid, xr, f"decode step {step} hidden", tol=2e-2)
    assert dec.cache.get_total_written() == T + 6
    with pytest.raises(ValueError, match="kv_bits"):
        cfg.kv_bits = 8
        TPDecoder(cfg, batch=1, device=dev, seed=7)


def test_fp16_prefill_is_bit_identical_with_separate_norms_and_rotation(monkeypatch):
    from qextract_infer_b200 import _C
    from qextract_infer_b200.tp_decoder import TPDecoder
    dev = torch.device("cuda", 0)
    cfg = _tiny_cfg()
    toks = torch.randint(0, cfg.vocab, (2, 100), generator=torch.Generator().manual_seed(4)).to(dev)
    hidden, rings = [], []

    def separate(qkv, hq, hkv, qn, kn, eps, cos, sin):
        B, n, _ = qkv.shape
        q, k, v = qkv.view(B, n, -1, qn.numel()).split([hq, hkv, hkv], 2)

        def rope(x):
            xf = x.float()
            half = x.size(-1) // 2
            rot = torch.cat([-xf[..., half:], xf[..., :half]], dim=-1)
            return (xf * cos[:, None, :] + rot * sin[:, None, :]).half()

        return (rope(_C.fused_rmsnorm(q.contiguous(), qn, eps)), rope(_C.fused_rmsnorm(k.contiguous(), kn, eps)),
                v.contiguous())

    for fused in (True, False):
        if not fused:
            monkeypatch.setattr(_C, "qk_norm_rope", separate)
        dec = TPDecoder(cfg, batch=2, device=dev, seed=7)
        _, h = dec.prefill(toks, chunk=64, return_hidden=True)
        hidden.append(h)
        rings.append((dec.cache.k.clone(), dec.cache.v.clone()))
    assert torch.equal(*hidden)
    assert torch.equal(rings[0][0], rings[1][0]) and torch.equal(rings[0][1], rings[1][1])
