"""The decoder with an adapter and sampling settings for each sequence, against its
fp32 torch restatement: prompts in chunks (the tensor-core GEMM and the GEMV beside the
adapters of many rows), decode steps, the drawn tokens from the decoder's own logits.
Tolerance: that of the decoder's test (1e-2 of the largest value; the projection is
rounded once more before the adapters are added, 2^-12 of it)."""

import numpy as np
import pytest
import torch

from oracle import dequantize_gptq
from oracle.requests import sample_ref
from tests import decoder_ref
from tests.test_decoder_gpu import _close, _tiny_cfg

pytestmark = pytest.mark.gpu


def _dense(lin, device):
    W = dequantize_gptq(lin.qweight.cpu().numpy(), lin.scales.cpu().numpy(), lin.qzeros.cpu().numpy(), lin.group)
    return (torch.from_numpy(np.asarray(W, dtype=np.float32)).to(device), lin.lora_A.float(), lin.lora_B.float(),
            lin.lora_scales.tolist(), lin.splits)


class Ref(decoder_ref.RefDecoder):
    ids = []

    def _lin(self, x, p):
        W, A, B, scales, splits = p
        y = x @ W
        r = B.size(1)
        for b, a in enumerate(self.ids):
            if 0 <= a < len(scales):
                at = 0
                for j, width in enumerate(splits):
                    y[b, at:at + width] += scales[a] * (x[b] @ A[a][:, j * r:(j + 1) * r] @ B[a][:, at:at + width])
                    at += width
        return y


def _make(monkeypatch, batch, ids, **more):
    from qextract_infer_b200.tp_decoder import TPDecoder
    monkeypatch.setattr(decoder_ref, "_dense", _dense)
    cfg = _tiny_cfg()
    cfg.adapters = 3
    for name, v in more.items():
        setattr(cfg, name, v)
    dec = TPDecoder(cfg, batch=batch, device=torch.device("cuda", 0), seed=7)
    for L in dec.layers:
        for name in ("qkv", "o", "gate_up", "down"):
            L[name].lora_B.mul_(10)  # adapters that change the outputs by about as much as the projections do
    dec.adapter_ids.copy_(torch.tensor(ids))
    ref = Ref(dec)
    ref.ids = ids
    return dec, ref


@pytest.mark.parametrize("ids", [[0, 2, -1], [1, 1, 1], [-1, 5, -1]])
@pytest.mark.parametrize("chunk", [64, 30])
def test_prefill_and_decode_with_adapters(monkeypatch, ids, chunk):
    dec, ref = _make(monkeypatch, 3, ids)
    T = 100
    toks = torch.randint(0, dec.cfg.vocab, (3, T), generator=torch.Generator().manual_seed(4)).cuda()
    _, hid = dec.prefill(toks, chunk=chunk, return_hidden=True)
    for t in range(T):
        xr = ref.token(toks[:, t])
    _close(hid, xr, "prefill hidden")
    for step in range(3):
        tok = torch.randint(0, dec.cfg.vocab, (3,), generator=torch.Generator().manual_seed(50 + step)).cuda()
        _, hid = dec.decode_step(tok, return_hidden=True)
        xr = ref.token(tok)
        _close(hid, xr, f"decode step {step} hidden")


def test_adapters_change_the_outputs(monkeypatch):
    toks = torch.randint(0, 1024, (3, 40), generator=torch.Generator().manual_seed(4)).cuda()
    hidden = []
    for ids in ([0, 1, 2], [0, 1, -1], [2, 1, 2]):
        dec, _ = _make(monkeypatch, 3, ids)
        hidden.append(dec.prefill(toks, return_hidden=True)[1])
    assert torch.equal(hidden[0][:2], hidden[1][:2]) and torch.equal(hidden[0][1:], hidden[2][1:])  # the others' bits stay
    scale = hidden[0].float().abs().max()
    assert (hidden[0][2] - hidden[1][2]).abs().max() > 0.1 * scale and (hidden[0][0] - hidden[2][0]).abs().max() > 0.1 * scale


@pytest.mark.parametrize("adapters,kv_bits", [(0, 16), (3, 16), (3, 4)])
def test_sampled_steps(monkeypatch, adapters, kv_bits):
    """tokens are those of the step's logits; temperature 0 is the greedy step; a captured step follows
    numbers, settings and adapters"""
    from qextract_infer_b200.tp_decoder import Sampling, TPDecoder
    cfg = _tiny_cfg()
    cfg.adapters, cfg.kv_bits = adapters, kv_bits
    dec = TPDecoder(cfg, batch=4, device=torch.device("cuda", 0), seed=7)
    toks = torch.randint(0, cfg.vocab, (4, 20), generator=torch.Generator().manual_seed(4)).cuda()
    g = torch.Generator(device="cuda").manual_seed(1)
    s = Sampling(torch.rand(4, generator=g, device="cuda"), torch.tensor([0.0, 0.5, 1.0, 3.0], device="cuda"), 50, 0.95,
                 torch.tensor([0.0, 0.0, 0.01, 0.0], device="cuda"))

    def drawn(hidden):
        logits = dec._greedy_logits(hidden)  # torch's product: only rows without a near tie are compared
        return logits, sample_ref(logits.cpu().numpy(), s.u.cpu().numpy(), s.temperature.cpu().numpy(), [50] * 4,
                                  np.full(4, 0.95, np.float32), s.min_p.cpu().numpy())

    tok, hid = dec.prefill(toks, return_hidden=True, sampling=s)
    assert tok.shape == (4,) and s.logprobs.shape == (4,) and (s.logprobs <= 0).all()
    from qextract_infer_b200 import _C
    h = _C.fused_rmsnorm(hid, dec.final_norm, cfg.rms_eps)
    logits = _C.lm_head_logits(h, dec.lm_head)
    _close(logits, drawn(hid)[0], "logits", tol=2e-3)
    want, lp = sample_ref(logits.cpu().numpy(), s.u.cpu().numpy(), s.temperature.cpu().numpy(), [50] * 4,
                          np.full(4, 0.95, np.float32), s.min_p.cpu().numpy())
    assert tok.tolist() == want.tolist() and np.allclose(s.logprobs.cpu().numpy(), lp, rtol=1e-6, atol=1e-7)
    # greedy by temperature 0
    count = dec.cache.get_total_written()
    zero = Sampling(s.u, 0.0)
    a = dec.decode_step(tok, sampling=zero)
    dec.cache._write_count = count
    b = dec.decode_step(tok)
    assert torch.equal(a, b) and (zero.logprobs == 0).all()
    # captured
    dec.cache._write_count = count
    graph = torch.cuda.CUDAGraph()
    held = tok.clone()
    with torch.cuda.graph(graph):
        out = dec.decode_step(held, sampling=s)
    captured = s.logprobs
    for i in range(3):
        s.u.copy_(torch.rand(4, generator=g, device="cuda"))
        s.temperature.copy_(torch.tensor([1.0, 0.0, 2.0, 0.3]).roll(i))
        if adapters:
            dec.adapter_ids.copy_(torch.tensor([i - 1, 2, 1, 0]))
        held.copy_(toks[:, i])
        graph.replay()
        got, got_lp = out.clone(), captured.clone()
        dec.cache._write_count = count
        eager = dec.decode_step(held, sampling=s)
        assert torch.equal(got, eager) and torch.equal(got_lp, s.logprobs)
