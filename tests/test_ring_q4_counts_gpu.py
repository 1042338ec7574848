"""Counts on the device that are outside 0 .. 2^62 - 1 are taken as the nearer end: nothing
outside the storage is written, and the other sequences are as they would be alone."""

import pytest
import torch

pytestmark = pytest.mark.gpu
LAST = (1 << 62) - 1


@pytest.mark.parametrize("S,W,T", [(4, 60, 1), (4, 60, 7), (0, 100, 300), (17, 8, 40)])
@pytest.mark.parametrize("wrong,taken", [((1 << 63) - 1, LAST), ((1 << 63) - 4, LAST), (1 << 62, LAST), (-1, 0), (-(1 << 63), 0)])
def test_a_count_outside_the_range(S, W, T, wrong, taken):
    from qextract_infer_b200 import _C
    B, H, D, group, pad = 3, 2, 128, 64, 1 << 16
    g = torch.Generator(device="cuda").manual_seed(T)

    def halves(*shape):
        return torch.randn(*shape, generator=g, device="cuda").half()

    k, v, q, one = halves(B, T, H, D), halves(B, T, H, D), halves(B, T, 4, D), halves(B, 4, D)
    results = []
    for count in (wrong, taken):
        rings, outer = [], []
        for t, fill in zip(_C.ring_q4_storage(B, H, D, S, W, group), (0x5A, 0x1230)):
            flat = torch.full((2 * pad + t.numel(),), fill, dtype=t.dtype, device="cuda")
            rings.append(flat[pad:-pad].view(t.shape))
            outer.append((flat, fill))
        counts = torch.tensor([50, count, 1000], device="cuda")
        att = _C.prefill_attention_q4(q, k, v, *rings, counts, S, W)
        _C.ring_append_q4(k, v, *rings, counts, S, W)
        dec = _C.decode_attention_q4(one, *rings, counts, S, W)
        torch.cuda.synchronize()
        for flat, fill in outer:
            assert (flat[:pad] == fill).all() and (flat[-pad:] == fill).all()
        results.append((*rings, att, dec))
    for a, b in zip(*results):
        assert torch.equal(a, b)
    alone = [t.fill_(f) for t, f in zip(_C.ring_q4_storage(1, H, D, S, W, group), (0x5A, 0x1230))]
    _C.ring_append_q4(k[:1].contiguous(), v[:1].contiguous(), *alone, 50, S, W)
    assert all(torch.equal(a[:, :1], b) for a, b in zip(results[0], alone))
