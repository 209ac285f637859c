"""Packed attention with several times more pairs of query tiles than the GPU has SMs: what a CTA carries from one pair to
the next (rings, slots, phases, scores issued ahead), against float64."""
import numpy as np
import pytest
import torch

from helpers import ext
from oracle import grouped as og

pytestmark = pytest.mark.gpu

# pairs of one to six key tiles, with and without a second query tile, in an order that changes both from pair to pair
LENS = [1, 700, 3, 129, 400, 64, 257, 0, 130, 515, 5, 128, 127, 650, 300, 90, 40, 385, 256, 200]


@pytest.mark.parametrize("H,kv,D,causal", [(24, 8, 128, True), (16, 8, 64, True), (16, 8, 128, False), (8, 8, 64, False), (48, 24, 128, True)])
def test_varlen_more_pairs_than_ctas(H, kv, D, causal):
    e, T, group = ext(), sum(LENS), H // kv
    pairs = sum(-(-n // (2 * (128 // group))) for n in LENS) * kv
    assert pairs >= 1.5 * torch.cuda.get_device_properties(0).multi_processor_count
    g = torch.Generator(device="cuda").manual_seed(H + D)
    x = torch.randn(T, H + 2 * kv, D, device="cuda", generator=g)
    x[:, H + kv:] = x[:, H + kv:] * torch.exp(torch.randn(T, kv, 1, device="cuda", generator=g)) + 0.3
    x[:, :H] *= torch.exp(1.5 * torch.rand(T, H, 1, device="cuda", generator=g))              # some rows move their reference
    codes, scales = e.quantize_per_token(x)
    split = lambda t: (t[:, :H], t[:, H:H + kv], t[:, H + kv:])  # noqa: E731
    cu = torch.tensor(np.concatenate([[0], np.cumsum(LENS)]), dtype=torch.int32, device="cuda")
    out = e.int8_attention_varlen(*split(codes), *split(scales), cu, max(LENS), causal)
    assert torch.equal(out, e.int8_attention_varlen(*split(codes), *split(scales), cu, max(LENS), causal))
    cn, sn, got = codes.cpu().numpy(), scales.cpu().numpy(), out.float().cpu().numpy()
    for h in (0, kv - 1):                                                  # the heads of a sequence are pairs of their own
        at, k, v = slice(h * group, (h + 1) * group), slice(H + h, H + h + 1), slice(H + kv + h, H + kv + h + 1)
        want, bound = og.varlen_attention(cn[:, at], cn[:, k], cn[:, v], sn[:, at], sn[:, k], sn[:, v], cu.tolist(), causal)
        off = np.abs(got[:, at] - want)
        assert (off <= bound).all(), (h, (off / bound).max())
    # every head: a sequence alone, where a CTA has one pair at most
    ends = cu.tolist()
    for b in (1, 4, 13, 18):
        one = slice(ends[b], ends[b + 1])
        alone = e.int8_attention_varlen(*[t[one] for t in split(codes)], *[t[one] for t in split(scales)],
                                        torch.tensor([0, LENS[b]], dtype=torch.int32, device="cuda"), LENS[b], causal)
        assert torch.equal(out[one], alone)
    e.check_status()
