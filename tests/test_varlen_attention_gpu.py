"""INT8 attention over packed sequences (grouped heads, causal or not) against its float64 restatement."""
import numpy as np
import pytest
import torch

from helpers import cabi, ext
from oracle import grouped as og

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _case(T, H, kv, D, seed, spread=1.0):
    """Slices of one [T, H + 2 kv, D] tensor of codes, as the fused quantiser leaves them."""
    g = _gen(seed)
    x = torch.randn(T, H + 2 * kv, D, device="cuda", generator=g) * spread
    x[:, H + kv:] = x[:, H + kv:] * torch.exp(torch.randn(T, kv, 1, device="cuda", generator=g)) + 0.3
    codes, scales = ext().quantize_per_token(x)
    return [codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv], scales[:, H + kv:]]


def _cu(lens, first=0):
    return torch.tensor(np.concatenate([[first], first + np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _check(out, args, cu, causal):
    want, bound = og.varlen_attention(*[a.cpu().numpy() for a in args], cu.cpu().tolist(), causal)
    got = out.float().cpu().numpy()
    off = np.abs(got - want)
    inside = np.zeros(len(got), dtype=bool)
    inside[int(cu[0]):int(cu[-1])] = True
    assert (off <= bound)[inside].all(), (off[inside] / bound[inside]).max()
    assert not got[~inside].any()


@pytest.mark.parametrize("H,kv,D,causal,lens", [
    (1, 1, 64, True, [1]), (12, 12, 64, True, [67, 1, 0, 64, 65]), (8, 2, 128, True, [130, 63, 0, 0, 257, 2]), (4, 4, 128, False, [129, 1, 64]),
    (14, 2, 256, True, [100, 33]), (14, 2, 256, False, [70, 193]), (6, 2, 64, True, [300]), (16, 1, 128, True, [40, 200, 8, 7]), (5, 1, 64, False, [0, 5, 131]),
    (64, 1, 64, True, [3, 150]), (24, 8, 128, True, [511, 512]), (3, 1, 256, True, [1, 2, 3, 126, 127, 128, 0])])
def test_varlen(H, kv, D, causal, lens):
    e = ext()
    args = _case(sum(lens), H, kv, D, seed=H + D + len(lens))
    cu = _cu(lens)
    out = e.int8_attention_varlen(*args, cu, max(lens), causal)
    assert out.dtype == torch.float16 and out.shape == (sum(lens), H, D)
    _check(out, args, cu, causal)
    assert torch.equal(out, e.int8_attention_varlen(*[a.contiguous() for a in args], cu, max(lens), causal))
    e.check_status()


def test_varlen_rows_outside_every_sequence_are_zero_and_a_longer_sequence_is_cut():
    e = ext()
    lens = [50, 90]
    args = _case(170, 8, 2, 64, seed=2)
    cu = _cu(lens, first=7)                                                # rows 0..6 and 147.. belong to nobody
    _check(e.int8_attention_varlen(*args, cu, 90), args, cu, True)
    out = e.int8_attention_varlen(*args, cu, 64)                           # the second sequence is cut to 64
    ref = [a.clone() for a in args]
    want, bound = og.varlen_attention(*[a.cpu().numpy() for a in ref], [7, 57, 121], True)
    got = out.float().cpu().numpy()
    assert (np.abs(got - want) <= bound)[7:121].all() and not got[121:].any() and not got[:7].any()
    damaged = torch.tensor([7, -900, 10 ** 9], dtype=torch.int32, device="cuda")   # read inside [0, T]
    e.int8_attention_varlen(*args, damaged, 170)
    torch.cuda.synchronize()
    e.check_status()


@pytest.mark.parametrize("causal", [True, False])
def test_varlen_what_a_row_does_not_see_cannot_reach_it(causal):
    """NaN and infinite scales: in other sequences, behind the last one and, with the mask, in later positions."""
    e = ext()
    lens = [70, 100, 33]
    q, k, v, sq, sk, sv = _case(220, 4, 2, 128, seed=9)
    cu = _cu(lens)
    good = e.int8_attention_varlen(q, k, v, sq, sk, sv, cu, 100, causal)
    for scale in (0, 1):
        for value in (float("nan"), float("inf"), -float("inf")):
            sk2, sv2 = sk.clone(), sv.clone()
            (sk2 if scale == 0 else sv2)[160, 0] = value                   # position 90 of the second sequence, key head 0
            sk2[203:], sv2[203:] = float("nan"), float("nan")              # rows of no sequence
            out = e.int8_attention_varlen(q, k, v, sq, sk2, sv2, cu, 100, causal)
            touched = torch.zeros(220, 4, dtype=torch.bool)
            touched[160 if causal else 70:170, :2] = True
            assert torch.equal(out[~touched], good[~touched])
            if value != value or scale == 1:
                assert not torch.isfinite(out[touched].float()).any()


def test_varlen_scales_of_any_size_and_zero():
    e = ext()
    lens = [90, 70]
    q, k, v, sq, sk, sv = _case(160, 4, 1, 64, seed=4)
    cu = _cu(lens)
    for f in (1e-4, 300.0):                                                # values far from 1, and spread by 2^20 inside a sequence
        sv2 = sv * f
        sv2[10:40] *= 2.0 ** -20
        args = [q, k, v, sq, sk, sv2]
        _check(e.int8_attention_varlen(*args, cu, 90), args, cu, True)
    sq0, sv0 = sq.clone(), sv.clone()
    sq0[5] = 0                                                             # all scores equal: the mean of what the row sees
    sv0[90:] = 0                                                           # a sequence whose values are zero
    args = [q, k, v, sq0, sk, sv0]
    _check(e.int8_attention_varlen(*args, cu, 90), args, cu, True)


def test_varlen_peaked_scores_move_the_maximum():
    e = ext()
    args = _case(700, 4, 2, 128, seed=6, spread=12.0)
    cu = _cu([400, 300])
    _check(e.int8_attention_varlen(*args, cu, 400), args, cu, True)


def test_varlen_one_key_head_each_agrees_with_the_prefill_op():
    """Not causal, equal lengths, one key head per query head: what int8_attention_forward computes."""
    e = ext()
    B, H, S, D = 2, 4, 200, 128
    x = torch.randn(3, B, H, S, D, device="cuda", generator=_gen(1))
    codes, scales = e.quantize_per_token(x)
    a = e.int8_attention_forward(codes[0], codes[1], codes[2], *[s.reshape(-1) for s in scales])
    rows = [c.transpose(1, 2).reshape(B * S, H, D) for c in codes]
    sc = [s.transpose(1, 2).reshape(B * S, H) for s in scales]
    b = e.int8_attention_varlen(*rows, *sc, _cu([S] * B), S, False).view(B, S, H, D).transpose(1, 2)
    assert (a.float() - b.float()).abs().max() < 2e-3


def test_varlen_bad_strides_are_refused():
    e = ext()
    args = _case(20, 4, 2, 64, seed=1)
    cu = _cu([20])
    wide = torch.zeros(20, 4 * 64 + 8, dtype=torch.int8, device="cuda")[:, :256].view(20, 4, 64)
    with pytest.raises(RuntimeError, match="multiple of 16"):
        e.int8_attention_varlen(wide, *args[1:], cu, 20)
    with pytest.raises(RuntimeError, match="contiguous"):
        e.int8_attention_varlen(*args[:3], args[3].t().contiguous().t(), *args[4:], cu, 20)
    with pytest.raises(RuntimeError, match="key heads"):
        e.int8_attention_varlen(args[0][:, :3], args[1], args[2], args[3][:, :3], args[4], args[5], cu, 20)
    with pytest.raises(RuntimeError, match="cu_seqlens"):
        e.int8_attention_varlen(*args, cu.long(), 20)
    assert e.int8_attention_varlen(*[a[:0] for a in args], cu, 20).shape == (0, 4, 64)
    assert cabi().load().i8tk_attention_varlen_workspace_bytes(0, 1, 4, 2, 64) == 0
