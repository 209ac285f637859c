"""Attention over scores of any finite size: up to where fp32 no longer holds a difference of 1 between two scores, and
far beyond.  There a row's result is the value of its largest score, or a mean over the scores that fp32 cannot tell
from it."""
import numpy as np
import pytest
import torch

from helpers import ext

pytestmark = pytest.mark.gpu


def _codes(T, H, kv, D, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes, scales = ext().quantize_per_token(torch.randn(T, H + 2 * kv, D, device="cuda", generator=g))
    return [codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv], scales[:, H + kv:]]


def _cu(lens):
    return torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")


def _hull(s, v):
    """s [L] scores in log2 units, v [L, D] values, float64 -> (low, high) [D] that a result may lie between, and the
    number of candidates: the values whose score is within what four roundings of a score (2^-24 of the largest) and 50
    log2 units leave to the largest -- below that a probability is zero in fp16 --, widened by 2^-11 for the rounding of
    p * scale and of the result (half a step of fp16 each), by 2^-25 for the smallest fp16 result, by as much of a
    candidate's p * scale, which is scaled to 2^6 and more for the largest scale, and by the weights left out."""
    best = s.max()
    near = v[s >= best - 4 * 2.0 ** -24 * abs(best) - 50]
    most = np.abs(v).max()
    slack = 1.05 * (2.0 ** -10 * np.abs(near).max(0) + 2.0 ** -25 + (len(near) - 1) * 2.0 ** -31 * most + 2.0 ** -50 * len(s) * most)
    return near.min(0) - slack, near.max(0) + slack, len(near)


def _check_varlen(out, args, lens, causal):
    """Every row between the bounds; returns how many rows had a single candidate."""
    q, k, v, sq, sk, sv = (a.double().cpu().numpy() for a in args)
    got = out.double().cpu().numpy()
    assert np.isfinite(got).all()
    H, kv, D = q.shape[1], k.shape[1], q.shape[2]
    at, single = 0, 0
    for n in lens:
        for h in range(H):
            g = h // (H // kv)
            s = (q[at:at + n, h] * sq[at:at + n, h, None]) @ (k[at:at + n, g] * sk[at:at + n, g, None]).T / np.sqrt(D) * np.log2(np.e)
            vv = v[at:at + n, g] * sv[at:at + n, g, None]
            for i in range(n):
                m = i + 1 if causal else n
                lo, hi, c = _hull(s[i, :m], vv[:m])
                single += c == 1
                assert (lo <= got[at + i, h]).all() and (got[at + i, h] <= hi).all(), (i, h)
        at += n
    return single


@pytest.mark.parametrize("D", [64, 128, 256])
@pytest.mark.parametrize("e", [16, 21, 23, 26, 28, 31, 40, 64, 100])
def test_varlen_large_scores(D, e):
    op, lens = ext().int8_attention_varlen, [300, 7, 129]
    args = _codes(sum(lens), 4, 2, D, seed=e)
    args[3], args[4] = args[3] * 2.0 ** (e // 2), args[4] * 2.0 ** (e - e // 2)
    for causal in (True, False):
        out = op(*args, _cu(lens), max(lens), causal)
        single = _check_varlen(out, args, lens, causal)
        assert single > 0.5 * 4 * sum(lens) or e < 21
        assert torch.equal(out, op(*args, _cu(lens), max(lens), causal))
    ext().check_status()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_varlen_scores_become_large_on_the_way(D):
    """Some keys, some queries, or the keys of a later tile only: rows with and without large scores side by side."""
    op, lens = ext().int8_attention_varlen, [420]
    base = _codes(420, 4, 2, D, seed=D)
    for first, last, f in ((150, 151, 2.0 ** 40), (0, 1, 2.0 ** 33), (260, 420, 2.0 ** 29), (390, 400, 2.0 ** 24), (100, 300, 2.0 ** 70)):
        for which in (3, 4):
            args = [a.clone() for a in base]
            args[which][first:last] *= f
            for causal in (True, False):
                out = op(*args, _cu(lens), 420, causal)
                _check_varlen(out, args, lens, causal)
                if which == 3 or causal:                                       # the rows that it does not concern keep their bits
                    keep = torch.ones(420, dtype=torch.bool)
                    keep[first:last if which == 3 else 420] = False
                    assert torch.equal(out[keep], op(*base, _cu(lens), 420, causal)[keep])
    ext().check_status()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_varlen_equal_largest_scores_share_the_row(D):
    args = _codes(200, 2, 1, D, seed=3)
    args[1][[20, 90, 150]] = args[0][40:41, :1]                                # the key that fits query 40 best, three times
    args[4][[20, 90, 150]] = 1.0
    args[4][[i for i in range(200) if i not in (20, 90, 150)]] = 2.0 ** -3
    args[4] = args[4] * 2.0 ** 36
    out = ext().int8_attention_varlen(*args, _cu([200]), 200, False)
    vv = (args[2].double() * args[5].double()[..., None])[[20, 90, 150], 0]
    want = vv.mean(0)
    slack = 1.05 * (2.0 ** -11 * (vv.abs().mean(0) + want.abs()) + 2.0 ** -24)
    assert ((out[40, 0].double() - want).abs() <= slack).all()
    assert torch.isfinite(out).all()


@pytest.mark.parametrize("D", [64, 128, 256])
def test_varlen_an_infinite_score_is_nan_in_its_rows_only(D):
    base = _codes(300, 2, 1, D, seed=4)
    good = ext().int8_attention_varlen(*base, _cu([300]), 300, True)
    args = [a.clone() for a in base]
    args[3][200] = float("inf")
    out = ext().int8_attention_varlen(*args, _cu([300]), 300, True)
    keep = torch.arange(300) != 200
    assert out[200].isnan().all() and torch.equal(out[keep], good[keep])


@pytest.mark.parametrize("D", [64, 128, 256])
def test_varlen_scores_of_minus_infinity_are_left_out(D):
    """Key scales of infinity where the products are negative: no probability, in the first tile or later, and a row that
    has only such scores at first starts where it has others."""
    args = _codes(400, 2, 1, D, seed=5)
    args[1][:200] = -args[0][250:251, :1]                                      # against query 250 of head 0
    args[4][:200] = float("inf")
    out = ext().int8_attention_varlen(*args, _cu([400]), 400, True)
    q, k, v, sq, sk, sv = (a.double().cpu().numpy() for a in args)
    s = (k[200:251, 0] @ q[250, 0]) * sk[200:251, 0] * sq[250, 0] / np.sqrt(D) * np.log2(np.e)
    vv = v[200:251, 0] * sv[200:251, 0, None]
    p = np.exp2(s - s.max())
    p /= p.sum()
    want, spread = p @ vv, p @ np.abs(vv)
    slack = 1.05 * (2.0 ** -11 * (spread + np.abs(want)) + 51 * 2.0 ** -31 * np.abs(v[:251, 0] * sv[:251, 0, None]).max() + 2.0 ** -25)
    assert (np.abs(out[250, 0].double().cpu().numpy() - want) <= slack).all()
