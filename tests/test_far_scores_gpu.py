"""Attention over scores of any finite size: up to where fp32 no longer holds a difference of 1 between two scores, and
far beyond.  There a row's result is the value of its largest score, or a mean over the scores that fp32 cannot tell
from it."""
import numpy as np
import pytest
import torch

from helpers import ext
from oracle import grouped as og

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


# ---- 4-bit decode ------------------------------------------------------------------------------------
def _cache(lens, kv, D, page, seed, f=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    need = [-(-n // page) for n in lens]
    pool = torch.zeros(sum(need), kv, ext().int4_kv_block_bytes(page, D), dtype=torch.uint8, device="cuda")
    order = torch.randperm(sum(need), device="cuda", generator=g).int()
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        pos = torch.arange(n, device="cuda")
        slots = table[b, (pos // page)].long() * page + pos % page
        k, v = (torch.randn(n, kv, D, device="cuda", generator=g) for _ in range(2))
        k, v = k.half(), (v * f).half()
        ext().kv_append_quantize_int4(k, v, pool, slots, page)
        at += need[b]
    return pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _rows(pool, table, b, h, n, page, D):
    blocks = [og.int4_unblock(pool[p, h], page, D) for p in table[b, :-(-n // page)]]
    return [[np.concatenate([blk[i][x] for blk in blocks])[:n].astype(np.float64) for x in range(3)] for i in (0, 1)]


@pytest.mark.parametrize("H,kv,D,page,lens", [(4, 4, 64, 16, [3000, 1]), (8, 2, 128, 32, [300, 5, 129]), (4, 2, 128, 128, [2, 700]), (24, 2, 64, 64, [400]),
                                              (7, 1, 64, 16, [129, 64])])
@pytest.mark.parametrize("e,f", [(16, 1.0), (21, 2.0 ** -9), (23, 1.0), (24, 16.0), (25, 4.0), (26, 2.0 ** -5), (27, 2.0 ** -7), (28, 2.0 ** -9), (31, 1.0),
                                 (40, 64.0), (64, 1.0), (100, 1.0)])
def test_int4_decode_large_scores(H, kv, D, page, lens, e, f):
    """A score is put together from s (q . c - 8 Q) + z Q per group, with up to eight roundings of half a step (2^-24) of
    these parts.  p * s is rounded to fp16 (2^-11 of up to 8 steps s), the result too; where p * s is below the range,
    half the smallest fp16 number (2^-25) times 8 for each candidate.  The values' size moves the reference."""
    pool, table, ln = _cache(lens, kv, D, page, H + D, f)
    q, sq = ext().quantize_per_token(torch.randn(len(lens), H, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(e)))
    far = sq * 2.0 ** e
    if e % 2 == 0:
        far[:, ::2] = sq[:, ::2]                                               # every other head as it was
    out = ext().int4_decode_attention_paged(q, far, pool, table, ln, max(lens), page)
    got, qn, sn, pn, tn = out.double().cpu().numpy(), q.double().cpu().numpy(), far.double().cpu().numpy(), pool.cpu().numpy(), table.cpu().numpy()
    assert np.isfinite(got).all()
    single = 0
    for b, n in enumerate(lens):
        for j in range(H):
            (kc, ks, kz), (vc, vs, vz) = _rows(pn, tn, b, j // (H // kv), n, page, D)
            qg = qn[b, j].reshape(-1, 64)
            dot, total = np.einsum("lgc,gc->lg", kc.reshape(n, -1, 64), qg), qg.sum(-1)
            unit = sn[b, j] * np.log2(np.e) / np.sqrt(D)
            s = unit * (ks * (dot - 8 * total) + kz * total).sum(-1)
            size = unit * (ks * (np.abs(dot) + 8 * np.abs(total)) + np.abs(kz * total)).sum(-1).max()
            v = og.int4_values(vc, vs, vz)
            near = s >= s.max() - 2 * 8 * 2.0 ** -24 * size - 50
            slack = 1.05 * (2.0 ** -11 * (8 * vs[near].max() + np.abs(v[near]).max()) + 2.0 ** -22 * near.sum() + 2.0 ** -50 * n * np.abs(v).max())
            assert (v[near].min(0) - slack <= got[b, j]).all() and (got[b, j] <= v[near].max(0) + slack).all(), (b, j)
            single += near.sum() == 1
    assert single > 0.3 * len(lens) * H
    assert torch.equal(out, ext().int4_decode_attention_paged(q, far, pool, table, ln, max(lens), page))
    ext().check_status()
