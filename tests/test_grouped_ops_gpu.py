"""Grouped-head operators on the GPU against their float64 restatements (oracle/grouped.py): q/k norm +
rotation (+ quantiser), the 4-bit paged cache, decode attention over it."""
import numpy as np
import pytest
import torch

from helpers import cabi, ext
from oracle import grouped as og

pytestmark = pytest.mark.gpu
TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _np(t):
    return t.float().cpu().numpy().astype(np.float64)


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _qk_inputs(T, H, kv, D, dtype, seed, reach=500, rotary=None):
    g = _gen(seed)
    x = (torch.randn(T, (H + 2 * kv) * D, device="cuda", generator=g) * 2).to(TYPES[dtype])
    pos = torch.randint(0, reach, (T,), device="cuda", generator=g, dtype=torch.int32)
    table = torch.from_numpy(og.rope_table(reach, rotary or D)).cuda()
    qw, kw = (1 + 0.3 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
    return x, pos, table, qw, kw


def _close_float(got, want, parts, dtype):
    """half a step of the type, and 2^-19 of the summands for the fp32 arithmetic (rsqrt, two products, a sum)"""
    half = torch.finfo(TYPES[dtype]).eps / 2
    tol = half * np.abs(want) * 1.001 + 2.0 ** -19 * parts + 2.0 ** -25
    assert (np.abs(got - want) <= tol).all(), np.abs(got - want).max()


@pytest.mark.parametrize("T,H,kv,D,rotary,interleaved,dtype,norm,rotate", [
    (1, 4, 1, 128, 128, False, "bf16", True, True), (3, 1, 1, 64, 32, True, "fp16", True, True), (37, 14, 2, 256, 256, False, "fp16", True, True),
    (5, 3, 3, 64, 64, False, "bf16", False, True), (130, 32, 8, 128, 64, False, "fp16", True, True), (9, 8, 2, 128, 16, True, "bf16", True, True),
    (7, 5, 1, 256, 128, False, "bf16", True, False), (2, 2, 2, 64, 64, False, "fp16", False, False), (64, 16, 4, 64, 48, False, "fp16", True, True)])
def test_qk_norm_rope(T, H, kv, D, rotary, interleaved, dtype, norm, rotate):
    e = ext()
    x, pos, table, qw, kw = _qk_inputs(T, H, kv, D, dtype, seed=T + D, rotary=rotary)
    args = (pos if rotate else None, table if rotate else None, qw if norm else None, kw if norm else None)
    host = [None if t is None else t.cpu().numpy() for t in args]
    want = og.qk_norm_rope(_np(x).reshape(T, H + 2 * kv, D), H, kv, *host, eps=1e-6, interleaved=interleaved)
    size = np.abs(want).max(-1, keepdims=True) * 2
    _close_float(_np(e.qk_norm_rope(x, H, kv, *args, 1e-6, interleaved)), want[:, :H + kv], size[:, :H + kv], dtype)

    k_out = torch.full((T, kv, D), 7.0, device="cuda", dtype=TYPES[dtype])
    codes, scales = e.qk_norm_rope_quantize(x, H, kv, *args, 1e-6, interleaved, k_out)
    assert codes.shape == (T, H + 2 * kv, D) and scales.shape == (T, H + 2 * kv)
    amax = np.abs(want).max(-1)
    assert np.allclose(_np(scales) * 127, np.maximum(amax, 1e-8), rtol=2.0 ** -18)
    # a code is the nearest integer to y / scale: half a step, and what fp32 may move a quotient of up to 127 by
    assert (np.abs(_np(codes) - want / _np(scales)[..., None]) <= 0.5 + 127 * 2.0 ** -17).all()
    _close_float(_np(k_out), want[:, H:H + kv], size[:, H:H + kv], dtype)


def test_qk_value_heads_are_the_per_token_quantiser_and_rows_may_be_strided():
    e = ext()
    T, H, kv, D = 53, 6, 2, 128
    wide = torch.randn(T, (H + 2 * kv) * D + 24, device="cuda", generator=_gen(3)).half()
    wide[7] = 0
    x = wide[:, 8:8 + (H + 2 * kv) * D]
    assert x.stride(0) % 8 == 0
    codes, scales = e.qk_norm_rope_quantize(x, H, kv)
    c2, s2 = e.quantize_per_token(x.contiguous().view(T, H + 2 * kv, D))
    assert torch.equal(codes, c2) and torch.equal(scales, s2)             # no norm, no rotation: the quantiser, bit for bit
    assert torch.equal(e.qk_norm_rope(x, H, kv), x.contiguous().view(T, H + 2 * kv, D)[:, :H + kv])


def test_qk_position_outside_the_table_shows_in_its_token_only():
    e = ext()
    x, pos, table, qw, kw = _qk_inputs(6, 4, 2, 64, "fp16", seed=5, rotary=32)
    good = e.qk_norm_rope(x, 4, 2, pos, table, qw, kw)
    gc, gs = e.qk_norm_rope_quantize(x, 4, 2, pos, table, qw, kw)
    bad = pos.clone()
    bad[2], bad[4] = 500, -1
    out = e.qk_norm_rope(x, 4, 2, bad, table, qw, kw)
    codes, scales = e.qk_norm_rope_quantize(x, 4, 2, bad, table, qw, kw)
    keep = [0, 1, 3, 5]
    assert torch.equal(out[keep], good[keep]) and torch.equal(codes[keep], gc[keep]) and torch.equal(scales[keep], gs[keep])
    assert out[[2, 4]][..., :32].isnan().all() and torch.equal(out[[2, 4]][..., 32:], good[[2, 4]][..., 32:])
    assert scales[[2, 4]][:, :6].isnan().all() and torch.equal(scales[[2, 4]][:, 6:], gs[[2, 4]][:, 6:])


def test_qk_no_tokens():
    e = ext()
    x = torch.empty(0, 8 * 64, device="cuda", dtype=torch.float16)
    assert e.qk_norm_rope(x, 4, 2).shape == (0, 6, 64)
    codes, scales = e.qk_norm_rope_quantize(x, 4, 2)
    assert codes.shape == (0, 8, 64) and scales.shape == (0, 8)


# ---- 4-bit cache ------------------------------------------------------------------------------------
def _pool(pages, kv, page, D, seed=0):
    n = ext().int4_kv_block_bytes(page, D)
    return torch.randint(0, 256, (pages, kv, n), dtype=torch.uint8, device="cuda", generator=_gen(seed))


@pytest.mark.parametrize("T,kv,D,page,dtype", [(1, 1, 64, 16, "fp16"), (17, 3, 128, 16, "bf16"), (200, 2, 64, 128, "fp16"), (77, 8, 128, 64, "fp16"),
                                               (33, 5, 64, 32, "bf16")])
def test_int4_append_is_bit_exact_and_touches_its_rows_only(T, kv, D, page, dtype):
    e = ext()
    g = _gen(T)
    k = (torch.randn(T, kv, D, device="cuda", generator=g) * torch.exp(2 * torch.randn(T, kv, 1, device="cuda", generator=g))).to(TYPES[dtype])
    v = torch.randn(T, kv, D, device="cuda", generator=g).to(TYPES[dtype])
    k[0] = 0.5                                                            # no spread: scale 0
    v[0, :, :64] = torch.arange(64, device="cuda").to(v.dtype) * 0.25     # ties between codes
    pages = T // page + 3
    pool = _pool(pages, kv, page, D)
    before = pool.clone()
    slots = torch.randperm(pages * page, device="cuda", generator=g)[:T]
    skip = torch.zeros(T, dtype=torch.bool)
    if T > 4:
        slots[3], slots[T - 1] = -1, pages * page                         # a padding row, and one past the pool
        skip[3] = skip[T - 1] = True
    e.kv_append_quantize_int4(k, v, pool, slots, page)
    want = before.cpu().numpy().copy()
    kn, vn, sl = k.float().cpu().numpy(), v.float().cpu().numpy(), slots.cpu().numpy()
    G = D // 64
    for t in range(T):
        if skip[t]:
            continue
        p, r = divmod(int(sl[t]), page)
        for h in range(kv):
            row = og.int4_block(kn[t, h][None], vn[t, h][None])           # codes k, codes v, pairs k, pairs v of one row
            b = want[p, h]
            b[r * D // 2:(r + 1) * D // 2] = row[:D // 2]
            b[(page + r) * D // 2:(page + r + 1) * D // 2] = row[D // 2:D]
            b[page * D + r * 4 * G:page * D + (r + 1) * 4 * G] = row[D:D + 4 * G]
            b[page * D + (page + r) * 4 * G:page * D + (page + r + 1) * 4 * G] = row[D + 4 * G:]
    assert np.array_equal(pool.cpu().numpy(), want)

    kd, vd = e.kv_dequantize_int4(pool, slots, page, D)
    for got, src in ((kd, kn), (vd, vn)):
        vals = og.int4_values(*og.int4_quantize(src)).astype(np.float16)
        vals[skip.numpy()] = 0
        assert np.array_equal(got.cpu().numpy(), vals)


def test_int4_append_takes_slices_of_a_projection_and_extreme_values():
    e = ext()
    T, kv, D, page = 19, 2, 128, 16
    qkv = torch.randn(T, 8 * D, device="cuda", generator=_gen(1)).bfloat16()
    k, v = qkv[:, 4 * D:6 * D].view(T, kv, D), qkv[:, 6 * D:].view(T, kv, D)
    k[3, 0, 5] = 1e30                                                     # saturates at the fp16 range
    k[4, 1, 7] = -float("inf")
    v[5, 0, 3] = float("nan")                                             # unspecified codes, but only in its group
    a, b = _pool(3, kv, page, D), _pool(3, kv, page, D)
    slots = torch.arange(T, device="cuda")
    e.kv_append_quantize_int4(k, v, a, slots, page)
    e.kv_append_quantize_int4(k.contiguous(), v.contiguous(), b, slots, page)
    assert torch.equal(a, b)
    kd, vd = e.kv_dequantize_int4(a, slots, page, D)
    assert torch.isfinite(kd.float()).all() and kd[3, 0, 5] > 6e4 and kd[4, 1, 7] < -6e4
    vn = v.float().cpu().numpy().copy()
    vn[5, 0, :64] = 0
    vals = og.int4_values(*og.int4_quantize(vn)).astype(np.float16)
    got = vd.cpu().numpy()
    got[5, 0, :64] = vals[5, 0, :64]
    assert np.array_equal(got, vals)


# ---- decode attention over it -----------------------------------------------------------------------
def _decode_case(B, H, kv, D, page, lens, seed, spread=1.0):
    """A pool whose unused pages and positions hold random bytes (their pairs may be NaN or infinite)."""
    g = _gen(seed)
    need = [-(-n // page) for n in lens]
    pages = sum(need) + 3
    pool = _pool(pages, kv, page, D, seed)
    order = torch.randperm(pages, device="cuda", generator=g)
    table = torch.full((B, max(1, max(need))), -12345, dtype=torch.int32, device="cuda")
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n].int()
        if lens[b]:
            pos = torch.arange(lens[b], device="cuda")
            slots = order[at + pos // page] * page + pos % page
            k = torch.randn(lens[b], kv, D, device="cuda", generator=g) * spread
            v = torch.randn(lens[b], kv, D, device="cuda", generator=g) + 0.5
            ext().kv_append_quantize_int4(k.half(), v.half(), pool, slots, page)
        at += n
    q, sq = ext().quantize_per_token(torch.randn(B, H, D, device="cuda", generator=g) * 1.5)
    return q, sq, pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda")


def _check_decode(out, q, sq, pool, table, lens, page, which=None):
    B, H, D = q.shape
    pn, tn, qn, sn, on = pool.cpu().numpy(), table.cpu().numpy(), q.cpu().numpy(), sq.cpu().numpy(), _np(out)
    kv = pn.shape[1]
    for b in (range(B) if which is None else which):
        n = int(lens[b])
        if n == 0:
            assert not on[b].any()
            continue
        both = ([], [])
        for h in range(kv):
            blocks = [og.int4_unblock(pn[p, h], page, D) for p in tn[b, :-(-n // page)]]
            for i in (0, 1):
                both[i].append([np.concatenate([blk[i][x] for blk in blocks])[:n] for x in range(3)])
        keys, values = ([np.stack([row[x] for row in both[i]]) for x in range(3)] for i in (0, 1))
        want, bound = og.int4_decode(qn[b], sn[b], keys, values)
        off = np.abs(on[b] - want)
        assert (off <= bound).all(), (b, n, (off / bound).max())


@pytest.mark.parametrize("H,kv,D,page,lens", [
    (1, 1, 64, 16, [1]), (8, 8, 64, 16, [5, 0, 129, 16]), (4, 1, 128, 32, [127, 128, 1]), (32, 8, 128, 16, [1000]), (24, 8, 64, 64, [300, 65, 2, 0, 700]),
    (16, 1, 128, 128, [513, 64, 0]), (16, 1, 64, 32, [1025, 31]), (14, 2, 128, 64, [4097]), (9, 1, 128, 16, [3, 260]), (15, 5, 64, 128, [1, 1, 2, 128, 129]),
    (32, 2, 128, 16, [777, 12])])
def test_int4_decode(H, kv, D, page, lens):
    e = ext()
    q, sq, pool, table, ln = _decode_case(len(lens), H, kv, D, page, lens, seed=H + D)
    out = e.int4_decode_attention_paged(q, sq, pool, table, ln, max(lens), page)
    _check_decode(out, q, sq, pool, table, lens, page)
    assert torch.equal(out, e.int4_decode_attention_paged(q, sq, pool, table, ln, max(lens), page))
    e.check_status()


def test_int4_decode_many_requests_and_one_long():
    e = ext()
    rng = np.random.default_rng(4)
    lens = [int(x) for x in rng.integers(0, 200, 700)]
    lens[350], lens[699], lens[0] = 20011, 0, 0
    q, sq, pool, table, ln = _decode_case(len(lens), 4, 2, 64, 16, lens, seed=8, spread=3.0)
    out = e.int4_decode_attention_paged(q, sq, pool, table, ln, max(lens), 16)
    _check_decode(out, q, sq, pool, table, lens, 16, which=[0, 1, 2, 349, 350, 351, 500, 698, 699])
    for b in (3, 350, 600):                                                # alone, the runs are others
        one = e.int4_decode_attention_paged(q[b:b + 1], sq[b:b + 1], pool, table[b:b + 1].contiguous(), ln[b:b + 1], lens[b], 16)
        _check_decode(one, q[b:b + 1], sq[b:b + 1], pool, table[b:b + 1], [lens[b]], 16)


def test_int4_decode_peaked_and_flat_scores():
    """Scores far apart (one key takes all) and all equal (long sums of small probabilities)."""
    e = ext()
    for spread, seed in ((40.0, 1), (0.0, 2)):
        lens = [3000, 17]
        q, sq, pool, table, ln = _decode_case(2, 8, 2, 128, 32, lens, seed=seed, spread=spread)
        out = e.int4_decode_attention_paged(q, sq, pool, table, ln, 3000, 32)
        _check_decode(out, q, sq, pool, table, lens, 32)


def test_int4_decode_strided_queries_loose_bound_and_damaged_tables():
    e = ext()
    lens = [300, 90, 257]
    q, sq, pool, table, ln = _decode_case(3, 8, 2, 64, 16, lens, seed=23)
    good = e.int4_decode_attention_paged(q, sq, pool, table, ln, 300, 16)
    wide = torch.zeros(3, 12, 64, dtype=torch.int8, device="cuda")
    wide[:, :8] = q
    wsq = torch.full((3, 12), float("nan"), device="cuda")
    wsq[:, :8] = sq
    assert torch.equal(good, e.int4_decode_attention_paged(wide[:, :8], wsq[:, :8], pool, table, ln, 300, 16))
    loose = e.int4_decode_attention_paged(q, sq, pool, table, ln, table.size(1) * 16, 16)
    _check_decode(loose, q, sq, pool, table, lens, 16)
    torch.cuda.synchronize()
    e.check_status()

    bad = table.clone()
    bad[1, 2], bad[1, 4] = pool.size(0) + 1000, -7                         # never followed: page 0 is read in their place
    out = e.int4_decode_attention_paged(q, sq, pool, bad, ln, 300, 16)
    torch.cuda.synchronize()
    assert torch.equal(out[[0, 2]], good[[0, 2]])
    with pytest.raises(RuntimeError, match="page id"):
        e.check_status()
    odd = torch.tensor([300, -5, 10 ** 6], dtype=torch.int32, device="cuda")  # read as 300, 0 and the bound
    out = e.int4_decode_attention_paged(q, sq, pool, table, odd, 257, 16)
    torch.cuda.synchronize()
    assert not out[1].any()
    _check_decode(out[2:], q[2:], sq[2:], pool, table[2:], [257], 16)
    e.check_status()


def test_int4_decode_status_word_belongs_to_the_call():
    """Through the C ABI: word 0 of the workspace is set by a call that met a bad page and cleared by the next."""
    c, lib = cabi(), cabi().load()
    q, sq, pool, table, ln = _decode_case(1, 4, 1, 64, 16, [40], seed=3)
    n = lib.i8tk_decode_kv4_workspace_bytes(1, 4, 1, 40, 64)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")           # nothing in it is relied on
    out = torch.empty(1, 4, 64, dtype=torch.float16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    bad = table.clone()
    bad[0, 1] = 99
    for tab, want in ((bad, c.ERR_INVALID_ARGUMENT), (table, c.OK)):
        c.check(lib.i8tk_decode_attention_kv4(q.data_ptr(), 256, sq.data_ptr(), 4, pool.data_ptr(), tab.data_ptr(), ln.data_ptr(), out.data_ptr(),
                                              1, 4, 1, 40, 16, table.size(1), 64, pool.size(0), ws.data_ptr(), n, st))
        assert lib.i8tk_check_status_word(ws.data_ptr(), st) == want
    _check_decode(out, q, sq, pool, table, [40], 16)
