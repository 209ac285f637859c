"""Float64 restatements of the grouped-head operators, written from their formulas (numpy only).

Test infrastructure like the rest of this directory: the package does not import it.
"""
import numpy as np


def rope_table(rows, rotary, base=10000.0):
    """fp32 [rows, rotary]: cosines of the rotary/2 frequencies, then their sines (angles in 64 bits)."""
    inv = base ** (-np.arange(0, rotary, 2) / rotary)
    angle = np.arange(rows)[:, None] * inv
    return np.concatenate([np.cos(angle), np.sin(angle)], axis=1).astype(np.float32)


def qk_norm_rope(x, heads, kv_heads, positions=None, table=None, q_weight=None, k_weight=None, eps=1e-6, interleaved=False):
    """x [T, heads + 2 kv_heads, D] float64 -> the same with query and key heads normed and rotated."""
    y = np.array(x, dtype=np.float64)
    last = heads + kv_heads
    if q_weight is not None:
        for at, n, w in ((0, heads, q_weight), (heads, kv_heads, k_weight)):
            part = y[:, at:at + n]
            y[:, at:at + n] = part / np.sqrt((part ** 2).mean(-1, keepdims=True) + eps) * np.asarray(w, dtype=np.float64)
    if positions is not None:
        row = np.asarray(table, dtype=np.float64)[np.asarray(positions)][:, None]
        r = row.shape[-1]
        cos, sin = row[..., :r // 2], row[..., r // 2:]
        a_at, b_at = (slice(0, r, 2), slice(1, r, 2)) if interleaved else (slice(0, r // 2), slice(r // 2, r))
        a, b = y[:, :last, a_at].copy(), y[:, :last, b_at].copy()
        y[:, :last, a_at] = a * cos - b * sin
        y[:, :last, b_at] = b * cos + a * sin
    return y


def int4_quantize(x):
    """Rows [..., D] -> (codes 0..15 [..., D], scale fp16 [..., D/64], centre fp16 [..., D/64])."""
    x = np.clip(np.asarray(x, dtype=np.float32), -65504, 65504)
    v = x.reshape(*x.shape[:-1], -1, 64)
    lo, hi = v.min(-1), v.max(-1)
    s = ((hi - lo) / np.float32(15)).astype(np.float16)
    z = (lo + np.float32(8) * s.astype(np.float32)).astype(np.float16)
    sf, zf = s.astype(np.float32)[..., None], z.astype(np.float32)[..., None]
    n = np.rint(np.divide(v - zf, sf, out=np.zeros_like(v), where=sf > 0))
    return (np.clip(n, -8, 7) + 8).astype(np.uint8).reshape(x.shape), s, z


def int4_values(codes, s, z):
    """float64 values of codes [..., D] under (scale, centre) [..., D/64]."""
    rep = lambda t: np.repeat(np.asarray(t, dtype=np.float64), 64, axis=-1)  # noqa: E731
    return (codes.astype(np.float64) - 8) * rep(s) + rep(z)


def int4_pack_row(codes):
    """Codes [..., D] -> bytes [..., D/2]: word u*G + g of a row holds channels 64g + 8u .. + 7, lowest nibble first."""
    g = codes.shape[-1] // 64
    c = codes.reshape(*codes.shape[:-1], g, 8, 4, 2)
    return np.ascontiguousarray(np.moveaxis(c[..., 0] | (c[..., 1] << 4), -3, -2)).reshape(*codes.shape[:-1], -1)


def int4_block(k, v):
    """One page of one key head: k, v [page, D] -> its bytes."""
    parts, pairs = [], []
    for x in (k, v):
        c, s, z = int4_quantize(x)
        parts.append(int4_pack_row(c).reshape(-1))
        pairs.append(np.ascontiguousarray(np.stack([s, z], axis=-1)).view(np.uint8).reshape(-1))
    return np.concatenate(parts + pairs)


def int4_unblock(block, page, head_dim):
    """Bytes of one block -> ((codes, scale, centre) of the keys, the same of the values)."""
    g, n = head_dim // 64, page * head_dim // 2
    out = []
    for i in (0, 1):
        b = block[i * n:(i + 1) * n].reshape(page, 8, g, 4)
        codes = np.stack([b & 15, b >> 4], axis=-1).reshape(page, 8, g, 8)
        codes = np.moveaxis(codes, 2, 1).reshape(page, head_dim)
        at = 2 * n + i * page * g * 4
        pair = np.ascontiguousarray(block[at:at + page * g * 4]).view(np.float16).reshape(page, g, 2)
        out.append((codes, pair[..., 0], pair[..., 1]))
    return out


def softmax_rows(s):
    """exp(s - max) and its sum along the last axis; rows of -inf give zeros and sum 1."""
    m = s.max(-1, keepdims=True)
    p = np.exp(s - np.where(np.isfinite(m), m, 0.0))
    l = p.sum(-1, keepdims=True)
    return p, np.where(l > 0, l, 1.0)


def int4_decode(q, sq, keys, values):
    """One request: q [H, D] codes, sq [H]; keys, values: (codes [kv, L, D], scale, centre [kv, L, D/64]).
    Returns (out [H, D], bound [H, D]): the bound is what fp16 probabilities and an fp16 result may be off by --
    half a step (2^-11) of each p * scale, of which (code - 8) go into the sum, and of the result; plus half the
    smallest fp16 number for each p * scale below the normal range, the sum of p being at least a quarter of the
    sum over the true maximum (the kernel's reference may trail the maximum by 2 log2 units); 5 % for fp32 rounding
    of scores and the exponential (relative 2^-20 each, against 2^-11)."""
    H, D = q.shape
    kv = keys[0].shape[0]
    k, v = int4_values(*keys), int4_values(*values)
    qf = (q.astype(np.float64) * np.asarray(sq, dtype=np.float64)[:, None]).reshape(kv, H // kv, D)
    p, l = softmax_rows(np.einsum("hgd,hjd->hgj", qf, k) / np.sqrt(D))
    out = np.einsum("hgj,hjd->hgd", p, v) / l
    weight = np.repeat(values[1].astype(np.float64), 64, axis=-1)
    step = np.abs(values[0].astype(np.float64) - 8)
    spread = np.einsum("hgj,hjd->hgd", p, weight * step) / l
    tiny = 2.0 ** -25 * 4 * step.sum(1)[:, None] / l
    bound = 1.05 * (2.0 ** -11 * (spread + np.abs(out)) + tiny + 2.0 ** -25)
    return out.reshape(H, D), bound.reshape(H, D)


def varlen_attention(q, k, v, sq, sk, sv, cu, causal=True):
    """Packed INT8 attention: q [T, H, D], k, v [T, kv, D] codes, scales per row.  Returns (out [T, H, D], bound):
    half a step of every fp16 p * scale (2^-11 of the sum of p |v|) and of the fp16 result, with 5 % for the fp32
    parts; for products below the fp16 range 2^-31 of the sequence's largest |v| for each key (p * scale is scaled
    so that the largest scale of the sequence is at least 2^6, and half the smallest fp16 number is 2^-25); and for
    the three fp32 roundings of a score s, which move its probability by 3 * 2^-24 * |s| and the sum by as much."""
    T, H, D = q.shape
    kv = k.shape[1]
    out, bound = np.zeros((T, H, D)), np.zeros((T, H, D))
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        for h in range(kv if n > 0 else 0):
            at = slice(h * (H // kv), (h + 1) * (H // kv))
            qf = q[a:b, at].astype(np.float64) * sq[a:b, at, None].astype(np.float64)
            kf = k[a:b, h].astype(np.float64) * sk[a:b, h, None].astype(np.float64)
            vf = v[a:b, h].astype(np.float64) * sv[a:b, h, None].astype(np.float64)
            s = np.einsum("igd,jd->gij", qf, kf) / np.sqrt(D)
            if causal:
                s = np.where(np.arange(n)[None, :] <= np.arange(n)[:, None], s, -np.inf)
            p, l = softmax_rows(s)
            o = np.einsum("gij,jd->gid", p / l, vf)
            spread = np.einsum("gij,jd->gid", p / l, np.abs(vf))
            size = np.abs(np.where(np.isfinite(s), s, 0.0)).max(-1, keepdims=True)
            tiny = 2.0 ** -25 * n * 127 * float(sv[a:b, h].max()) / 64 / l
            out[a:b, at] = o.transpose(1, 0, 2)
            step = 2.0 ** -11 + 3 * 2.0 ** -24 * size
            bound[a:b, at] = (1.05 * (step * (spread + np.abs(o)) + tiny + 2.0 ** -25)).transpose(1, 0, 2)
    return out, bound
