"""The grouped-head INT8 / 4-bit serving operators: cases, plain forms, and what each has to move.

Four operators, in the order a layer uses them:

  qk        per-head RMS norm of queries and keys, position rotation and (in the quantised form) the
            per-token INT8 quantiser, in one pass over the fused QKV projection
  varlen    INT8 attention over packed prompts of different lengths with grouped heads
  append    new key and value rows into a paged cache held in 4 bits (and read back as values)
  decode    attention of one query token per request over that cache

A cache block holds one page of one key/value head: the keys' codes [page, D/2], the values' codes
[page, D/2], then (scale, centre) fp16 pairs [page, D/64, 2] of the keys and of the values.  A value is
scale * (code - 8) + centre, one pair for 64 consecutive channels.  Byte 4*(u*G + g) + b of a row (G = D/64,
u = 0..7) holds channels 64*g + 8*u + 2*b (low nibble) and + 2*b + 1 (high nibble).
"""
import math

import numpy as np
import torch

own = False


def _ops():
    import importlib
    return importlib.import_module("int8-transformer-kernels_b200").int8_ext


# ---- cases ------------------------------------------------------------------------------------------
def listed():
    return [
        # one token of one request: what latency costs before attention in a decode step
        dict(name="qk_one_token", op="qk", tokens=1, heads=32, kv_heads=8, head_dim=128, dtype="bf16", quant=False,
             rotary=128, interleaved=False, norm=True, reach=32768),
        # a decode batch of a smaller model, half of each head rotated, neighbouring pairs
        dict(name="qk_batch_64", op="qk", tokens=61, heads=24, kv_heads=8, head_dim=64, dtype="fp16", quant=True,
             rotary=32, interleaved=True, norm=True, reach=8192),
        # a packed prompt of 8 thousand tokens on its way into INT8 attention
        dict(name="qk_prompt_8k", op="qk", tokens=8192, heads=32, kv_heads=8, head_dim=128, dtype="bf16", quant=True,
             rotary=128, interleaved=False, norm=True, reach=131072),
        # a handful of short chat turns, ordinary heads
        dict(name="varlen_short", op="varlen", seqs=5, longest=67, mix="mixed", heads=12, kv_heads=12, head_dim=64, causal=True),
        # a prefill batch of a server: sixteen prompts of different lengths
        dict(name="varlen_mixed", op="varlen", seqs=16, longest=2048, mix="mixed", heads=32, kv_heads=8, head_dim=128, causal=True),
        # one long document
        dict(name="varlen_long", op="varlen", seqs=1, longest=8192, mix="equal", heads=32, kv_heads=8, head_dim=128, causal=True),
        # an encoder's batch: no causal mask, odd lengths, wide heads, seven query heads on one key head
        dict(name="varlen_encoder", op="varlen", seqs=6, longest=1111, mix="mixed", heads=14, kv_heads=2, head_dim=256, causal=False),
        # the new tokens of a decode step
        dict(name="append_32", op="append", tokens=32, kv_heads=8, head_dim=128, page=64, dtype="bf16"),
        # a prompt's keys and values into the cache
        dict(name="append_prompt_16k", op="append", tokens=16384, kv_heads=8, head_dim=128, page=16, dtype="fp16"),
        # one request with a short history: latency
        dict(name="decode_one", op="decode", seqs=1, longest=1000, mix="equal", heads=32, kv_heads=8, head_dim=128, page=16),
        # an ordinary batch with as many key heads as query heads
        dict(name="decode_mha", op="decode", seqs=24, longest=4096, mix="mixed", heads=12, kv_heads=12, head_dim=64, page=32),
        # a full server: 32 requests, histories up to 32 thousand positions
        dict(name="decode_32k", op="decode", seqs=32, longest=32768, mix="mixed", heads=32, kv_heads=8, head_dim=128, page=64),
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _groups(rng, most):
    """(query heads, key heads) with at most `most` query heads on a key head."""
    kv = rng.choice([1, 2, 4, 8, 12])
    return kv * rng.choice([g for g in (1, 2, 3, 4, 5, 7, 8, 16) if g <= most and kv * g <= 64]), kv


def draw(rng):
    op = rng.choice(["qk", "varlen", "append", "decode"])
    mix = rng.choice(["mixed", "equal"])
    if op == "qk":
        heads, kv = _groups(rng, 16)
        d = rng.choice([64, 128, 256])
        most = max(1, 8192 * 48 * 128 // ((heads + 2 * kv) * d))
        return dict(op=op, tokens=_log(rng, 1, min(most, 30000)), heads=heads, kv_heads=kv, head_dim=d, dtype=rng.choice(["fp16", "bf16"]),
                    quant=rng.random() < 0.5, rotary=rng.choice([d, d // 2]), interleaved=rng.random() < 0.3, norm=rng.random() < 0.8,
                    reach=_log(rng, 64, 131072))
    if op == "varlen":
        heads, kv = _groups(rng, 16)
        seqs, d = _log(rng, 1, 24), rng.choice([64, 128, 128, 256])
        most = min(8192, int(math.sqrt(2.0e9 * min(1.0, 128 / d) / (seqs * heads))))
        return dict(op=op, seqs=seqs, longest=_log(rng, 1, most), mix=mix, heads=heads, kv_heads=kv, head_dim=d, causal=rng.random() < 0.8)
    if op == "append":
        kv, d = rng.choice([1, 2, 4, 8, 12]), rng.choice([64, 128])
        return dict(op=op, tokens=_log(rng, 1, 16384 * 8 * 128 // (kv * d) if kv * d > 512 else 20000), kv_heads=kv, head_dim=d,
                    page=rng.choice([16, 32, 64, 128]), dtype=rng.choice(["fp16", "bf16"]))
    heads, kv = _groups(rng, 16)
    seqs, d = _log(rng, 1, 64), rng.choice([64, 128])
    most = min(65536, 16 * 32768 * 8 * 128 // (seqs * kv * d))
    return dict(op=op, seqs=seqs, longest=_log(rng, 1, most), mix=mix, heads=heads, kv_heads=kv, head_dim=d, page=rng.choice([16, 32, 64, 128]))


def _lengths(case):
    """The sequences' lengths: all the longest, or spread evenly over the range in a fixed shuffled order."""
    n, longest = case["seqs"], case["longest"]
    if case["mix"] == "equal":
        return [longest] * n
    return [longest if i == 0 else max(1, math.ceil(longest * ((0.618033988749895 * i) % 1.0))) for i in range(n)]


# ---- inputs -----------------------------------------------------------------------------------------
_TYPES = {"fp16": torch.float16, "bf16": torch.bfloat16}


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(int(seed) & 0x7FFFFFFF)


def _randn(g, *shape, dtype=torch.float32):
    return torch.randn(*shape, device="cuda", generator=g, dtype=torch.float32).to(dtype)


def _int8_rows(x):
    """Symmetric INT8 codes of the rows of x and their fp32 scales."""
    scale = x.abs().amax(dim=-1).clamp_min(1e-8) / 127.0
    return torch.round(x / scale[..., None]).clamp_(-127, 127).to(torch.int8), scale


def _int4_rows(x):
    """(packed codes uint8 [..., D/2], (scale, centre) fp16 [..., D/64, 2]) of rows x [..., D]."""
    v = x.float().unflatten(-1, (-1, 64))
    low, high = v.amin(dim=-1), v.amax(dim=-1)
    scale = ((high - low) / torch.full_like(low, 15.0)).half()
    centre = (low + 8.0 * scale.float()).half()
    s, z = scale.float()[..., None], centre.float()[..., None]
    code = torch.where(s > 0, torch.round((v - z) / s), torch.zeros_like(v)).add_(8).clamp_(0, 15).to(torch.uint8)
    pairs = code.unflatten(-1, (8, 4, 2))                                    # [..., G, u, b, 2]
    packed = (pairs[..., 0] | (pairs[..., 1] << 4)).transpose(-3, -2)        # [..., u, G, b]
    return packed.flatten(-3), torch.stack([scale, centre], dim=-1)


def _norm_weight(g, d):
    return 1.0 + 0.2 * _randn(g, d)


def _rope(reach, rotary):
    """cos | sin of every position and frequency, angles in 64 bits."""
    inv = 10000.0 ** (-torch.arange(0, rotary, 2, device="cuda", dtype=torch.float64) / rotary)
    angle = torch.arange(reach, device="cuda", dtype=torch.float64)[:, None] * inv
    return torch.cat([angle.cos(), angle.sin()], dim=1).float().contiguous()


def prepare(case, seed):
    g = _gen(seed)
    op, d = case["op"], case["head_dim"]
    st = dict(case=case)
    if op == "qk":
        t, heads, kv = case["tokens"], case["heads"], case["kv_heads"]
        gain = torch.exp(0.3 * _randn(g, (heads + 2 * kv) * d))
        st["qkv"] = (_randn(g, t, (heads + 2 * kv) * d) * gain).to(_TYPES[case["dtype"]])
        st["positions"] = torch.randint(0, case["reach"], (t,), device="cuda", generator=g, dtype=torch.int32)
        st["rope"] = _rope(case["reach"], case["rotary"])
        st["q_weight"] = _norm_weight(g, d) if case["norm"] else None
        st["k_weight"] = _norm_weight(g, d) if case["norm"] else None
    elif op == "varlen":
        lens = _lengths(case)
        t, heads, kv = sum(lens), case["heads"], case["kv_heads"]
        gain = torch.exp(0.3 * _randn(g, d))
        st["q"], st["sq"] = _int8_rows(_randn(g, t, heads, d) * gain)
        st["k"], st["sk"] = _int8_rows(_randn(g, t, kv, d) * gain)
        st["v"], st["sv"] = _int8_rows(_randn(g, t, kv, d) * torch.exp(0.3 * _randn(g, t, kv, 1)))
        st["cu"] = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    elif op == "append":
        t, kv, page = case["tokens"], case["kv_heads"], case["page"]
        gain = torch.exp(0.3 * _randn(g, kv, d))
        st["k"] = (_randn(g, t, kv, d) * gain).to(_TYPES[case["dtype"]])
        st["v"] = (_randn(g, t, kv, d) * torch.exp(0.3 * _randn(g, t, 1, 1))).to(_TYPES[case["dtype"]])
        pages = -(-t // page) + 2
        st["pool"] = torch.zeros(pages, kv, page * (d + d // 8), dtype=torch.uint8, device="cuda")
        order = torch.randperm(pages, device="cuda", generator=g)
        at = torch.arange(t, device="cuda")
        st["slots"] = order[at // page] * page + at % page
    else:
        lens = _lengths(case)
        n, longest, kv, page = len(lens), case["longest"], case["kv_heads"], case["page"]
        need = [-(-x // page) for x in lens]
        pages = sum(need) + 1
        order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
        table = torch.zeros(n, max(need), dtype=torch.int32, device="cuda")
        fits = torch.arange(max(need), device="cuda")[None, :] < torch.tensor(need, device="cuda")[:, None]
        table[fits] = order[: sum(need)]
        st["table"], st["lens"] = table, torch.tensor(lens, dtype=torch.int32, device="cuda")
        gain = torch.exp(0.3 * _randn(g, d))
        st["pool"] = _random_pool(g, pages, kv, page, d, gain)
        st["q"], st["sq"] = _int8_rows(_randn(g, n, case["heads"], d) * gain)
    return st


def _random_pool(g, pages, kv, page, d, gain):
    pool = torch.empty(pages, kv, page * (d + d // 8), dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 27) // (kv * page * d))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        kc, km = _int4_rows(torch.randn(n, kv, page, d, device="cuda", generator=g) * gain)
        vc, vm = _int4_rows(torch.randn(n, kv, page, d, device="cuda", generator=g))
        pool[at:at + n] = torch.cat([kc.flatten(2), vc.flatten(2), km.flatten(2).view(torch.uint8), vm.flatten(2).view(torch.uint8)], dim=2)
    return pool


# ---- one pass ---------------------------------------------------------------------------------------
def run(st):
    op = st["case"]["op"]
    if own:
        return {"qk": _own_qk, "varlen": _own_varlen, "append": _own_append, "decode": _own_decode}[op](st)
    return {"qk": _plain_qk, "varlen": _plain_varlen, "append": _plain_append, "decode": _plain_decode}[op](st)


def _own_qk(st):
    c, ops = st["case"], _ops()
    args = (st["qkv"], c["heads"], c["kv_heads"], st["positions"], st["rope"], st["q_weight"], st["k_weight"], 1e-6, c["interleaved"])
    if not c["quant"]:
        return ops.qk_norm_rope(*args)
    codes, scales = ops.qk_norm_rope_quantize(*args)
    return ops.dequantize_per_token(codes, scales)


def _own_varlen(st):
    c = st["case"]
    return _ops().int8_attention_varlen(st["q"], st["k"], st["v"], st["sq"], st["sk"], st["sv"], st["cu"], c["longest"], c["causal"])


def _own_append(st):
    c, ops = st["case"], _ops()
    ops.kv_append_quantize_int4(st["k"], st["v"], st["pool"], st["slots"], c["page"])
    return ops.kv_dequantize_int4(st["pool"], st["slots"], c["page"], c["head_dim"])


def _own_decode(st):
    c = st["case"]
    return _ops().int4_decode_attention_paged(st["q"], st["sq"], st["pool"], st["table"], st["lens"], c["longest"], c["page"])


def _rotate(x, cos, sin, interleaved):
    """x [T, H, R] with cos, sin [T, 1, R/2]."""
    if interleaved:
        a, b = x[..., 0::2], x[..., 1::2]
        return torch.stack([a * cos - b * sin, b * cos + a * sin], dim=-1).flatten(-2)
    a, b = x.chunk(2, dim=-1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], dim=-1)


def _plain_qk(st):
    c = st["case"]
    heads, kv, d, rotary = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"]
    x = st["qkv"].float().unflatten(-1, (-1, d))
    qk, v = x[:, :heads + kv], x[:, heads + kv:]
    if c["norm"]:
        weight = torch.cat([st["q_weight"].expand(heads, d), st["k_weight"].expand(kv, d)])
        qk = qk * torch.rsqrt(qk.square().mean(dim=-1, keepdim=True) + 1e-6) * weight
    cos, sin = st["rope"][st["positions"].long()][:, None].chunk(2, dim=-1)
    qk = torch.cat([_rotate(qk[..., :rotary], cos, sin, c["interleaved"]), qk[..., rotary:]], dim=-1)
    if not c["quant"]:
        return qk.to(st["qkv"].dtype)
    y = torch.cat([qk, v], dim=1)
    scale = y.abs().amax(dim=-1, keepdim=True).clamp_min(1e-8) / torch.full((1,), 127.0, device=y.device)
    return (torch.round(y / scale).clamp_(-127, 127) * scale).half()


def _plain_varlen(st):
    c = st["case"]
    kv, d, longest = c["kv_heads"], c["head_dim"], c["longest"]
    group = c["heads"] // kv
    start, count = st["cu"][:-1].long(), st["cu"].long().diff()
    at = torch.arange(longest, device="cuda")
    valid = at[None, :] < count[:, None]                                      # [B, L]
    rows = (start[:, None] + at).clamp_max(st["q"].size(0) - 1)
    q = (st["q"].float() * st["sq"][..., None])[rows].unflatten(2, (kv, group)).permute(0, 2, 3, 1, 4).flatten(2, 3)   # [B, kv, g*L, d]
    k = (st["k"].float() * st["sk"][..., None])[rows].permute(0, 2, 3, 1)     # [B, kv, d, L]
    v = (st["v"].float() * st["sv"][..., None])[rows].transpose(1, 2)         # [B, kv, L, d]
    s = (q @ k).mul_(1.0 / math.sqrt(d))
    gone = ~valid[:, None, None, None, :]
    if c["causal"]:
        gone = gone | (at[None, :] > at[:, None])
    s.unflatten(2, (group, longest)).masked_fill_(gone, -math.inf)
    s.sub_(s.amax(dim=-1, keepdim=True)).exp_()
    o = (s @ v).div_(s.sum(dim=-1, keepdim=True))
    o = o.unflatten(2, (group, longest)).permute(0, 3, 1, 2, 4).flatten(2, 3)  # [B, L, heads, d]
    return o[valid].half()


def _plain_append(st):
    k, v = st["k"], st["v"]
    x = torch.stack([k, v]).float().unflatten(-1, (-1, 64))
    low, high = x.amin(dim=-1, keepdim=True), x.amax(dim=-1, keepdim=True)
    scale = ((high - low) / torch.full_like(low, 15.0)).half().float()
    centre = (low + 8.0 * scale).half().float()
    code = torch.where(scale > 0, torch.round((x - centre) / scale), torch.zeros_like(x)).clamp_(-8, 7)
    both = (code * scale + centre).flatten(-2).half()
    return both[0], both[1]


def _unpack(codes, pairs):
    """fp32 rows [..., D] of packed codes [..., D/2] and (scale, centre) pairs [..., G, 2]."""
    g = pairs.size(-2)
    b = codes.unflatten(-1, (8, g, 4)).transpose(-3, -2)                       # [..., G, u, b]
    code = torch.stack([b & 15, b >> 4], dim=-1).flatten(-3).float()           # [..., G, 64]
    s, z = pairs.float().unbind(-1)
    return code.sub_(8).mul_(s[..., None]).add_(z[..., None]).flatten(-2)


def _plain_decode(st):
    c = st["case"]
    n, kv, d, page, longest = c["seqs"], c["kv_heads"], c["head_dim"], c["page"], c["longest"]
    block = st["pool"][st["table"].long()].transpose(1, 2)                     # [B, kv, pages, bytes]
    kc, vc, km, vm = block.split([page * d // 2, page * d // 2, page * d // 16, page * d // 16], dim=-1)

    def rows(codes, pairs):
        pairs = pairs.contiguous().view(torch.float16).unflatten(-1, (page, d // 64, 2))
        return _unpack(codes.unflatten(-1, (page, d // 2)), pairs).flatten(2, 3)[:, :, :longest]

    q = (st["q"].float() * st["sq"][..., None]).unflatten(1, (kv, -1))         # [B, kv, g, d]
    s = (q @ rows(kc, km).transpose(2, 3)).mul_(1.0 / math.sqrt(d))
    s.masked_fill_((torch.arange(longest, device="cuda") >= st["lens"][:, None])[:, None, None], -math.inf)
    p = s.sub_(s.amax(dim=-1, keepdim=True)).exp_()
    return (p @ rows(vc, vm)).div_(p.sum(dim=-1, keepdim=True)).flatten(1, 2).half()


# ---- what a pass cannot do without ------------------------------------------------------------------
def work(case):
    d, op = case["head_dim"], case["op"]
    if op == "qk":
        rows = case["tokens"] * (case["heads"] + case["kv_heads"])
        every = rows + case["tokens"] * case["kv_heads"]
        table = min(case["tokens"], case["reach"]) * case["rotary"] * 4
        if case["quant"]:
            return {"bytes": every * d * 4 + table, "flops": every * d * 12.0}
        return {"bytes": rows * d * 4 + table, "flops": rows * d * 10.0}
    if op == "varlen":
        lens = _lengths(case)
        pairs = sum(x * (x + 1) // 2 if case["causal"] else x * x for x in lens)
        t, h, kv = sum(lens), case["heads"], case["kv_heads"]
        return {"bytes": t * (h * (3 * d + 4) + 2 * kv * (d + 4)), "flops": 4.0 * d * h * pairs}
    if op == "append":
        rows = case["tokens"] * case["kv_heads"] * 2
        return {"bytes": rows * (2 * d + d / 2 + d / 16 + 2 * d) + case["tokens"] * 8, "flops": rows * d * 8.0}
    at = sum(_lengths(case))
    return {"bytes": at * case["kv_heads"] * (d + d // 8) + case["seqs"] * case["heads"] * (3 * d + 4), "flops": 4.0 * d * case["heads"] * at}


# ---- the definitions in 64 bits ---------------------------------------------------------------------
def exact(case, seed):
    st = prepare(case, seed)
    return {"qk": _exact_qk, "varlen": _exact_varlen, "append": _exact_append, "decode": _exact_decode}[case["op"]](st)


def _exact_qk(st):
    c = st["case"]
    h, kv, d, r = c["heads"], c["kv_heads"], c["head_dim"], c["rotary"]
    x = st["qkv"].double().view(c["tokens"], h + 2 * kv, d).clone()
    if c["norm"]:
        for lo, n, w in ((0, h, st["q_weight"]), (h, kv, st["k_weight"])):
            y = x[:, lo:lo + n]
            x[:, lo:lo + n] = y / torch.sqrt(y.pow(2).sum(-1, keepdim=True) / d + 1e-6) * w.double()
    row = st["rope"].double()[st["positions"].long()]
    turn = torch.complex(row[:, :r // 2], row[:, r // 2:])[:, None]            # a pair as a complex number
    head = x[:, :h + kv, :r]
    first, second = (head[..., 0::2], head[..., 1::2]) if c["interleaved"] else (head[..., :r // 2], head[..., r // 2:])
    z = torch.complex(first, second) * turn
    if c["interleaved"]:
        x[:, :h + kv, 0:r:2], x[:, :h + kv, 1:r:2] = z.real, z.imag
    else:
        x[:, :h + kv, :r // 2], x[:, :h + kv, r // 2:r] = z.real, z.imag
    if not c["quant"]:
        return x[:, :h + kv]
    step = x.abs().amax(-1, keepdim=True).clamp_min(1e-8) / 127
    return torch.round(x / step) * step


def _exact_varlen(st):
    c = st["case"]
    kv, d = c["kv_heads"], c["head_dim"]
    g, cu = c["heads"] // kv, st["cu"].tolist()
    out = torch.zeros(cu[-1], c["heads"], d, dtype=torch.float64, device="cuda")
    for a, b in zip(cu[:-1], cu[1:]):
        n = b - a
        for h in range(kv):
            k = st["k"][a:b, h].double() * st["sk"][a:b, h, None].double()
            v = st["v"][a:b, h].double() * st["sv"][a:b, h, None].double()
            q = st["q"][a:b, h * g:(h + 1) * g].double() * st["sq"][a:b, h * g:(h + 1) * g, None].double()
            s = torch.einsum("igd,jd->gij", q, k) / math.sqrt(d)
            if c["causal"]:
                s += torch.full((n, n), -math.inf, dtype=torch.float64, device="cuda").triu(1)
            out[a:b, h * g:(h + 1) * g] = torch.einsum("gij,jd->igd", torch.softmax(s, dim=-1), v)
    return out


def _exact_append(st):
    both = []
    for x in (st["k"], st["v"]):
        y = x.double().view(*x.shape[:-1], -1, 64)
        top, bottom = y.max(-1, keepdim=True).values, y.min(-1, keepdim=True).values
        s = ((top - bottom) / torch.tensor(15.0, dtype=torch.float64, device="cuda")).half().double()
        z = (bottom + 8 * s).half().double()
        n = torch.round((y - z) / s.clamp_min(1e-30)).clamp(-8, 7)
        both.append((z + n * s).view(x.shape))
    return both[0], both[1]


def _exact_decode(st):
    c = st["case"]
    kv, d, page = c["kv_heads"], c["head_dim"], c["page"]
    g = c["heads"] // kv
    out = torch.zeros(c["seqs"], c["heads"], d, dtype=torch.float64, device="cuda")
    channel = torch.arange(d, device="cuda")
    word = ((channel % 64) // 8 * (d // 64) + channel // 64) * 4 + channel % 8 // 2   # the byte of each channel
    for i, n in enumerate(st["lens"].tolist()):
        block = st["pool"][st["table"][i, :-(-n // page)].long()]                     # [pages, kv, bytes]
        cut = [page * d // 2, page * d, page * d + page * d // 16, page * d + page * d // 8]
        two = []
        for lo, hi, mlo, mhi in ((0, cut[0], cut[1], cut[2]), (cut[0], cut[1], cut[2], cut[3])):
            byte = block[..., lo:hi].reshape(-1, kv, page, d // 2)[..., word].int()
            code = torch.where(channel % 2 == 0, byte % 16, byte // 16).double() - 8
            pair = block[..., mlo:mhi].contiguous().view(torch.float16).reshape(-1, kv, page, d // 64, 2).double()
            pair = pair.repeat_interleave(64, dim=3)
            x = code * pair[..., 0] + pair[..., 1]
            two.append(x.permute(1, 0, 2, 3).reshape(kv, -1, d)[:, :n])
        q = (st["q"][i].double() * st["sq"][i, :, None].double()).view(kv, g, d)
        s = torch.einsum("hgd,hjd->hgj", q, two[0]) / math.sqrt(d)
        out[i] = torch.einsum("hgj,hjd->hgd", torch.softmax(s, dim=-1), two[1]).reshape(c["heads"], d)
    return out
