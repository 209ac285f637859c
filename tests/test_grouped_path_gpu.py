"""The grouped-head operators as a model runs them, one after another: packed prompts through q/k norm + rotation +
quantiser and attention, their keys and values into the 4-bit cache, then decode steps over it -- eagerly, on another
stream, and from captured graphs."""
import numpy as np
import pytest
import torch

from helpers import cabi, ext
from oracle import grouped as og

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


class Layer:
    """What a program keeps: weights, rotation table, cache pool and page table."""

    def __init__(self, H, kv, D, page, lens, steps, dtype, seed):
        g = _gen(seed)
        self.H, self.kv, self.D, self.page, self.B = H, kv, D, page, len(lens)
        self.e = ext()
        self.qw, self.kw = (1 + 0.2 * torch.randn(D, device="cuda", generator=g) for _ in range(2))
        self.table = torch.from_numpy(og.rope_table(max(lens) + steps + 1, D)).cuda()
        need = [-(-(n + steps) // page) for n in lens]
        order = torch.randperm(sum(need) + 2, device="cuda", generator=g).int()
        self.pages = torch.zeros(self.B, max(need), dtype=torch.int32, device="cuda")
        at = 0
        for b, n in enumerate(need):
            self.pages[b, :n] = order[at:at + n]
            at += n
        self.pool = torch.zeros(sum(need) + 2, kv, self.e.int4_kv_block_bytes(page, D), dtype=torch.uint8, device="cuda")
        self.lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
        self.bound = max(lens) + steps
        self.width = (H + 2 * kv) * D
        self.dtype = dtype

    def slots(self, req, pos):
        return self.pages[req, pos // self.page].long() * self.page + pos % self.page

    def values(self, qkv):
        return qkv[:, (self.H + self.kv) * self.D:].unflatten(1, (self.kv, self.D))

    def prompt(self, qkv, cu, pos, req, longest):
        k_rot = torch.empty(len(qkv), self.kv, self.D, device="cuda", dtype=self.dtype)
        codes, scales = self.e.qk_norm_rope_quantize(qkv, self.H, self.kv, pos, self.table, self.qw, self.kw, 1e-6, False, k_rot)
        H, kv = self.H, self.kv
        out = self.e.int8_attention_varlen(codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv],
                                           scales[:, H + kv:], cu, longest)
        self.e.kv_append_quantize_int4(k_rot, self.values(qkv), self.pool, self.slots(req, pos.long()), self.page)
        return out

    def step(self, qkv):
        """One new token for every request, at the end of what it has."""
        k_rot = torch.empty(self.B, self.kv, self.D, device="cuda", dtype=self.dtype)
        codes, scales = self.e.qk_norm_rope_quantize(qkv, self.H, self.kv, self.lens, self.table, self.qw, self.kw, 1e-6, False, k_rot)
        self.e.kv_append_quantize_int4(k_rot, self.values(qkv), self.pool, self.slots(torch.arange(self.B, device="cuda"), self.lens.long()), self.page)
        self.lens += 1
        return self.e.int4_decode_attention_paged(codes[:, :self.H], scales[:, :self.H], self.pool, self.pages, self.lens, self.bound, self.page)


def _cached(layer, b, n):
    """(codes, scale, centre) of the keys and of the values of request b's n cached rows, from the pool's bytes."""
    pool, pages = layer.pool.cpu().numpy(), layer.pages.cpu().numpy()
    both = ([], [])
    for h in range(layer.kv):
        blocks = [og.int4_unblock(pool[p, h], layer.page, layer.D) for p in pages[b, :-(-n // layer.page)]]
        for i in (0, 1):
            both[i].append([np.concatenate([blk[i][x] for blk in blocks])[:n] for x in range(3)])
    return [[np.stack([row[x] for row in both[i]]) for x in range(3)] for i in (0, 1)]


def _check_cache(layer, history):
    """Every cached value is within half a step of its group of the exact one, and what rounding adds: of the rotated
    key to its type (at most 2^-9 of the value, bf16), of the pair to fp16 (2^-11 of centre and of eight steps, which
    are at most the group's largest value each), and clamping to the end code that these roundings may cause (the same
    again): together below 2^-7 of the group's largest value."""
    for b, rows in enumerate(history):
        x = np.stack(rows).reshape(-1, layer.H + 2 * layer.kv, layer.D)
        y = og.qk_norm_rope(x, layer.H, layer.kv, np.arange(len(x)), layer.table.cpu().numpy(), layer.qw.cpu().numpy(), layer.kw.cpu().numpy())
        for got, want in zip(_cached(layer, b, len(x)), (y[:, layer.H:layer.H + layer.kv], y[:, layer.H + layer.kv:])):
            want = want.transpose(1, 0, 2)
            step = np.repeat(got[1].astype(np.float64), 64, axis=-1)
            top = np.repeat(np.abs(want).reshape(*want.shape[:2], -1, 64).max(-1), 64, axis=-1)
            assert (np.abs(og.int4_values(*got) - want) <= 0.5 * step + 2.0 ** -7 * top).all()


@pytest.mark.parametrize("H,kv,D,page,dtype", [(8, 2, 128, 32, torch.bfloat16), (6, 6, 64, 16, torch.float16)])
def test_prompt_then_decode(H, kv, D, page, dtype):
    """Each attention against float64 attention over the codes that it was given, within the bounds of the oracle; the
    codes' way there: the cache against the exact rotated keys and the values."""
    lens, steps = [70, 33, 129], 3
    layer = Layer(H, kv, D, page, lens, steps, dtype, seed=D)
    g = _gen(7)
    draw = lambda n: torch.randn(n, layer.width, device="cuda", generator=g).to(dtype)  # noqa: E731
    qkv = draw(sum(lens))
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    pos = torch.cat([torch.arange(n, device="cuda") for n in lens]).int()
    req = torch.cat([torch.full((n,), b, device="cuda") for b, n in enumerate(lens)])
    out = layer.prompt(qkv, cu, pos, req, max(lens))
    codes, scales = (t.cpu().numpy() for t in layer.e.qk_norm_rope_quantize(qkv, H, kv, pos, layer.table, layer.qw, layer.kw))
    split = lambda t: (t[:, :H], t[:, H:H + kv], t[:, H + kv:])  # noqa: E731
    want, bound = og.varlen_attention(*split(codes), *split(scales), cu.cpu().tolist(), True)
    assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()
    host = qkv.float().cpu().numpy().astype(np.float64)
    history = [list(host[a:b]) for a, b in zip(cu.tolist()[:-1], cu.tolist()[1:])]
    _check_cache(layer, history)
    side = torch.cuda.Stream()
    for s in range(steps):
        new = draw(layer.B)
        qc, qs = layer.e.qk_norm_rope_quantize(new, H, kv, layer.lens, layer.table, layer.qw, layer.kw)
        if s == 1:                                                         # a step on a stream of its own
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                got = layer.step(new)
            torch.cuda.current_stream().wait_stream(side)
        else:
            got = layer.step(new)
        for b, x in enumerate(new.float().cpu().numpy().astype(np.float64)):
            history[b].append(x)
            want, bound = og.int4_decode(qc[b, :H].cpu().numpy(), qs[b, :H].cpu().numpy(), *_cached(layer, b, lens[b] + s + 1))
            assert (np.abs(got[b].float().cpu().numpy() - want) <= bound).all()
    _check_cache(layer, history)
    layer.e.check_status()


def test_captured_steps_replay_with_new_inputs_and_share_nothing():
    """Two graphs of a decode step over two caches, captured one after the other, replayed interleaved: each gives what
    the eager step gives on a copy of its cache."""
    made = []
    for seed in (1, 2):
        layer = Layer(16, 4, 128, 64, [100, 7, 300], 8, torch.float16, seed)
        layer.pool.copy_(torch.randint(0, 100, layer.pool.shape, device="cuda", generator=_gen(seed)).to(torch.uint8))
        twin = Layer(16, 4, 128, 64, [100, 7, 300], 8, torch.float16, seed)
        twin.pool.copy_(layer.pool)
        x = torch.randn(3, layer.width, device="cuda", generator=_gen(seed + 10)).half()
        keep = layer.pool.clone(), layer.lens.clone()
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer.step(x)                                                  # warm-up outside the capture
        torch.cuda.current_stream().wait_stream(side)
        layer.pool.copy_(keep[0])
        layer.lens.copy_(keep[1])
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = layer.step(x)
        made.append((layer, twin, x, graph, out))
    for k in range(3):
        for i, (layer, twin, x, graph, out) in enumerate(made):
            x.copy_(torch.randn(x.shape, device="cuda", generator=_gen(100 * k + i)).half())
            graph.replay()
        for layer, twin, x, graph, out in made:
            want = twin.step(x)
            assert torch.equal(out, want) and torch.equal(layer.pool, twin.pool) and torch.equal(layer.lens, twin.lens)


def test_captured_prompt():
    e = ext()
    H, kv, D, lens = 8, 2, 128, [200, 5, 64]
    g = _gen(3)
    x = torch.randn(sum(lens), H + 2 * kv, D, device="cuda", generator=g)
    codes, scales = e.quantize_per_token(x)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    call = lambda: e.int8_attention_varlen(codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv],  # noqa: E731
                                           scales[:, H + kv:], cu, sum(lens))
    call()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = call()
    for shape in (lens, [1, 268, 0]):                                      # other lengths under the same graph
        cu.copy_(torch.tensor(np.concatenate([[0], np.cumsum(shape)]), dtype=torch.int32))
        graph.replay()
        assert torch.equal(out, call())


def test_two_streams_at_once():
    """Long calls of attention and decode on two streams over the same inputs: each has a workspace of its own."""
    e = ext()
    H, kv, D, n = 16, 4, 64, 3000
    codes, scales = e.quantize_per_token(torch.randn(n, H + 2 * kv, D, device="cuda", generator=_gen(5)))
    cu = torch.tensor([0, 1000, n], dtype=torch.int32, device="cuda")
    pages = -(-n // 16)
    pool = torch.zeros(pages, kv, e.int4_kv_block_bytes(16, D), dtype=torch.uint8, device="cuda")
    kvs = e.dequantize_per_token(codes, scales)
    e.kv_append_quantize_int4(kvs[:, H:H + kv], kvs[:, H + kv:], pool, torch.arange(n, device="cuda"), 16)
    table, ln = torch.arange(pages, device="cuda").int()[None].repeat(2, 1), torch.tensor([n, 77], dtype=torch.int32, device="cuda")

    def both():
        a = e.int8_attention_varlen(codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv], scales[:, H + kv:], cu, n)
        return a, e.int4_decode_attention_paged(codes[:2, :H], scales[:2, :H], pool, table, ln, n, 16)

    want = both()
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = []
    for _ in range(4):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(both())
    torch.cuda.synchronize()
    for a, b in got:
        assert torch.equal(a, want[0]) and torch.equal(b, want[1])
    e.check_status()


def test_offsets_past_32_bits():
    """A pool and a projection of more than 4 GiB, touched at both ends."""
    e = ext()
    kv, D, page = 8, 128, 128
    block = e.int4_kv_block_bytes(page, D)
    pages = (1 << 32) // (kv * block) + 200
    pool = torch.empty(pages, kv, block, dtype=torch.uint8, device="cuda")
    ids = [0, pages - 1, pages // 2, pages - 2]
    n = 500
    g = _gen(2)
    k, v = (torch.randn(n, kv, D, device="cuda", generator=g).half() for _ in range(2))
    pos = torch.arange(n, device="cuda")
    slots = torch.tensor(ids, device="cuda")[pos // page] * page + pos % page
    e.kv_append_quantize_int4(k, v, pool, slots, page)
    small = torch.zeros(4, kv, block, dtype=torch.uint8, device="cuda")
    e.kv_append_quantize_int4(k, v, small, pos, page)
    a, b = e.kv_dequantize_int4(pool, slots, page, D), e.kv_dequantize_int4(small, pos, page, D)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    q, sq = e.quantize_per_token(torch.randn(1, 32, D, device="cuda", generator=g))
    ln = torch.tensor([n], dtype=torch.int32, device="cuda")
    far = e.int4_decode_attention_paged(q, sq, pool, torch.tensor([ids], dtype=torch.int32, device="cuda"), ln, n, page)
    near = e.int4_decode_attention_paged(q, sq, small, torch.arange(4, device="cuda").int()[None], ln, n, page)
    assert torch.equal(far, near)
    del pool
    T, H = 360000, 32                                                       # 2.2e9 values
    x = torch.empty(T, (H + 2 * kv) * D, device="cuda", dtype=torch.bfloat16)
    rows = torch.tensor([0, 1, T // 2, T - 2, T - 1], device="cuda")
    x[rows] = torch.randn(5, x.size(1), device="cuda", generator=g).bfloat16()
    codes, scales = e.qk_norm_rope_quantize(x, H, kv)
    c5, s5 = e.qk_norm_rope_quantize(x[rows], H, kv)
    assert torch.equal(codes[rows], c5) and torch.equal(scales[rows], s5)
    assert torch.equal(e.qk_norm_rope(x, H, kv)[rows], e.qk_norm_rope(x[rows], H, kv))


def test_many_short_sequences():
    e = ext()
    rng = np.random.default_rng(3)
    lens = [int(v) for v in rng.integers(0, 6, 4000)]
    H, kv, D = 4, 2, 64
    x = torch.randn(sum(lens), H + 2 * kv, D, device="cuda", generator=_gen(8))
    codes, scales = e.quantize_per_token(x)
    cu = torch.tensor(np.concatenate([[0], np.cumsum(lens)]), dtype=torch.int32, device="cuda")
    args = [codes[:, :H], codes[:, H:H + kv], codes[:, H + kv:], scales[:, :H], scales[:, H:H + kv], scales[:, H + kv:]]
    out = e.int8_attention_varlen(*args, cu, 5)
    want, bound = og.varlen_attention(*[a.cpu().numpy() for a in args], cu.cpu().tolist(), True)
    assert (np.abs(out.float().cpu().numpy() - want) <= bound).all()


def test_status_of_varlen_through_the_c_abi():
    """Nothing in the workspace is relied on, and the status word of a good call is clean."""
    c, lib = cabi(), cabi().load()
    e = ext()
    codes, scales = e.quantize_per_token(torch.randn(90, 6, 64, device="cuda", generator=_gen(4)))
    cu = torch.tensor([0, 40, 90], dtype=torch.int32, device="cuda")
    want = e.int8_attention_varlen(codes[:, :4], codes[:, 4:5], codes[:, 5:], scales[:, :4], scales[:, 4:5], scales[:, 5:], cu, 50)
    n = lib.i8tk_attention_varlen_workspace_bytes(90, 2, 4, 1, 64)
    ws = torch.full((n,), 255, dtype=torch.uint8, device="cuda")
    out = torch.empty(90, 4, 64, dtype=torch.float16, device="cuda")
    st = torch.cuda.current_stream().cuda_stream
    p, s = codes.data_ptr(), scales.data_ptr()
    for _ in range(2):
        c.check(lib.i8tk_attention_varlen(p, 384, p + 256, 384, p + 320, 384, s, 6, s + 16, 6, s + 20, 6, cu.data_ptr(), out.data_ptr(), 90, 2, 50,
                                          4, 1, 64, 1, ws.data_ptr(), n, st))
        assert lib.i8tk_check_status_word(ws.data_ptr(), st) == c.OK
        assert torch.equal(out, want)
