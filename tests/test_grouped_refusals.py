"""Refusals of the grouped-head operators: host-side checks, no GPU needed."""
import pytest
import torch

from helpers import cabi, ext


def test_c_abi_refuses_before_anything_runs():
    c = cabi()
    lib, P = c.load(), 4096                                        # P: an aligned address that nothing reads
    qk = lambda **o: lib.i8tk_qk_norm_rope(*{**dict(qkv=P, dtype=0, stride=1024, qw=None, kw=None, pos=None, rope=None, rows=0, R=0,  # noqa: E731
                                                    inter=0, eps=1e-6, out=P, T=1, H=4, kv=2, D=128, st=None), **o}.values())
    bad, no, al = c.ERR_INVALID_ARGUMENT, c.ERR_UNSUPPORTED, c.ERR_ALIGNMENT
    assert qk(qkv=None) == bad and qk(dtype=2) == bad and qk(T=0) == bad and qk(stride=1016) == bad and qk(stride=1028) == bad
    assert qk(out=None) == bad and qk(qw=P) == bad and qk(pos=P) == bad
    assert qk(D=96) == no and qk(pos=P, rope=P, rows=4, R=24) == no and qk(pos=P, rope=P, rows=4, R=144) == no
    assert qk(qkv=P + 8) == al and qk(out=P + 2) == al

    ap = lambda **o: lib.i8tk_kv4_append(*{**dict(k=P, v=P, dtype=0, ks=256, vs=256, pool=P, slots=P, T=1, kv=2, D=128, page=16,  # noqa: E731
                                                  pages=4, st=None), **o}.values())
    assert ap(k=None) == bad and ap(pool=None) == bad and ap(ks=248) == bad and ap(vs=260) == bad and ap(pages=0) == bad and ap(dtype=5) == bad
    assert ap(page=8) == no and ap(D=256) == no and ap(v=P + 4) == al
    assert lib.i8tk_kv4_block_bytes(16, 64) == 1152 and lib.i8tk_kv4_block_bytes(48, 64) == 0 and lib.i8tk_kv4_block_bytes(16, 256) == 0
    assert lib.i8tk_kv4_dequantize(P, P, None, P, 1, 2, 128, 16, 4, None) == bad

    de = lambda **o: lib.i8tk_decode_attention_kv4(*{**dict(q=P, qs=512, sq=P, ss=4, pool=P, tab=P, lens=P, out=P, B=1, H=4, kv=2, L=64,  # noqa: E731
                                                            page=16, mp=4, D=128, pages=4, ws=P, n=1 << 30, st=None), **o}.values())
    assert de(q=None) == bad and de(L=0) == bad and de(L=65) == bad and de(qs=496) == bad and de(ss=3) == bad and de(pages=0) == bad
    assert de(D=256) == no and de(page=24) == no and de(H=5) == no and de(H=34) == no and de(pool=P + 8) == al
    assert de(ws=None) == c.ERR_WORKSPACE and de(n=64) == c.ERR_WORKSPACE and de(ws=P + 16) == al
    assert lib.i8tk_decode_kv4_workspace_bytes(1, 34, 2, 64, 128) == 0 and lib.i8tk_decode_kv4_workspace_bytes(1, 32, 2, 64, 128) > 0


def test_varlen_c_abi_refuses_before_anything_runs():
    c = cabi()
    lib, P = c.load(), 4096
    bad, no, al = c.ERR_INVALID_ARGUMENT, c.ERR_UNSUPPORTED, c.ERR_ALIGNMENT
    va = lambda **o: lib.i8tk_attention_varlen(*{**dict(q=P, qs=512, k=P, ks=256, v=P, vs=256, sq=P, sqs=4, sk=P, sks=2, sv=P, svs=2,  # noqa: E731
                                                        cu=P, out=P, T=10, B=2, L=10, H=4, kv=2, D=128, causal=1, ws=P, n=1 << 40,
                                                        st=None), **o}.values())
    assert va(q=None) == bad and va(cu=None) == bad and va(T=0) == bad and va(B=0) == bad and va(L=0) == bad
    assert va(qs=496) == bad and va(ks=264) == bad and va(vs=128) == bad and va(sqs=3) == bad and va(sks=1) == bad
    assert va(D=96) == no and va(H=5) == no and va(H=130) == no and va(T=1 << 31) == no
    assert va(q=P + 8) == al and va(out=P + 2) == al and va(ws=P + 16) == al
    assert va(ws=None) == c.ERR_WORKSPACE and va(n=1000) == c.ERR_WORKSPACE
    size = lib.i8tk_attention_varlen_workspace_bytes
    assert size(10, 2, 5, 2, 128) == 0 and size(10, 2, 4, 2, 96) == 0 and size(1 << 31, 2, 4, 2, 128) == 0
    # room for every slot of 64 positions that sequences of any lengths can take, twice head_dim bytes each
    assert size(1000, 7, 4, 2, 128) >= 2 * (1000 // 64 + 7) * 64 * 2 * 128


def test_ops_refuse_what_they_cannot_take():
    e = ext()
    h = torch.zeros(2, 8 * 64, dtype=torch.float16)
    for call in (lambda: e.qk_norm_rope(h, 4, 2), lambda: e.qk_norm_rope_quantize(h, 4, 2),
                 lambda: e.kv_append_quantize_int4(h.view(2, 8, 64), h.view(2, 8, 64), torch.zeros(1, 8, 1152, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64), 16),
                 lambda: e.kv_dequantize_int4(torch.zeros(1, 8, 1152, dtype=torch.uint8), torch.zeros(2, dtype=torch.int64), 16, 64),
                 lambda: e.int8_attention_varlen(*[torch.zeros(2, 4, 64, dtype=torch.int8)] * 3, *[torch.zeros(2, 4)] * 3,
                                                 torch.tensor([0, 2], dtype=torch.int32), 2),
                 lambda: e.int4_decode_attention_paged(torch.zeros(1, 4, 64, dtype=torch.int8), torch.zeros(1, 4), torch.zeros(1, 2, 1152, dtype=torch.uint8),
                                                       torch.zeros(1, 1, dtype=torch.int32), torch.zeros(1, dtype=torch.int32), 16, 16)):
        with pytest.raises(RuntimeError, match="CUDA"):
            call()
    with pytest.raises(RuntimeError, match="page_size"):
        e.int4_kv_block_bytes(24, 64)
    assert e.int4_kv_block_bytes(64, 128) == 64 * 144
