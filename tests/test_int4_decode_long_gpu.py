"""4-bit decode over long contexts: what the sums of unsigned codes leave behind when the middle code is taken out."""
import pytest
import torch

from helpers import ext

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("H,kv,D,page", [(4, 4, 64, 16), (4, 2, 128, 64), (8, 2, 64, 32), (8, 2, 128, 16), (14, 2, 64, 128), (7, 1, 128, 32), (12, 1, 128, 16), (32, 2, 64, 64)])
def test_values_of_the_middle_code_give_exactly_zero(H, kv, D, page):
    """scale * (8 - 8) + 0 at every position, under any probabilities: sum P * 8 less the same sum."""
    e, lens = ext(), [20011, 3, 700]
    g = torch.Generator(device="cuda").manual_seed(H + D)
    need = [-(-n // page) for n in lens]
    pool = torch.randint(0, 256, (sum(need), kv, e.int4_kv_block_bytes(page, D)), dtype=torch.uint8, device="cuda", generator=g)
    table, at = torch.zeros(len(lens), max(need), dtype=torch.int32, device="cuda"), 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, device="cuda").int()
        at += n
    G = D // 64

    def pairs(scale, centre):
        return torch.stack([scale, centre], dim=-1).half().view(torch.uint8).reshape(sum(need), kv, -1)

    shape = (sum(need), kv, page, G)
    pool[..., page * D // 2:page * D] = 0x88
    pool[..., page * D:page * D + page * G * 4] = pairs(0.1 + 0.2 * torch.rand(shape, device="cuda", generator=g), torch.randn(shape, device="cuda", generator=g) * 0.2)
    pool[..., page * D + page * G * 4:] = pairs(torch.exp(torch.randn(shape, device="cuda", generator=g)), torch.zeros(shape, device="cuda"))
    q, sq = e.quantize_per_token(torch.randn(len(lens), H, D, device="cuda", generator=g))
    out = e.int4_decode_attention_paged(q, sq, pool, table, torch.tensor(lens, dtype=torch.int32, device="cuda"), max(lens), page)
    assert not out.any(), out.abs().max()
    e.check_status()
