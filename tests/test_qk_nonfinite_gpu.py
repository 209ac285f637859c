"""q/k norm + rotation over heads that hold a NaN or an infinity: the quantised form shows them as the other forms do."""
import pytest
import torch

from helpers import ext
from oracle import grouped as og

pytestmark = pytest.mark.gpu
BAD = (float("nan"), float("inf"), -float("inf"))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("D,norm,rotary,interleaved", [(64, True, 0, False), (128, True, 128, False), (256, True, 64, True), (128, False, 64, False),
                                                       (64, False, 64, True), (128, True, 64, False)])
def test_a_head_with_a_nan_or_an_infinity_gets_a_nan_scale(D, norm, rotary, interleaved, dtype):
    e, T, H, kv = ext(), 9, 8, 2
    g = torch.Generator(device="cuda").manual_seed(D)
    x = torch.randn(T, H + 2 * kv, D, device="cuda", generator=g).to(dtype)
    pos = torch.randint(0, 50, (T,), device="cuda", generator=g, dtype=torch.int32) if rotary else None
    table = torch.from_numpy(og.rope_table(50, rotary)).cuda() if rotary else None
    w = 1 + 0.2 * torch.randn(D, device="cuda", generator=g) if norm else None
    call = lambda t, k: e.qk_norm_rope_quantize(t.view(T, -1), H, kv, pos, table, w, w, 1e-6, interleaved, k)  # noqa: E731
    k0, k1 = (torch.empty(T, kv, D, device="cuda", dtype=dtype) for _ in range(2))
    good, scales0 = call(x, k0)
    y = x.clone()
    at = [(0, 0, 0), (1, 7, D - 1), (2, 8, 5), (3, 9, rotary // 2 + 1), (4, 3, D // 2), (4, 4, 0), (8, 9, D - 3)]
    for n, (t, h, d) in enumerate(at):
        y[t, h, d] = BAD[n % 3]
    codes, scales = call(y, k1)
    hit = torch.zeros(T, H + 2 * kv, dtype=torch.bool)
    for t, h, _ in at:
        hit[t, h] = True
    assert scales[hit].isnan().all()
    assert torch.equal(scales[~hit], scales0[~hit]) and torch.equal(codes[~hit], good[~hit])
    assert torch.equal(k1[~hit[:, H:H + kv]], k0[~hit[:, H:H + kv]])
    # the unquantised form has something that is not finite in the same heads and nowhere else
    assert torch.equal((~torch.isfinite(e.qk_norm_rope(y.view(T, -1), H, kv, pos, table, w, w, 1e-6, interleaved).float())).any(-1).cpu(), hit[:, :H + kv])
    assert torch.equal((~torch.isfinite(k1.float())).any(-1).cpu(), hit[:, H:H + kv])


def test_heads_that_are_only_quantised_follow_the_quantiser():
    e, T, H, kv, D = ext(), 5, 2, 1, 128
    x = torch.randn(T, H + 2 * kv, D, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1)).half()
    for n, v in enumerate(BAD):
        x[n, 3, 7 * n] = v                                                     # a value head
        x[n, 0, 9] = v                                                         # a query head, neither normed nor rotated
    codes, scales = e.qk_norm_rope_quantize(x.view(T, -1), H, kv)
    want, ws = e.quantize_per_token(x)
    keep = torch.isfinite(x)
    assert torch.equal(scales, ws) and torch.equal(codes[keep], want[keep])
