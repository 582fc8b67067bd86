"""The text-serving operators where they can go wrong: at the ends of their types' ranges, among thousands of keys, and
behind tables wider than what is held.  Each against its definition in 64 bits."""
import math

import pytest
import torch

import dit_hip as dh
from test_gpu_text_serving import BF16, F8, F32, Pool, e4m3, ints, power, rand, round_bf16, same, turned

pytestmark = pytest.mark.gpu


# -------------------------------------------------------------------- cache --
@pytest.mark.parametrize("half,rot", [(True, 64), (True, 32), (False, 64), (False, 38)])
@pytest.mark.parametrize("mul", [1.0, 1.5, 0.75])
@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("dtype", [F8, BF16])
def test_append_of_keys_next_to_the_end_of_fp32(dtype, io, mul, half, rot):
    """Pairs of which one end leaves fp32's range, and pairs that only 64 bits keep within it: an end beyond the range is not
    finite, the other is held like any."""
    n, D, P = 96, 64, 16
    g = torch.Generator().manual_seed(5)
    size = torch.tensor([3.3e38, 2.9e38, 2.5e38, 2e38, 1e37, 1.0])[torch.randint(0, 6, (n, 1, D), generator=g)]
    k = (size * torch.where(torch.rand((n, 1, D), generator=g) < 0.5, 1.0, -1.0)).to(io).cuda()
    r = dh.Rotary(dh.rotary_freqs(rot), half=half, attn_factor=mul)
    pool = Pool(40, [n], 1, D, P, dtype)
    dh.cache_append(pool.cache, k, torch.zeros_like(k), pool.table, ints(0, n), ints(0), rot=r)
    want = turned(k, torch.arange(n, device="cuda"), r.freq, half, mul)
    beyond = want.to(F32).isinf()
    assert 0 < int(beyond.sum()) < beyond.numel() // 2
    for j in range(0, n, P):
        p, x, out = pool.rows[0][j // P], want[j:j + P, 0], beyond[j:j + P, 0]
        got = pool.cache.k[p, 0]
        if dtype == BF16:
            w = round_bf16(x)
            same(got, torch.where(w.abs() >= 2.0 ** 128, torch.copysign(torch.full_like(w, math.inf), w), w), f"page {p}")
            continue
        e = power(torch.where(out, 0.0, x.abs()).amax())
        assert pool.cache.k_scale[p, 0].item() - 127 == e.item()
        same(got, e4m3(torch.where(out, math.nan, x) * torch.exp2(-e)), f"page {p}")
