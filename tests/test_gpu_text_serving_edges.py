"""The text-serving operators where they can go wrong: at the ends of their types' ranges, among thousands of keys, and
behind tables wider than what is held.  Each against its definition in 64 bits."""
import math

import pytest
import torch

import dit_hip as dh
from test_gpu_text_serving import BF16, F8, F32, F64, Pool, e4m3, ints, power, rand, round_bf16, same, turned

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------- rotary --
@pytest.mark.parametrize("mul", [1.0, 0.9, 1.1, 1.25, 1.3465736])
def test_rotary_cosine_and_sine(mul):
    """(1, 0) turned is (cos, sin) times the factor: off by at most 2^-23 of it.  (The angle rounded to fp32 once, the
    series, and the product by the factor: 2^-23.04 at most over every fp32 angle up to pi / 4.)"""
    T, n = 60000, 64
    x = torch.zeros((T, 1, 2 * n), dtype=F32, device="cuda")
    x[..., :n] = 1.0
    pos = torch.randint(0, 100000, (T,), dtype=torch.int32, generator=torch.Generator().manual_seed(1)).cuda()
    freq = torch.rand(n, generator=torch.Generator().manual_seed(2)).cuda()
    y, _ = dh.rotary(x, None, pos, dh.Rotary(freq, half=True, attn_factor=mul))
    a = pos.to(F64)[:, None] * freq.to(F64)
    f = torch.tensor(mul, dtype=F32).to(F64).item()
    off = torch.stack(((y[:, 0, :n].to(F64) - f * torch.cos(a)).abs().amax(), (y[:, 0, n:].to(F64) - f * torch.sin(a)).abs().amax()))
    # beside it the angles' own rounding in 64 bits, in the reference too
    assert off.max().item() <= 2.0 ** -23 * f + 4 * 2.0 ** -53 * 1e5, f"2^{math.log2(off.max().item() / f):.3f} of the factor"


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
