"""Calls at the edges of the text operators; formulas and bounds are
test_gpu_attn_masked's and test_gpu_lora's."""
import pytest
import torch

import dit_hip as dh
from test_gpu_attn_masked import check, oracle, rand
from test_gpu_lora import case, hold, q8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


# A softmax does not see what is added to the whole table, and exp of it alone is out of
# range from 88.7 on: weights come from differences, also where the queries end inside a
# tile.  The bound's 4 u of the scores' size holds: a weight's exponent is the sum of the
# bias in log2 (one rounding), lse (the reference's addition and its scaling: two) and its
# scaling back (one), and their difference is exact.
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", [(2, 2, 2, 1, 150, 64), (1, 2, 1, 33, 90, 128), (1, 4, 2, 37, 500, 64), (2, 2, 2, 70, 70, 64),
                                              (1, 2, 2, 70, 200, 128), (1, 2, 2, 128, 130, 64), (1, 24, 24, 700, 700, 64),
                                              (1, 24, 12, 701, 350, 128)])
def test_bias_shifted_by_a_constant(dtype, B, H, Hkv, Sq, Skv, D):
    print(f"shifted bias {dtype} {B, H, Hkv, Sq, Skv, D}", flush=True)
    q, k, v = rand(1, (B, Sq, H, D), dtype, D ** -0.5), rand(2, (B, Skv, Hkv, D), dtype), rand(3, (B, Skv, Hkv, D), dtype)
    do, table = rand(4, (B, Sq, H, D), dtype), rand(5, (32, H), F32)
    for shift in (100.0, -100.0):
        check(q, k, v, do, rel=dh.RelBias(table + shift, 128, True), scale=1.0)


# The few-row products of four and of eight waves (one or several workgroups per CU), ranks in one
# and several parts, in chunks of 8 and not.
@pytest.mark.parametrize("quant", [False, True])
@pytest.mark.parametrize("N,K,R,n", [(4096, 1024, 16, 12), (8192, 256, 64, 20), (16384, 128, 20, 9), (4096, 2048, 100, 16)])
def test_few_rows_have_the_same_bits_whoever_shares_the_step(N, K, R, n, quant):
    M = 16
    x, w, lora = case(11, M, N, K, R, n)
    wq, value = q8(w) if quant else (w, w)
    rows = (torch.arange(M, dtype=torch.int32, device="cuda") * 7 + 3) % (n + 1) - 1
    both = dh.lora_gemm(x, wq, lora, rows)
    hold(both, x, value, lora, rows)
    for order in (torch.arange(M - 1, -1, -1, device="cuda"), (torch.arange(M, device="cuda") * 5 + 2) % M):
        assert torch.equal(dh.lora_gemm(x[order].contiguous(), wq, lora, rows[order].contiguous()), both[order])
    for m in range(M):
        only = torch.where(torch.arange(M, device="cuda") == m, rows, -1).to(torch.int32)
        assert torch.equal(dh.lora_gemm(x, wq, lora, only)[m], both[m]), f"row {m} beside rows without adapters"
        assert torch.equal(dh.lora_gemm(x[m:m + 1], wq, lora, rows[m:m + 1])[0], both[m]), f"row {m} alone"


# As for calls of few keys: two independent roundings, 1.41 of one, within 1.5.  The kept keys lie side
# by side (left padding) or anywhere.
@pytest.mark.parametrize("apart", [False, True])
@pytest.mark.parametrize("kept,Skv,D", [(9, 77, 64), (9, 500, 64), (24, 500, 64), (40, 500, 64), (24, 1500, 64), (9, 300, 128)])
def test_gradients_of_few_kept_keys_are_two_roundings_off(kept, Skv, D, apart):
    B, H, Sq = 3, 16, 300
    q, k, v, do = (rand(90 + i, (B, n, H, D), BF16) for i, n in enumerate((Sq, Skv, Skv, Sq)))
    mask = torch.zeros((B, Skv), dtype=torch.uint8, device="cuda")
    for b in range(B):
        at = rand(94 + b, (Skv,), F32).argsort()[:kept] if apart else slice(Skv - kept, Skv)
        mask[b, at] = 1
    o, lse = dh.cross_attn(q, k, v, kv_mask=mask, return_lse=True)
    want = oracle(q, k, v, do, kv_mask=mask)
    for name, got in zip(("dq", "dk", "dv"), dh.cross_attn_bwd(do, q, k, v, o, lse, kv_mask=mask)):
        w = want[name][0]
        once = (w.to(BF16).double() - w).norm()
        assert (got.double() - w).norm() <= 1.5 * once, f"{name}: {((got.double() - w).norm() / once).item():.2f}"


# A wide weight of few k: four waves with a block of 64 k at most, the last columns past N.
@pytest.mark.parametrize("M", [1, 5, 16])
@pytest.mark.parametrize("N,K", [(16500, 64), (16384, 192), (40000, 256), (16390, 320)])
def test_few_rows_of_short_sums(N, K, M):
    x, w, lora = case(31, M, N, K, 8, 1)
    none = torch.full((M,), -1, dtype=torch.int32, device="cuda")
    bias, add = rand(37, (N,), F32), rand(38, (M, N), F32)
    hold(dh.gemm(x, w, bias=bias, addend=add, out_dtype=F32), x, w, lora, none, bias, add)
    assert torch.equal(dh.gemm(x, w), dh.lora_gemm(x, w, lora, none))


# A table entry of -inf leaves its bucket's keys out; a query that has none left is all zeros.  Two
# kernels' results of one formula: each rounds its weights and its output, by u of v's size each.
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_bias_of_minus_infinity_leaves_keys_out(dtype):
    B, H, Sq, Skv, D = 2, 2, 70, 300, 64
    q, k, v, do = (rand(41 + i, (B, n, H, D), dtype) for i, n in enumerate((Sq, Skv, Skv, Sq)))
    table = rand(45, (32, H), F32)
    table[15] = table[31] = -torch.inf  # distance 113 and more, both sides
    table[:, 1] = -torch.inf            # every key of the second head
    rel = dh.RelBias(table, 128, True)
    o, lse = dh.rel_attn(q, k, v, rel, return_lse=True)
    dq, dk, dv, dt = dh.rel_attn_bwd(do, q, k, v, o, lse, rel)
    for t in (o, dq, dk, dv):
        assert torch.isfinite(t).all() and (t[:, :, 1] == 0).all()
    assert (lse[:, 1] == -torch.inf).all() and (dt[:, 1] == 0).all() and (dt[[15, 31]] == 0).all()
    # The same by a mask, query by query: keys of bucket 15 and 31 dropped for the first head.
    buckets = dh.rel_buckets(Skv + Sq, 32, 128, True).cuda()
    off = torch.arange(Skv, device="cuda")[None, :] - torch.arange(Sq, device="cuda")[:, None]
    left_out = torch.isin(buckets[(off + Skv + Sq - 1).long()], torch.tensor([15, 31], device="cuda", dtype=torch.int32))
    for i in (0, 33, 69):
        part = table[:, :1].clone()
        part[[15, 31]] = 0.0
        mask = (~left_out[i])[None].expand(B, Skv).contiguous()
        want = dh.rel_attn(q[:, i:i + 1, :1], k[:, :, :1], v[:, :, :1], dh.RelBias(part, 128, True),
                           q_pos=torch.full((B,), i, dtype=torch.int32, device="cuda"), kv_mask=mask)
        u = torch.finfo(dtype).eps / 2
        err = (o[:, i, 0].double() - want[:, 0, 0].double()).abs().max().item()
        assert err <= (4 * u if dtype == BF16 else 64 * u) * v.abs().max().item()


def test_gradients_of_scale_zero():
    B, H, Sq, Skv, D = 1, 2, 40, 90, 64
    q, k, v, do = (rand(51 + i, (B, n, H, D), F32) for i, n in enumerate((Sq, Skv, Skv, Sq)))
    check(q, k, v, do, scale=0.0)


# Keys that lie more than 2^32 bytes apart, read and written.
@pytest.mark.parametrize("Sq", [1, 130])
def test_keys_beyond_four_gigabytes(Sq):
    H, Skv, D = 2, 700, 64
    step = (1 << 23) - 136  # elements from token to token, the most there may be: below 2^24 - 256 bytes
    room = torch.zeros(Skv * step, dtype=BF16, device="cuda")
    wide = room.as_strided((1, Skv, H, D), (Skv * step, step, D, 1))
    q, k, v, do = (rand(61 + i, (1, n, H, D), BF16) for i, n in enumerate((Sq, Skv, Skv, Sq)))
    wide.copy_(k)
    assert (Skv - 1) * step * 2 > 1 << 32
    o, lse = dh.cross_attn(q, wide, v, return_lse=True)
    want, want_lse = dh.cross_attn(q, k, v, return_lse=True)
    assert torch.equal(o, want) and torch.equal(lse, want_lse)
    assert torch.equal(dh.cross_attn(q, v, wide), dh.cross_attn(q, v, k))
    for a, b in zip(dh.cross_attn_bwd(do, q, wide, v, o, lse), dh.cross_attn_bwd(do, q, k, v, o, lse)):
        assert torch.equal(a, b)
