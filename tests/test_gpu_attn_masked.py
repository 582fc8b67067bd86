"""Masked attention with shared key heads and the relative position bias, forward
and backward, against the same formulas in 64 bits.

Tolerances.  Outputs are the formula's value rounded once, off by at most u =
eps / 2 of the value (bf16 2^-8, fp32 2^-24), plus what the kernel rounds inside:
bf16 rounds the softmax weights (and dS) to bf16 for the second product, each by
at most u of itself, so an output element is off by at most u times the sum of
the magnitudes of its terms (S below); delta and lse come from values rounded that way as
well, a second such part.  fp32 products sum n terms: n u times S at most,
sqrt(n) u in practice; 16 sqrt(n) u S is asked for.  A score of size x (the sum of its
terms' magnitudes) is off by a few fp32 u of x, its weight by that much of itself: 4 u x.
So |got - want| <= u |want| + c S with c = 2 u (bf16; 3 u where a rounded o enters
through delta) or 16 sqrt(n) u (fp32), plus 4 u x of fp32 in both."""
import math

import pytest
import torch

import dit_hip as dh

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U = {BF16: torch.finfo(BF16).eps / 2, F32: torch.finfo(F32).eps / 2}


def rand(seed, shape, dtype, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def keep_of(B, n, kv_len, kv_mask):
    keep = torch.ones((B, n), dtype=torch.bool, device="cuda")
    if kv_len is not None:
        keep &= torch.arange(n, device="cuda") < kv_len[:, None]
    if kv_mask is not None:
        keep &= kv_mask != 0
    return keep


def bucket_of(off, buckets, distance, two_sided):
    side = buckets // 2 if two_sided else buckets
    near = side // 2
    d = abs(off) if two_sided else max(-off, 0)
    t = d
    if d >= near:
        t = near
        while t < side - 1 and d ** (side - near) >= near ** (side - t - 1) * distance ** (t + 1 - near):
            t += 1
    return t + (side if two_sided and off > 0 else 0)


def bucket_index(Sq, Skv, q_pos, rel):
    """[B or 1, Sq, Skv] buckets."""
    pos = [0] if q_pos is None else q_pos.tolist()
    tab = rel.table
    memo = {}

    def f(off):
        if off not in memo:
            memo[off] = bucket_of(off, tab.shape[0], rel.distance, rel.two_sided)
        return memo[off]

    return torch.tensor([[[f(j - i - p) for j in range(Skv)] for i in range(Sq)] for p in pos], device="cuda")


def oracle(q, k, v, do=None, kv_len=None, kv_mask=None, scale=None, rel=None, q_pos=None):
    """{name: (value, sum of the magnitudes of its terms)} in 64 bits."""
    B, Sq, H, D = q.shape
    Skv, Hkv = k.shape[1:3]
    G = H // Hkv
    scale = D ** -0.5 if scale is None else scale
    keep = keep_of(B, Skv, kv_len, kv_mask)[:, None, None, :]
    q64 = q.double().transpose(1, 2).contiguous()
    z = keep[:, 0, 0, :, None, None]
    k64 = torch.where(z, k.double(), 0.0).repeat_interleave(G, 2).transpose(1, 2).contiguous()
    v64 = torch.where(z, v.double(), 0.0).repeat_interleave(G, 2).transpose(1, 2).contiguous()
    x = (q64 @ k64.transpose(2, 3).contiguous()) * scale
    if rel is not None:
        idx = bucket_index(Sq, Skv, q_pos, rel)
        x = x + rel.table.double()[idx].permute(0, 3, 1, 2)
    x = x.masked_fill(~keep, -math.inf)
    lse = torch.logsumexp(x, -1)
    p = torch.exp(x - torch.where(lse == -math.inf, 0.0, lse)[..., None])
    o = p @ v64
    x_size = (q64.abs() @ k64.abs().transpose(2, 3).contiguous()).max().item() * scale if x.numel() else 0.0
    if rel is not None:
        x_size += rel.table.abs().max().item()
    out = {"x": x_size, "o": (o.transpose(1, 2), (p @ v64.abs()).transpose(1, 2)), "lse": (lse, None)}
    if do is None:
        return out
    g = do.double().transpose(1, 2).contiguous()
    dp = g @ v64.transpose(2, 3).contiguous()
    delta = (p * dp).sum(-1, keepdim=True)
    ds = p * (dp - delta)
    # Magnitudes: dP and delta are themselves sums of rounded terms.
    size = p * (dp.abs() + (p * dp.abs()).sum(-1, keepdim=True) + (g.abs() * (p @ v64.abs())).sum(-1, keepdim=True))

    def heads(t):
        return t.reshape(B, Hkv, G, Skv, D).sum(2).transpose(1, 2)

    T = lambda t: t.transpose(2, 3).contiguous()  # noqa: E731
    out["dq"] = ((ds @ k64 * scale).transpose(1, 2), (size @ k64.abs() * scale).transpose(1, 2))
    out["dk"] = (heads(T(ds) @ q64 * scale), heads(T(size) @ q64.abs() * scale))
    out["dv"] = (heads(T(p) @ g), heads(T(p) @ g.abs()))
    if rel is not None:
        b_idx = idx.expand(B, Sq, Skv).reshape(-1)
        for name, t in (("v", ds), ("s", size)):
            tab = torch.zeros(rel.table.shape, dtype=torch.float64, device="cuda")
            tab.index_add_(0, b_idx, t.permute(0, 2, 3, 1).reshape(-1, H))
            out["dtable" + name] = tab
        out["dtable"] = (out.pop("dtablev"), out.pop("dtables"))
    return out


def hold(name, got, wants, dtype, n, c=2.0):
    value, size = wants[name]
    u = U[dtype]
    assert got.shape == value.shape, name
    part = (c * u if dtype == BF16 else 16 * math.sqrt(n) * u) + 4 * U[F32] * wants["x"]
    bound = u * value.abs() + part * size + 1e-30
    err = (got.double() - value).abs()
    assert torch.isfinite(got).all(), f"{name}: not finite"
    worst = (err / bound).max().item() if err.numel() else 0.0
    assert worst <= 1, f"{name}: {worst:.2f} times the bound"


def check(q, k, v, do=None, rel=None, q_pos=None, **kw):
    want = oracle(q, k, v, do, rel=rel, q_pos=q_pos, **kw)
    n, dt = q.shape[3] + k.shape[1], q.dtype
    if rel is None:
        o, lse = dh.cross_attn(q, k, v, return_lse=True, **kw)
    else:
        o, lse = dh.rel_attn(q, k, v, rel, q_pos=q_pos, return_lse=True, **kw)
    hold("o", o, want, dt, n)
    w = want["lse"][0]
    assert torch.equal(torch.isinf(lse), torch.isinf(w))
    # fp32 scores and sums in both types: sqrt(n) u of the scores' size.
    d = (lse.double() - w)[~torch.isinf(w)].abs()
    assert d.numel() == 0 or d.max().item() <= U[F32] * (16 * math.sqrt(n) + 4 * want["x"])
    if do is None:
        return o
    if rel is None:
        grads = dh.cross_attn_bwd(do, q, k, v, o, lse, **kw)
    else:
        grads = dh.rel_attn_bwd(do, q, k, v, o, lse, rel, q_pos=q_pos, **kw)
    nb = n + q.shape[1] * (q.shape[2] // k.shape[2])
    for name, t in zip(("dq", "dk", "dv"), grads):
        hold(name, t, want, dt, nb, 3.0)
    if rel is not None:  # fp32 in both types: no rounded value enters
        hold("dtable", grads[3], want, F32, q.shape[0] * q.shape[1] * k.shape[1])
    return o, *grads


# ---- lengths, widths, shared heads ---------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D", [
    (1, 1, 1, 1, 1, 64), (2, 3, 3, 1, 33, 128), (1, 4, 2, 5, 64, 8), (2, 6, 2, 31, 65, 72), (1, 2, 1, 33, 129, 128),
    (3, 4, 4, 128, 77, 64), (1, 8, 2, 130, 200, 40), (2, 2, 2, 300, 31, 128), (1, 24, 24, 1400, 96, 64),
    (1, 16, 4, 1, 2600, 128), (5, 2, 1, 2, 1111, 96),
])
def test_attention_and_gradients(dtype, B, H, Hkv, Sq, Skv, D):
    print(f"attention {dtype} {B, H, Hkv, Sq, Skv, D}", flush=True)
    q, k, v = rand(1, (B, Sq, H, D), dtype), rand(2, (B, Skv, Hkv, D), dtype), rand(3, (B, Skv, Hkv, D), dtype)
    check(q, k, v, rand(4, (B, Sq, H, D), dtype))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Sq,Skv", [(1, 700), (40, 100), (700, 150)])
def test_lengths_and_masks(dtype, Sq, Skv):
    B, H, D = 6, 4, 64
    q, k, v = rand(5, (B, Sq, H, D), dtype), rand(6, (B, Skv, H, D), dtype), rand(7, (B, Skv, H, D), dtype)
    do = rand(8, (B, Sq, H, D), dtype)
    kv_len = torch.tensor([0, 1, 64, Skv, Skv + 9, -3], dtype=torch.int32, device="cuda")
    mask = (rand(9, (B, Skv), F32) > 0).to(torch.uint8)
    mask[3] = 0      # nothing kept
    mask[2, :64] = 0  # nothing kept below its length
    mask[1, 0] = 255  # any nonzero byte
    for kw in ({"kv_len": kv_len}, {"kv_mask": mask}, {"kv_len": kv_len, "kv_mask": mask}):
        print(f"masks {dtype} {Sq, Skv} {list(kw)}", flush=True)
        # What is not kept holds NaN and infinities.
        gone = ~keep_of(B, Skv, kw.get("kv_len"), kw.get("kv_mask"))
        k2, v2 = k.clone(), v.clone()
        k2[gone] = math.nan
        v2[gone] = math.inf
        o, dq, dk, dv = check(q, k2, v2, do, **kw)
        empty = gone.all(1)
        assert (o[empty] == 0).all() and (dq[empty] == 0).all() and (dk[gone] == 0).all() and (dv[gone] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_left_padding_and_bool_mask(dtype):
    B, Sq, Skv, H, D = 2, 70, 260, 2, 128
    q, k, v = rand(10, (B, Sq, H, D), dtype), rand(11, (B, Skv, H, D), dtype), rand(12, (B, Skv, H, D), dtype)
    mask = torch.zeros((B, Skv + 3), dtype=torch.bool, device="cuda")[:, :Skv]
    mask[0, 200:] = True
    mask[1, 131] = True
    check(q, k, v, rand(13, (B, Sq, H, D), dtype), kv_mask=mask)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_views_strides_and_repeated_inputs(dtype):
    B, Sq, Skv, H, D = 2, 50, 90, 2, 64
    qkv = rand(14, (Sq, B, 3, H, D), dtype)  # token-major, a slice of a wider projection
    q = qkv[:, :, 1].transpose(0, 1)
    kv = rand(15, (1, Skv, 2, 1, D), dtype)  # one request's states for all, one head for all
    k, v = kv[:, :, 0].expand(B, Skv, H, D), kv[:, :, 1].expand(B, Skv, H, D)
    check(q, k, v, rand(16, (B, H, Sq, D), dtype).transpose(1, 2))
    out = torch.zeros((B, Sq, H, 2 * D), dtype=dtype, device="cuda")
    dh.cross_attn(q, k, v, out=out[..., D:])
    assert torch.equal(out[..., D:], dh.cross_attn(q, k, v)) and (out[..., :D] == 0).all()


def test_scores_far_apart_and_scale_zero():
    B, Sq, Skv, H, D = 1, 200, 300, 2, 64
    q, k, v = rand(17, (B, Sq, H, D), F32, 30.0), rand(18, (B, Skv, H, D), F32), rand(19, (B, Skv, H, D), F32)
    check(q, k, v)
    o = dh.cross_attn(q, k, v, scale=0.0)
    want = v.double().mean(1, keepdim=True).expand(B, Sq, H, D)
    assert (o.double() - want).abs().max().item() <= 300 * U[F32]


# Rounding errors of dS and of the result are independent and of one size: sqrt(2) = 1.41 of one
# rounding's in the mean square; of 1e4 values and more that mean is within 3 %.
@pytest.mark.parametrize("Skv", [9, 24, 40, 64, 65, 130])
def test_gradients_of_few_keys_are_two_roundings_off(Skv):
    B, H, Sq, D = 3, 16, 300, 64
    q, k, v, do = (rand(90 + i, (B, n, H, D), BF16) for i, n in enumerate((Sq, Skv, Skv, Sq)))
    o, lse = dh.cross_attn(q, k, v, return_lse=True)
    want = oracle(q, k, v, do)
    for name, got in zip(("dq", "dk", "dv"), dh.cross_attn_bwd(do, q, k, v, o, lse)):
        w = want[name][0]
        once = (w.to(BF16).double() - w).norm()
        assert (got.double() - w).norm() <= 1.5 * once, f"{name}: {((got.double() - w).norm() / once).item():.2f}"


# ---- the bias ------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,Hkv,Sq,Skv,D,buckets,distance,two_sided", [
    (1, 2, 2, 1, 1, 64, 32, 128, True), (2, 3, 3, 40, 40, 64, 32, 128, True), (2, 2, 1, 200, 333, 64, 32, 128, True),
    (1, 4, 4, 333, 200, 128, 32, 128, False), (1, 2, 2, 100, 100, 72, 4, 2, True), (1, 2, 2, 90, 150, 64, 2, 2, False),
    (1, 1, 1, 70, 1200, 64, 128, 1024, True), (1, 2, 2, 130, 140, 32, 64, 33, False),
])
def test_bias_and_its_gradient(dtype, B, H, Hkv, Sq, Skv, D, buckets, distance, two_sided):
    print(f"bias {dtype} {B, H, Hkv, Sq, Skv, D, buckets, distance, two_sided}", flush=True)
    q, k, v = rand(21, (B, Sq, H, D), dtype, D ** -0.5), rand(22, (B, Skv, Hkv, D), dtype), rand(23, (B, Skv, Hkv, D), dtype)
    rel = dh.RelBias(rand(24, (buckets, H), F32), distance, two_sided)
    check(q, k, v, rand(25, (B, Sq, H, D), dtype), rel=rel, scale=1.0)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("Sq", [1, 37])
def test_bias_with_positions_lengths_and_masks(dtype, Sq):
    B, H, Skv, D = 4, 2, 600, 64
    q, k, v = rand(31, (B, Sq, H, D), dtype), rand(32, (B, Skv, H, D), dtype), rand(33, (B, Skv, H, D), dtype)
    kv_len = torch.tensor([600, 77, 0, 300], dtype=torch.int32, device="cuda")
    q_pos = torch.tensor([599, 76, -5, 2 ** 31 - 1], dtype=torch.int32, device="cuda")
    mask = (rand(34, (B, Skv), F32) > -0.5).to(torch.uint8)
    wide = rand(35, (32, H + 3), F32)
    rel = dh.RelBias(wide[:, :H], 128, False)
    kw = {"kv_len": kv_len, "kv_mask": mask}
    check(q, k, v, rand(36, (B, Sq, H, D), dtype), rel=rel, q_pos=q_pos, **kw)


def test_gradients_against_differences():
    B, Sq, Skv, H, D = 1, 6, 40, 2, 16
    q, k, v, do = (rand(40 + i, s, F32) for i, s in enumerate(((B, Sq, H, D), (B, Skv, 1, D), (B, Skv, 1, D), (B, Sq, H, D))))
    rel = dh.RelBias(rand(44, (8, H), F32), 20, True)
    o, lse = dh.rel_attn(q, k, v, rel, return_lse=True)
    grads = dh.rel_attn_bwd(do, q, k, v, o, lse, rel)
    step = 2.0 ** -7
    for x, g, places in ((q, grads[0], (0, 91)), (k, grads[1], (5, 333)), (v, grads[2], (17, 600)), (rel.table, grads[3], (0, 9))):
        for at in places:
            side = []
            for s in (step, -step):
                old = x.view(-1)[at].item()
                x.view(-1)[at] = old + s
                side.append((oracle(q, k, v, rel=rel)["o"][0] * do.double()).sum().item())
                x.view(-1)[at] = old
            # a central difference is off by step^2 / 6 of the third derivative (order 10 here)
            assert abs((side[0] - side[1]) / (2 * step) - g.reshape(-1)[at].item()) <= 2e-3


# ---- use: streams, graphs, repeats -------------------------------------------------------
def test_same_bits_each_time_on_other_streams_and_without_workspace():
    B, H, Hkv, Skv, D = 2, 8, 2, 4000, 128
    q, k, v = rand(50, (B, 1, H, D), BF16), rand(51, (B, Skv, Hkv, D), BF16), rand(52, (B, Skv, Hkv, D), BF16)
    want = dh.cross_attn(q, k, v)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = dh.cross_attn(q, k, v)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got, want)
    out = torch.empty_like(q)
    a, room, _, _ = dh._attn_args(q, k, v, None, None, None, None, None, out)
    lib = dh.load()
    assert room == lib.dt_attn_fwd_workspace_bytes(dh.ctypes.addressof(a)) > 0
    dh.check(lib.dt_attn_fwd(dh.ctypes.addressof(a), out.data_ptr(), dh._strides3(out), None, None, 0, dh.stream()))
    hold("o", out, oracle(q, k, v), BF16, Skv)


def test_captured_training_step_replays():
    B, S, H, D = 2, 150, 4, 64
    q, k, v, do = (rand(60 + i, (B, S, H, D), BF16) for i in range(4))
    rel = dh.RelBias(rand(64, (32, H), F32), 128, True)
    kv_len = torch.tensor([150, 90], dtype=torch.int32, device="cuda")

    def step():
        o, lse = dh.rel_attn(q, k, v, rel, kv_len=kv_len, return_lse=True)
        return (o, *dh.rel_attn_bwd(do, q, k, v, o, lse, rel, kv_len=kv_len))

    step()
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):  # two graphs of the same call
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs = step()
        graphs.append((g, outs))
    for i in range(4):
        q.copy_(rand(70 + i, (B, S, H, D), BF16))
        kv_len.copy_(torch.tensor([150 - i, 90 + 10 * i], dtype=torch.int32))
        want = step()
        torch.cuda.synchronize()
        for g, outs in graphs:
            g.replay()
        torch.cuda.synchronize()
        for g, outs in graphs:
            for a, b in zip(outs, want):
                assert torch.equal(a, b), f"replay {i} differs"


def test_empty_calls():
    for shape_q, shape_k in (((0, 4, 2, 64), (0, 5, 2, 64)), ((2, 0, 2, 64), (2, 5, 2, 64)), ((2, 3, 2, 64), (2, 0, 2, 64))):
        q, k, v = rand(80, shape_q, BF16), rand(81, shape_k, BF16), rand(82, shape_k, BF16)
        rel = dh.RelBias(rand(83, (8, 2), F32), 16, True)
        o, lse = dh.rel_attn(q, k, v, rel, return_lse=True)
        dq, dk, dv, dt = dh.rel_attn_bwd(q, q, k, v, o, lse, rel)
        for t in (o, dq, dk, dv, dt):
            assert (t == 0).all()
        assert (lse == -math.inf).all()
