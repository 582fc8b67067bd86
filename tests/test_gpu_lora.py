"""Low-rank adapters beside a shared Linear (dt_lora_gemm) against the formula in 64
bits, each row with its own adapter.

Tolerance.  Operands are exact; sums of n fp32 terms are off by sqrt(n) u of the sum
of their magnitudes S (16 of it asked for, u = 2^-24), the rank-space values by 2^-17 of
themselves (two bf16 parts), the result by its one rounding: |got - want| <= eps / 2
|want| + (16 sqrt(K + R) u + 2^-17) S."""
import math

import pytest
import torch

import dit_hip as dh

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


def rand(seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def q8(w):
    n, k = w.shape
    blocks = dh.quantize_q8_0(w.float().contiguous())
    s = dh.q8_0_split(blocks, n, k)
    value = ((s.codes.float().view(n, -1, 32) - 128) * s.scales.t()[..., None]).to(BF16).view(n, k)
    return s, value


def hold(got, x, w, lora, rows, bias=None, addend=None):
    x64, w64 = x.double(), w.double()
    n, R, K = lora.a.shape
    want, size = x64 @ w64.t(), x64.abs() @ w64.abs().t()
    for a in range(n):
        at = (rows == a).nonzero()[:, 0]
        if not len(at):
            continue
        s = 1.0 if lora.scale is None else lora.scale[a].double()
        A, B = lora.a[a].double(), lora.b[a].double()
        want[at] += s * ((x64[at] @ A.t()) @ B.t())
        size[at] += abs(s) * ((x64[at].abs() @ A.abs().t()) @ B.abs().t())
    for t in (bias, addend):
        if t is not None:
            want += t.double()
            size += t.double().abs()
    u = torch.finfo(got.dtype).eps / 2
    bound = u * want.abs() + (16 * math.sqrt(K + R) * 2.0 ** -24 + 2.0 ** -17) * size + 1e-30
    assert torch.isfinite(got).all()
    worst = ((got.double() - want).abs() / bound).max().item()
    assert worst <= 1, f"{worst:.2f} times the bound"


def case(seed, M, N, K, R, n, scale=True):
    x, w = rand(seed, (M, K)), rand(seed + 1, (N, K), std=K ** -0.5)
    lora = dh.Lora(rand(seed + 2, (n, R, K), std=K ** -0.5), rand(seed + 3, (n, N, R), std=max(R, 1) ** -0.5),
                   rand(seed + 4, (n,), F32) if scale else None)
    return x, w, lora


def assign(seed, M, n, how):
    g = torch.Generator().manual_seed(seed)
    if how == "one":
        rows = torch.full((M,), n - 1)
    elif how == "none":
        rows = torch.full((M,), -1)
    elif how == "mixed":  # every row another, -1 and out of range among them
        rows = torch.randint(-1, n + 1, (M,), generator=g)
    else:  # requests of ragged lengths
        cuts = torch.sort(torch.randint(0, M + 1, (5,), generator=g))[0].tolist()
        rows = torch.empty(M, dtype=torch.int64)
        for i, (a, b) in enumerate(zip([0] + cuts, cuts + [M])):
            rows[a:b] = (i * 3) % (n + 1) - 1
    return rows.to(torch.int32).cuda()


# Each product configuration: a weight stream, 128 and 256 tiles, K ranges, any shape.
SHAPES = [(1, 128, 64, 16, 1), (1, 4096, 1024, 8, 3), (5, 2048, 576, 64, 40), (16, 1100, 1024, 20, 16), (17, 260, 512, 4, 2),
          (33, 1024, 1536, 33, 7), (100, 3, 40, 5, 3), (130, 130, 100, 1, 2), (200, 1024, 2048, 16, 4),
          (700, 2304, 512, 96, 5), (1030, 4096, 128, 512, 2), (2100, 2500, 192, 12, 6)]


# A stream of the weight: waves with no block of 64 k, fewer and more than they hold, uneven ends;
# four and eight waves; ranks in one and several parts, more adapters than waves.
@pytest.mark.parametrize("M,N,K,R,n", [(3, 200, 5184, 40, 2), (16, 130, 64, 16, 20), (2, 4096, 8192, 100, 1), (16, 8200, 4160, 64, 12),
                                       (9, 5000, 1536, 33, 9), (7, 16500, 1216, 8, 3), (16, 16384, 2624, 200, 16)])
def test_few_rows(M, N, K, R, n):
    x, w, lora = case(121, M, N, K, R, n)
    rows = (torch.arange(M, dtype=torch.int32, device="cuda") * 5 + 1) % (n + 1) - int(M > 4)
    hold(dh.lora_gemm(x, w, lora, rows), x, w, lora, rows)
    none = torch.full_like(rows, -7)
    assert torch.equal(dh.lora_gemm(x, w, lora, none), dh.gemm(x, w))
    hold(dh.gemm(x, w), x, w, lora, none)


@pytest.mark.parametrize("how", ["one", "mixed", "requests"])
@pytest.mark.parametrize("M,N,K,R,n", SHAPES)
def test_adapters_beside_bf16_weights(M, N, K, R, n, how):
    print(f"lora bf16 {M, N, K, R, n} {how}", flush=True)
    x, w, lora = case(1, M, N, K, R, n)
    rows = assign(9, M, n, how)
    bias = rand(10, (N,), F32)
    hold(dh.lora_gemm(x, w, lora, rows, bias=bias), x, w, lora, rows, bias)


@pytest.mark.parametrize("M,N,K,R,n", [s for s in SHAPES if s[2] % 32 == 0])
def test_adapters_beside_q8_0_weights(M, N, K, R, n):
    print(f"lora q8_0 {M, N, K, R, n}", flush=True)
    x, w, lora = case(21, M, N, K, R, n)
    wq, value = q8(w)
    for how in ("mixed", "requests"):
        rows = assign(29, M, n, how)
        hold(dh.lora_gemm(x, wq, lora, rows), x, value, lora, rows)


@pytest.mark.parametrize("M,N,K,R,n", [(3, 2048, 1024, 16, 4), (300, 512, 2560, 24, 4), (1500, 3000, 256, 16, 3)])
def test_fp32_output_addend_and_no_scale(M, N, K, R, n):
    x, w, lora = case(41, M, N, K, R, n, scale=False)
    rows = assign(49, M, n, "requests")
    add = rand(50, (M, N), F32)
    hold(dh.lora_gemm(x, w, lora, rows, addend=add, out_dtype=F32), x, w, lora, rows, addend=add)


def test_views_and_odd_strides():
    M, N, K, R, n = 70, 96, 136, 12, 3
    wide = rand(61, (M, K + 5))
    x = wide[:, 3:3 + K]
    w = rand(62, (N, K + 1), std=K ** -0.5)[:, :K]
    pool = rand(63, (n, R + 3, K + 2), std=K ** -0.5)[:, 1:R + 1, 1:K + 1]
    up = rand(64, (n, N, R + 7))[:, :, 3:R + 3]
    lora = dh.Lora(pool, up)
    rows = assign(65, M, n, "mixed")
    out = torch.zeros((M, N + 8), dtype=BF16, device="cuda")
    dh.lora_gemm(x, w, lora, rows, out=out[:, 4:N + 4])
    hold(out[:, 4:N + 4], x, w, lora, rows)
    assert (out[:, :4] == 0).all() and (out[:, N + 4:] == 0).all()
    # one adapter for all (stride 0)
    lora = dh.Lora(pool[:1].expand(n, R, K), up[:1].expand(n, N, R))
    hold(dh.lora_gemm(x, w, lora, rows), x, w, lora, rows)


@pytest.mark.parametrize("M", [9, 300])
def test_no_adapter_reaches_anothers_rows(M):
    """Rows without an adapter are the plain product's bit for bit, whatever the pool holds."""
    N, K, R, n = 2048, 1024, 16, 4
    x, w, lora = case(71, M, N, K, R, n)
    rows = assign(72, M, n, "mixed")
    clean = dh.lora_gemm(x, w, lora, rows)
    lora.a[1], lora.b[2] = math.nan, math.inf
    got = dh.lora_gemm(x, w, lora, rows)
    sick = (rows == 1) | (rows == 2)
    assert torch.equal(got[~sick], clean[~sick])
    assert not torch.isfinite(got[rows == 1]).any() and sick.any()
    none = assign(72, M, n, "none")
    assert torch.equal(dh.lora_gemm(x, w, lora, none), dh.gemm(x, w))
    assert torch.equal(dh.lora_gemm(x, w, dh.Lora(lora.a[:0], lora.b[:0]), none), dh.gemm(x, w))


def test_same_bits_alone_and_in_a_batch():
    """A request's rows do not depend on whose rows share its tiles."""
    N, K, R, n = 512, 256, 16, 4
    x, w, lora = case(81, 256, N, K, R, n)
    rows = torch.arange(256, dtype=torch.int32, device="cuda") // 64
    both = dh.lora_gemm(x, w, lora, rows)
    for a in range(4):
        alone = dh.lora_gemm(x, w, lora, torch.full((256,), a, dtype=torch.int32, device="cuda"))
        assert torch.equal(alone[64 * a:64 * a + 64], both[64 * a:64 * a + 64])


@pytest.mark.parametrize("N,K", [(512, 2048), (4096, 4096), (2560, 192)])
def test_many_adapters_in_a_tile(N, K):
    """Each row another adapter, ranks in several parts, the adapters shared out over K
    ranges: right, and a row's bits do not depend on whose rows share its tile."""
    M, R, n = 64, 40, 64
    x, w, lora = case(131, M, N, K, R, n)
    rows = (torch.arange(M, dtype=torch.int32, device="cuda") * 29) % n
    got = dh.lora_gemm(x, w, lora, rows)
    hold(got, x, w, lora, rows)
    for a in (0, 5, 63):
        alone = dh.lora_gemm(x, w, lora, torch.full_like(rows, a))
        at = (rows == a).nonzero()[0, 0]
        assert torch.equal(alone[at], got[at])


def test_captured_calls_replay():
    M, N, K, R, n = 200, 1024, 2048, 16, 4
    x, w, lora = case(91, M, N, K, R, n)
    rows = assign(92, M, n, "requests")
    dh.lora_gemm(x, w, lora, rows)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            y = dh.lora_gemm(x, w, lora, rows)
        graphs.append((g, y))
    for i in range(4):
        x.copy_(rand(93 + i, (M, K)))
        rows.copy_(assign(97 + i, M, n, "mixed"))
        want = dh.lora_gemm(x, w, lora, rows)
        torch.cuda.synchronize()
        for g, _ in graphs:
            g.replay()
        torch.cuda.synchronize()
        for _, y in graphs:
            assert torch.equal(y, want), f"replay {i}"


def test_without_room_for_k_ranges():
    M, N, K, R, n = 200, 1024, 2048, 16, 4
    x, w, lora = case(101, M, N, K, R, n)
    rows = assign(102, M, n, "requests")
    lib = dh.load()
    full, least = lib.dt_lora_gemm_workspace_bytes(M, N, K, R), M * 2 * 32 * 2
    assert full > least
    out = torch.empty((M, N), dtype=BF16, device="cuda")
    p = dh.GemmProblem(x.data_ptr(), K, w.data_ptr(), K, out.data_ptr(), N, None, 0, None, M, N, K, None, 0)
    s = dh.LoraArgs(lora.a.data_ptr(), K, R * K, lora.b.data_ptr(), R, N * R, lora.scale.data_ptr(), rows.data_ptr(), n, R)
    ws = torch.empty(least, dtype=torch.uint8, device="cuda")
    dh.check(lib.dt_lora_gemm(dh.ctypes.addressof(p), dh.ctypes.addressof(s), dh.BF16, ws.data_ptr(), least, dh.stream()))
    hold(out, x, w, lora, rows)


def test_empty_products():
    for M, N in ((0, 64), (5, 0)):
        x, w, lora = case(111, M, N, 64, 8, 2)
        assert dh.lora_gemm(x, w, lora, assign(112, M, 2, "one")).shape == (M, N)
