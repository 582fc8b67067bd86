"""Rotary positions, appending to a paged cache and the attention over it, each against
its definition in 64 bits, and together as a text model's steps run them.

A rounding is off by at most half a step: bf16 2^-8 of the value, fp32 2^-24."""
import math

import pytest
import torch

import dit_hip as dh

pytestmark = pytest.mark.gpu
BF16, F32, F64, F8 = torch.bfloat16, torch.float32, torch.float64, torch.float8_e4m3fn
HALF = {BF16: 2.0 ** -8, F32: 2.0 ** -24}


def rand(seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


# ------------------------------------------------------------------- rotary --
def turned(x, pos, freq, half, mul=1.0, sign=1.0):
    """x [..., H, D] in 64 bits, pos [...]."""
    x = x.to(F64)
    n = 2 * freq.numel()
    a = pos.to(F64)[..., None] * freq.to(F64)
    c, s = (torch.cos(a) * mul)[..., None, :], (torch.sin(a) * mul * sign)[..., None, :]
    u, v = (x[..., :n // 2], x[..., n // 2:n]) if half else (x[..., 0:n:2], x[..., 1:n:2])
    p, q = u * c - v * s, v * c + u * s
    y = torch.cat((p, q), -1) if half else torch.stack((p, q), -1).flatten(-2)
    return torch.cat((y, x[..., n:]), -1)


def reach(x, freq, half, mul):
    """|x| + |its partner|, the size of what a rotated element is a sum of; 0 behind the rotated part."""
    n = 2 * freq.numel()
    a = x.to(F64).abs()
    if half:
        r = a[..., :n // 2] + a[..., n // 2:n]
        r = torch.cat((r, r), -1)
    else:
        r = (a[..., 0:n:2] + a[..., 1:n:2]).repeat_interleave(2, -1)
    return torch.cat((r * abs(mul), torch.zeros_like(a[..., n:])), -1)


def check_turned(got, x, pos, freq, half, mul=1.0, sign=1.0):
    want = turned(x, pos, freq, half, mul, sign)
    # The result's rounding (behind the rotated part there is none); in fp32 the angle (2^-24 of up to pi/4,
    # and of its factor pi/2), the series (2 roundings at its end), the factor, two products and a sum: below 8 roundings of the terms.
    tol = HALF[x.dtype] * want.abs() * (reach(x, freq, half, mul) > 0) + 8 * 2.0 ** -24 * reach(x, freq, half, mul)
    over = (got.to(F64) - want).abs() - tol
    assert got.dtype == x.dtype and over.max().item() <= 0, f"over by {over.max().item():.3g}"


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("dim,rot", [(128, 128), (128, 64), (64, 64), (80, 32), (80, 20), (96, 2), (50, 18), (16, 0), (256, 256), (33, 32)])
@pytest.mark.parametrize("tokens,heads,kv_heads", [(1, 3, 1), (37, 5, 2), (700, 12, 4)])
def test_rotary(half, dtype, dim, rot, tokens, heads, kv_heads):
    q, k = rand(1, (tokens, heads, dim), dtype), rand(2, (tokens, kv_heads, dim), dtype)
    pos = torch.randint(0, 100000, (tokens,), dtype=torch.int32, generator=torch.Generator().manual_seed(3)).cuda()
    r = dh.Rotary(dh.rotary_freqs(rot, 10000.0, 4.0, 4096), half=half, attn_factor=1.25)
    qo, ko = dh.rotary(q, k, pos, r)
    check_turned(qo, q, pos, r.freq, half, 1.25)
    check_turned(ko, k, pos, r.freq, half, 1.25)
    dq, dk = dh.rotary_bwd(q, k, pos, r)
    check_turned(dq, q, pos, r.freq, half, 1.25, -1.0)
    check_turned(dk, k, pos, r.freq, half, 1.25, -1.0)


@pytest.mark.parametrize("half", [True, False])
def test_rotary_positions_of_any_size(half):
    pos = ints(0, 1, -1, 2 ** 31 - 1, -2 ** 31, 1 << 30, 123456789, -7)
    x = rand(4, (8, 2, 64), F32)
    r = dh.Rotary(torch.cat((dh.rotary_freqs(60), torch.tensor([0.0, 3.0], device="cuda"))), half=half)
    a = pos.to(F64)[:, None] * r.freq.to(F64)
    y, _ = dh.rotary(x, None, pos, r)
    want = turned(x, pos, r.freq, half)
    # beside fp32's roundings the angle's own in 64 bits, in the reference too: 2^-53 of up to 7e9 radians, a few times
    tol = 9 * 2.0 ** -24 * reach(x, r.freq, half, 1.0) + 4 * 2.0 ** -53 * a.abs().max() * reach(x, r.freq, half, 1.0)
    assert ((y.to(F64) - want).abs() <= tol).all()


def test_rotary_views_batches_and_in_place():
    """q and k inside one projection's rows, two sequences with positions of their own, written onto themselves."""
    B, S, H, K, D = 2, 19, 6, 2, 64
    rows = rand(5, (B, S, (H + 2 * K) * D))
    q, k = rows[..., :H * D].unflatten(-1, (H, D)), rows[..., H * D:(H + K) * D].unflatten(-1, (K, D))
    pos = torch.stack((torch.arange(S), 50 + torch.arange(S))).to(torch.int32).cuda()
    r = dh.Rotary(dh.rotary_freqs(D), half=True)
    before, q0, k0 = rows.clone(), q.clone(), k.clone()
    qo, ko = dh.rotary(q, k, pos, r)
    check_turned(qo, q0, pos, r.freq, True)
    assert torch.equal(rows, before)
    same = dh.rotary(q, k, pos, r, q_out=q, k_out=k)
    assert same[0] is q and torch.equal(q, qo) and torch.equal(k, ko) and torch.equal(rows[..., (H + K) * D:], before[..., (H + K) * D:])
    # one row of positions for both sequences (stride 0), rows off 16-byte alignment: the same bits
    shared = pos[:1].expand(B, S)
    want = dh.rotary(q0, k0, shared.contiguous(), r)
    pad = torch.empty((B, S, H, D + 3), dtype=BF16, device="cuda")
    off = pad[..., 3:]
    off.copy_(q0)
    got = dh.rotary(off, k0, shared, r, q_out=off)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_rotary_leaves_what_it_does_not_rotate():
    x = torch.full((3, 2, 48), math.nan, dtype=F32, device="cuda")
    x[..., 40] = math.inf
    x[..., 41] = -0.0
    x[..., :32] = rand(6, (3, 2, 32), F32)
    for half in (True, False):
        y, _ = dh.rotary(x, None, ints(1, 2, 3), dh.Rotary(dh.rotary_freqs(32), half=half))
        assert torch.equal(y[..., 32:].view(torch.int32), x[..., 32:].view(torch.int32)) and y[..., :32].isfinite().all()


def test_rotary_gradient_by_differences():
    """The gradient of sum(w rotary(x)) along a direction, against the change of the sum: the map is linear, so the
    difference quotient is exact but for fp32's roundings."""
    x, w, d = (rand(s, (11, 3, 32), F32) for s in (7, 8, 9))
    pos = torch.arange(11, dtype=torch.int32, device="cuda") * 17
    r = dh.Rotary(dh.rotary_freqs(24), half=False, attn_factor=0.75)
    f = lambda v: (dh.rotary(v, None, pos, r)[0].double() * w.double()).sum()  # noqa: E731
    g, _ = dh.rotary_bwd(w, None, pos, r)
    num = (f(x + d) - f(x - d)) / 2
    size = (w.double().abs() * (x.double().abs() + d.double().abs() + 1)).sum() * 2
    assert abs((g.double() * d.double()).sum() - num) <= 16 * 2.0 ** -24 * size


def test_rotary_of_nothing():
    r = dh.Rotary(dh.rotary_freqs(16))
    q = torch.empty((0, 4, 16), dtype=BF16, device="cuda")
    assert dh.rotary(q, q, torch.empty(0, dtype=torch.int32, device="cuda"), r)[0].shape == (0, 4, 16)


# -------------------------------------------------------------------- cache --
class Pool:
    """A cache full of NaN and odd scales, sequences with pages anywhere in it, and what it should hold in 64 bits."""

    def __init__(self, seed, lens, kv_heads, dim, page, dtype, spare=2):
        self.g = torch.Generator().manual_seed(seed)
        self.KH, self.D, self.P, self.dtype = kv_heads, dim, page, dtype
        need = [-(-n // page) for n in lens]
        self.pages = sum(need) + spare
        order = torch.randperm(self.pages, generator=self.g).tolist()
        width = max(need + [1]) + 1
        at = [sum(need[:b]) for b in range(len(lens))]
        self.rows = [[order[at[b] + j] if j < n else (-1 if j & 1 else self.pages + 5) for j in range(width)] for b, n in enumerate(need)]
        self.table = torch.tensor(self.rows, dtype=torch.int32).cuda()
        c = self.cache = dh.kv_cache(self.pages, kv_heads, page, dim, dtype)
        if dtype == F8:
            for t, s in ((c.k, c.k_scale), (c.v, c.v_scale)):
                t.view(torch.uint8).copy_(torch.where(torch.rand(t.shape, generator=self.g) < 0.5, 0x7f, 0xff))
                s.copy_(torch.randint(0, 256, s.shape, generator=self.g))
        else:
            c.k.fill_(math.nan)
            c.v.fill_(math.nan)

    def fill(self, b, k, v):
        """Sequence b's first tokens, [n, KH, D] in 64 bits, as definition of the append has them."""
        for j in range(0, k.shape[0], self.P):
            p = self.rows[b][j // self.P]
            kk, vv = k[j:j + self.P].transpose(0, 1), v[j:j + self.P].permute(1, 2, 0)
            n, c = kk.shape[1], self.cache
            if self.dtype == F8:
                ks, vs = power(kk.abs().amax((1, 2))), power(vv.abs().amax((1, 2)))
                c.k_scale[p], c.v_scale[p] = (ks + 127).to(torch.uint8), (vs + 127).to(torch.uint8)
                kk, vv = kk * torch.exp2(-ks)[:, None, None], vv * torch.exp2(-vs)[:, None, None]
                kk, vv = e4m3(kk), e4m3(vv)
            c.k[p, :, :n] = kk.to(self.dtype)
            c.v[p, :, :, :n] = vv.to(self.dtype)

    def held(self, b, n):
        """What sequence b's first n tokens' k and v stand for, [n, KH, D] in 64 bits."""
        c = self.cache
        rows = torch.tensor(self.rows[b][:-(-n // self.P)], dtype=torch.long, device="cuda")
        k, v = c.k[rows].to(F32).to(F64), c.v[rows].to(F32).to(F64).transpose(2, 3)
        if self.dtype == F8:
            k, v = (t * torch.exp2(s[rows].to(F64) - 127)[..., None, None] for t, s in ((k, c.k_scale), (v, c.v_scale)))
        return tuple(t.transpose(1, 2).reshape(-1, self.KH, self.D)[:n] for t in (k, v))


def power(most):
    """The least e >= -126 with most <= 448 2^e, by trying the neighbours of the logarithm."""
    e = torch.floor(torch.log2(most.clamp_min(2.0 ** -130) / 448)) - 1
    for _ in range(3):
        e = torch.where(most > 448 * torch.exp2(e), e + 1, e)
    return e.clamp_min(-126)


def e4m3(x):
    """The nearest e4m3 in 64 bits, ties to even; NaN for what is not finite."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.where(x.isfinite(), torch.round(x / step) * step, math.nan)


def starts(new, front=0):
    return torch.tensor([front + sum(new[:b]) for b in range(len(new) + 1)], dtype=torch.int32, device="cuda")


def same(got, want, what):
    """Bit for bit, any NaN for a NaN."""
    got, want = got.to(F32).to(F64), want.to(F64)
    bad = ~((got == want) | (got.isnan() & want.isnan()))
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()}, first {bad.nonzero()[0].tolist()}"


def test_conversions_to_e4m3():
    """Every code, every tie between two codes and the fp32 values next to them, through the append (k as it is,
    without a rotation, beside 448, which makes the scale 1)."""
    codes = torch.arange(127, dtype=torch.uint8).view(F8).to(F32)
    ties = (codes[1:] + codes[:-1]) / 2
    x = torch.cat((codes, ties, torch.nextafter(ties, torch.tensor(0.0)), torch.nextafter(ties, torch.tensor(1e9))))
    x = torch.cat((x, -x, torch.tensor([448.0])))
    x = torch.cat((x, torch.zeros(-x.numel() % 128))).view(-1, 1, 128).cuda()
    pool = Pool(1, [x.shape[0]], 1, 128, 16, F8)
    n = x.shape[0]
    dh.cache_append(pool.cache, x, x.flip(0), pool.table, ints(0, n), ints(0))
    k, v = pool.held(0, n)
    assert n <= 16 and pool.cache.k_scale[pool.rows[0][0], 0] == 127
    same(k, e4m3(x.to(F64)), "k")
    same(v, e4m3(x.flip(0).to(F64)), "v")


CASES = [  # (new tokens, past) of each sequence
    [(1, 0)], [(1, 5)], [(1, 63), (1, 64), (1, 65), (1, 0)], [(40, 0)], [(0, 7), (3, 14), (0, 0), (130, 61)], [(200, 100), (1, 300), (17, 0)],
]


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("io", [BF16, F32])
@pytest.mark.parametrize("kv_heads,dim,page,half,rot", [(2, 128, 64, True, 128), (3, 64, 16, False, 64), (1, 80, 32, True, 32), (5, 16, 256, False, 6),
                                                        (2, 112, 128, True, 112), (1, 128, 256, True, 64)])
@pytest.mark.parametrize("case", range(len(CASES)))
def test_append(dtype, io, kv_heads, dim, page, half, rot, case):
    new, past = zip(*CASES[case])
    heads, B, front = 2 * kv_heads, len(new), 2
    pool = Pool(10 + case, [n + p for n, p in CASES[case]], kv_heads, dim, page, dtype)
    T = front + sum(new) + 3
    k, v = rand(20 + case, (T, kv_heads, dim), io, 1.5), rand(30 + case, (T, kv_heads, dim), io, 0.01)
    k[:, 0] *= 300.0  # a head of another size
    q = rand(40 + case, (T, heads, dim), io)
    r = dh.Rotary(dh.rotary_freqs(rot), half=half, attn_factor=1.125)
    seq_start, pasts = starts(new, front), ints(*past)
    want_k, want_v, place = [], [], torch.zeros(T, dtype=torch.int32, device="cuda")
    for b in range(B):
        old_k, old_v = rand(50 + b, (past[b], kv_heads, dim), F64), rand(60 + b, (past[b], kv_heads, dim), F64)
        pool.fill(b, old_k, old_v)
        a, n = front + sum(new[:b]), new[b]
        place[a:a + n] = torch.arange(past[b], past[b] + n, dtype=torch.int32, device="cuda")
        want_k.append((pool.held(b, past[b])[0], turned(k[a:a + n], place[a:a + n], r.freq, half, 1.125)))
        want_v.append((pool.held(b, past[b])[1], v[a:a + n].to(F64)))
    before = [None if t is None else t.clone() for t in (pool.cache.k, pool.cache.v, pool.cache.k_scale, pool.cache.v_scale)]
    q_out = torch.full_like(q, 7.0)
    out = dh.cache_append(pool.cache, k, v, pool.table, seq_start, pasts, rot=r, q=q, q_out=q_out)
    assert out is q_out
    rows = slice(front, front + sum(new))
    check_turned(q_out[rows], q[rows], place[rows], r.freq, half, 1.125)
    assert (q_out[:front] == 7.0).all() and (q_out[front + sum(new):] == 7.0).all()
    # Every page of every sequence: codes of the new tokens and of the earlier ones by the page's new scale.
    touched = set()
    for b in range(B):
        for j in range(0, past[b] + new[b], page):
            p, n = pool.rows[b][j // page], min(page, past[b] + new[b] - j)
            if j + n <= past[b]:
                continue  # full before
            touched.add(p)
            for name, (old, fresh), turn in (("k", want_k[b], lambda t: t), ("v", want_v[b], lambda t: t.transpose(1, 2))):
                x = torch.cat((old, fresh))[j:j + n].transpose(0, 1)
                got = turn(getattr(pool.cache, name)[p])[:, :n]
                if dtype == BF16:
                    same(got, round_bf16(x), f"{name} page {p}")
                    continue
                held = max(past[b] - j, 0)
                ps = getattr(pool.cache, name + "_scale")
                was = before[2 if name == "k" else 3][p].to(F64) - 127
                e = power(x[:, held:].abs().amax((1, 2)))
                e = torch.maximum(e, was) if held else e
                assert torch.equal(ps[p].to(F64) - 127, e), f"{name} scale of page {p}"
                same(got, e4m3(x * torch.exp2(-e)[:, None, None]), f"{name} page {p}")
            rest = turn_rest(pool, before, p, n)
            assert rest
    for p in set(range(pool.pages)) - touched:
        for now, was in zip((pool.cache.k, pool.cache.v, pool.cache.k_scale, pool.cache.v_scale), before):
            assert was is None or torch.equal(now[p].contiguous().view(torch.uint8), was[p].contiguous().view(torch.uint8))


def round_bf16(x):
    """64 bits to bf16 at once (ties to even), in 64 bits."""
    m, e = torch.frexp(x)
    return torch.round(m * 256) * torch.exp2((e - 8).to(F64))  # torch.ldexp takes its power of two in fp32, next to it


def turn_rest(pool, before, p, n):
    """Rows of page p behind its last token are as they were."""
    k, v = pool.cache.k[p][:, n:], pool.cache.v[p][:, :, n:]
    return torch.equal(k.contiguous().view(torch.uint8), before[0][p][:, n:].contiguous().view(torch.uint8)) and \
        torch.equal(v.contiguous().view(torch.uint8), before[1][p][:, :, n:].contiguous().view(torch.uint8))


def test_append_sizes_and_values_at_the_edges():
    """Values that are not finite, zeros, the largest and the smallest: scales and codes by the definition."""
    inf, nan = math.inf, math.nan
    big = torch.finfo(BF16).max
    tokens = [[1.0, inf, -inf, nan], [0.0, 0.0, -0.0, 0.0], [big, -big, 1e30, 1.0], [1e-40, -3e-39, 0.0, 1e-38], [448.0, 448.0, 1.0, 2.0 ** -9],
              [450.0, 1.0, 2.0 ** -10, 0.0], [nan, inf, nan, -inf]]
    pool = Pool(3, [16] * len(tokens), 1, 16, 16, F8)
    x = torch.zeros((len(tokens), 1, 16), dtype=BF16)
    for i, t in enumerate(tokens):
        x[i, 0, :4] = torch.tensor(t)
    x = x.cuda()
    dh.cache_append(pool.cache, x, x, pool.table, torch.arange(len(tokens) + 1, dtype=torch.int32, device="cuda"), ints(*[0] * len(tokens)))
    for b in range(len(tokens)):
        p, t = pool.rows[b][0], x[b, 0].to(F64)
        most = torch.where(t.isfinite(), t.abs(), 0.0).amax()
        e = power(most)
        assert pool.cache.k_scale[p, 0].item() - 127 == e.item() == pool.cache.v_scale[p, 0].item() - 127
        same(pool.cache.k[p, 0, 0], e4m3(t * torch.exp2(-e)), f"token {b}")
        same(pool.cache.v[p, 0, :, 0], e4m3(t * torch.exp2(-e)), f"token {b}")


def test_append_token_by_token_holds_what_one_call_does():
    """A page's scale depends on its tokens alone; codes differ only where a value was rounded below 2^-6 of an earlier scale."""
    n, KH, D, P = 50, 2, 64, 32
    k, v = rand(70, (n, KH, D)), rand(71, (n, KH, D))
    k *= torch.linspace(0.01, 30, n, device="cuda")[:, None, None].to(BF16)  # the scale grows many times
    r = dh.Rotary(dh.rotary_freqs(D), half=True)
    one, many = Pool(5, [n], KH, D, P, F8), Pool(5, [n], KH, D, P, F8)
    dh.cache_append(one.cache, k, v, one.table, ints(0, n), ints(0), rot=r)
    for i in range(n):
        dh.cache_append(many.cache, k[i:i + 1], v[i:i + 1], many.table, ints(0, 1), ints(i), rot=r)
    rows = torch.tensor(one.rows[0][:2], device="cuda")
    assert torch.equal(one.cache.k_scale[rows], many.cache.k_scale[rows]) and torch.equal(one.cache.v_scale[rows], many.cache.v_scale[rows])
    for (a, b), s in zip(zip(one.held(0, n), many.held(0, n)), (one.cache.k_scale, one.cache.v_scale)):
        scale = torch.exp2(s[rows].to(F64) - 127).repeat_interleave(P, 0)[:n, :, None]
        # each rounding below 2^-6 of a scale is off by half of 2^-9 of it at most; scales at least double
        assert ((a - b).abs() <= 2 * 2.0 ** -9 * scale).all()
        normal = b.abs() >= 2.0 ** -6 * scale
        assert normal.any() and torch.equal(a[normal], b[normal])


def test_append_with_given_positions():
    pool = Pool(6, [9, 4], 1, 32, 16, BF16)
    k, v, q = rand(80, (8, 1, 32)), rand(81, (8, 1, 32)), rand(82, (8, 3, 32))
    pos = ints(7, 7, 3, 2 ** 30, -4, 0, 1, 2)
    r = dh.Rotary(dh.rotary_freqs(32), half=False)
    out = dh.cache_append(pool.cache, k, v, pool.table, ints(0, 5, 8), ints(4, 1), rot=r, pos=pos, q=q)
    check_turned(out, q, pos, r.freq, False)
    got = torch.cat((pool.held(0, 9)[0][4:], pool.held(1, 4)[0][1:]))
    want = turned(k, pos, r.freq, False)
    # one rounding, and both sides' angles in 64 bits: 2^-53 of 2^30 radians
    assert ((got - want).abs() <= 2.0 ** -8 * want.abs() + 2.0 ** -20 * 8).all()


def test_append_in_views_and_q_onto_itself():
    """q, k and v inside one projection's rows; q rotated in place; v appended without any rotation."""
    T, H, K, D = 21, 4, 2, 64
    rows = rand(83, (T, (H + 2 * K) * D))
    q, k, v = (rows[:, a * D:b * D].unflatten(1, (-1, D)) for a, b in ((0, H), (H, H + K), (H + K, H + 2 * K)))
    r = dh.Rotary(dh.rotary_freqs(D), half=True)
    a, b = Pool(7, [T], K, D, 16, F8), Pool(7, [T], K, D, 16, F8)
    want = dh.cache_append(a.cache, k.contiguous(), v.contiguous(), a.table, ints(0, T), ints(0), rot=r, q=q.contiguous())
    rest = rows[:, H * D:].clone()
    got = dh.cache_append(b.cache, k, v, b.table, ints(0, T), ints(0), rot=r, q=q, q_out=q)
    assert got is q and torch.equal(q, want) and torch.equal(rows[:, H * D:], rest)
    for x, y in zip(a.held(0, T), b.held(0, T)):
        same(x, y, "pages")


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("half", [True, False])
def test_append_with_nothing_to_rotate(dtype, half):
    """A rotation of no dims: k as it is, q copied."""
    a, b = Pool(8, [40, 3], 2, 48, 16, dtype), Pool(8, [40, 3], 2, 48, 16, dtype)
    k, v, q = rand(84, (30, 2, 48)), rand(85, (30, 2, 48)), rand(86, (30, 4, 48))
    args = ints(0, 28, 30), ints(10, 0)
    dh.cache_append(a.cache, k, v, a.table, *args)
    out = dh.cache_append(b.cache, k, v, b.table, *args, rot=dh.Rotary(torch.zeros(0, device="cuda"), half=half, attn_factor=3.0), q=q)
    assert torch.equal(out, q)
    for s, n in ((0, 38), (1, 2)):
        for x, y in zip(a.held(s, n), b.held(s, n)):
            same(x[10 if s == 0 else 0:], y[10 if s == 0 else 0:], "pages")


def test_append_of_keys_that_share_rows():
    """k and v one tensor, one head's rows standing for all (stride 0): sources may repeat."""
    pool, flat = Pool(9, [20], 3, 32, 16, F8), Pool(9, [20], 3, 32, 16, F8)
    x = rand(87, (20, 1, 32)).expand(20, 3, 32)
    r = dh.Rotary(dh.rotary_freqs(32), half=True)
    dh.cache_append(pool.cache, x, x, pool.table, ints(0, 20), ints(0), rot=r)
    dh.cache_append(flat.cache, x.contiguous(), x.contiguous(), flat.table, ints(0, 20), ints(0), rot=r)
    for x, y in zip(pool.held(0, 20), flat.held(0, 20)):
        same(x, y, "pages")


# ---------------------------------------------------------------- attention --
def attended(q, k, v, past, causal, scale):
    """o [n, H, D] in 64 bits and its tolerance: q [n, H, D], k and v [held, KH, D]."""
    n, H, D = q.shape
    k, v = (t.repeat_interleave(H // t.shape[1], 1).transpose(0, 1).contiguous() for t in (k, v))
    q = q.to(F64).transpose(0, 1).contiguous()
    x = q @ k.transpose(1, 2).contiguous() * scale
    seen = torch.ones((n, k.shape[1]), dtype=torch.bool, device="cuda")
    if causal:
        seen = seen.tril(past)
    x = x.masked_fill(~seen, -math.inf)
    p = torch.nan_to_num(torch.softmax(x, -1), 0.0)  # a row without keys: 0
    o = p @ v
    size = p @ v.abs()
    # Scores: fp32 sums of dim exact products (dim + 1 roundings of the sum of sizes), a product and a difference more.
    terms = (q.abs() @ k.abs().transpose(1, 2).contiguous()).masked_fill(~seen, 0.0) * scale
    off = (D + 4) * 2.0 ** -24 * terms.amax(-1, keepdim=True) + 4 * 2.0 ** -24 * x.masked_fill(~seen, 0.0).abs().amax(-1, keepdim=True)
    # A weight: bf16 (2^-8) and twice its score's error (its own and the sum's); the sums over keys in fp32; the result's rounding.
    keys = k.shape[1]
    tol = 2.0 ** -8 * o.abs() + (2.0 ** -8 + 2 * off + (keys + 64) * 2.0 ** -24) * size * (1 + 2.0 ** -7)
    return o.transpose(0, 1), tol.transpose(0, 1)


def check_attention(pool, q, new, past, got, causal=True, scale=None, front=0):
    D = q.shape[2]
    scale = D ** -0.5 if scale is None else scale
    for b, (n, p) in enumerate(zip(new, past)):
        if n == 0:
            continue
        a = front + sum(new[:b])
        want, tol = attended(q[a:a + n], *pool.held(b, n + p), p, causal, scale)
        err = (got[a:a + n].to(F64) - want).abs()
        assert (err <= tol).all(), f"sequence {b}: {int((~(err <= tol)).sum())} of {err.numel()}, worst {(err / tol).max().item():.3g}"


ATTN = [  # (new tokens, past) of each sequence
    [(1, 0)], [(1, 999)], [(1, 15), (1, 16), (1, 17), (1, 63), (1, 64), (1, 300)], [(0, 40), (1, 4000), (0, 0), (2, 70)], [(5, 0)], [(9, 130), (3, 2)],
    [(40, 0)], [(129, 0), (1, 700)], [(150, 333)], [(300, 0), (65, 64), (1, 1), (7, 1000)], [(1, 20 + 13 * b) for b in range(70)],
]
SHAPES = [(4, 4, 128, 64), (8, 2, 128, 16), (6, 2, 64, 32), (5, 1, 80, 128), (32, 2, 16, 16), (3, 3, 112, 256), (40, 1, 96, 64)]


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page", SHAPES)
@pytest.mark.parametrize("case", range(len(ATTN)))
def test_attention(dtype, heads, kv_heads, dim, page, case):
    new, past = zip(*ATTN[case])
    front = case % 3
    pool = Pool(100 + case, [n + p for n, p in ATTN[case]], kv_heads, dim, page, dtype)
    for b in range(len(new)):
        k, v = rand(200 + b, (new[b] + past[b], kv_heads, dim), F64), rand(300 + b, (new[b] + past[b], kv_heads, dim), F64)
        pool.fill(b, k * (1 + 3 * torch.rand(dim, device="cuda", generator=torch.Generator("cuda").manual_seed(b))), v * 2.0 ** (b % 5))
    T = front + sum(new) + 2
    q = rand(400 + case, (T, heads, dim))
    out = torch.full_like(q, 7.0)
    for causal in (True, False):
        got = dh.cache_attn(q, pool.cache, pool.table, starts(new, front), ints(*past), causal=causal, out=out)
        assert got is out and (out[:front] == 7.0).all() and (out[front + sum(new):] == 7.0).all()
        check_attention(pool, q, new, past, out, causal, front=front)
    assert torch.equal(out, dh.cache_attn(q, pool.cache, pool.table, starts(new, front), ints(*past), causal=False, out=torch.full_like(q, 7.0)))


def filled(seed, lens, kv_heads, dim, page, dtype, std=1.0):
    pool = Pool(seed, lens, kv_heads, dim, page, dtype)
    for b, n in enumerate(lens):
        pool.fill(b, rand(seed + 1 + b, (n, kv_heads, dim), F64, std), rand(seed + 51 + b, (n, kv_heads, dim), F64))
    return pool


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("new,past", [((1, 1), (50, 200)), ((40, 3), (30, 64)), ((130, 1), (0, 9))])
def test_attention_of_later_tokens_that_are_not_numbers(dtype, new, past):
    """A key or value that a row does not see may be NaN; one that it sees makes what it should of the row."""
    lens = [n + p for n, p in zip(new, past)]
    clean, pool = filled(600, lens, 2, 64, 16, dtype), filled(600, lens, 2, 64, 16, dtype)
    q = rand(601, (sum(new), 4, 64))
    args = pool.table, starts(new), ints(*past)
    base = dh.cache_attn(q, clean.cache, *args)
    t = lens[0] - 1  # the first sequence's last token, place t: seen by its last row alone
    p, off = pool.rows[0][t // 16], t % 16
    pool.cache.v[p, 1, 5, off] = math.nan
    got = dh.cache_attn(q, pool.cache, *args)
    last = new[0] - 1
    want = base.clone()
    want[last, 2:, 5] = math.nan  # heads of key head 1, element 5
    same(got, want, "v")
    pool.cache.v[p] = clean.cache.v[p]
    pool.cache.k[p, 0, off, 3] = math.nan
    got = dh.cache_attn(q, pool.cache, *args)
    want = base.clone()
    want[last, :2] = math.nan
    same(got, want, "k")
    if dtype == BF16:
        pool.cache.k[p] = clean.cache.k[p]
        pool.cache.v[p, 0, 7, off] = -math.inf
        got = dh.cache_attn(q, pool.cache, *args)
        want = base.clone()
        want[last, :2, 7] = -math.inf
        same(got, want, "inf")


def test_attention_to_pages_that_are_none():
    """Missing pages in the middle: their tokens are not attended to; none left: 0.  Tokens past the table: not there."""
    P, n = 16, 80
    for dtype in (F8, BF16):
        pool = filled(700, [n, n, n], 1, 32, P, dtype)
        table = pool.table.clone()
        table[0, 1], table[0, 3] = -1, pool.pages
        table[1, :] = -1
        q = rand(701, (6, 2, 32))
        got = dh.cache_attn(q, pool.cache, table, ints(0, 2, 4, 6), ints(n - 2, n - 2, n - 2))
        k, v = pool.held(0, n)
        keep = torch.ones(n, dtype=torch.bool, device="cuda")
        keep[16:32] = keep[48:64] = False
        for i in range(2):
            at = keep.clone()
            at[n - 1 + i:] = False
            want, tol = attended(q[i:i + 1], k[at], v[at], 0, False, 32 ** -0.5)
            assert ((got[i:i + 1].to(F64) - want).abs() <= tol).all()
        assert (got[2:4] == 0).all()
        # a table of two pages: 32 places
        short = dh.cache_attn(q, pool.cache, pool.table[:, :2], ints(0, 2, 4, 6), ints(n - 2, n - 2, n - 2))
        want, tol = attended(q[:2], k[:32], v[:32], 0, False, 32 ** -0.5)
        assert ((short[:2].to(F64) - want).abs() <= tol).all()
        empty = dh.cache_attn(q, pool.cache, pool.table[:, :0], ints(0, 2, 4, 6), ints(0, 5, 7))
        assert (empty == 0).all()


def test_attention_of_extreme_scores():
    """Scores far apart, a scale of 0, and scores of -inf only (a row of weight on nothing is 0)."""
    for dtype in (F8, BF16):
        for new, past in (((1,), (600,)), ((90,), (45,))):
            pool = filled(720, [new[0] + past[0]], 2, 128, 64, dtype, std=20.0)
            q = rand(721, (new[0], 4, 128), std=8.0)
            args = pool.table, starts(new), ints(*past)
            for scale in (None, 0.0, 4.0, 1e-30):
                check_attention(pool, q, new, past, dh.cache_attn(q, pool.cache, *args, scale=scale), scale=scale)
    pool = filled(730, [100], 1, 32, 32, BF16)
    pool.cache.k[:, :, :, 0] = -math.inf
    q = torch.zeros((3, 1, 32), dtype=BF16, device="cuda")
    q[:, :, 0] = 1.0
    assert (dh.cache_attn(q, pool.cache, pool.table, ints(0, 3), ints(97)) == 0).all()


def test_attention_in_views_on_another_stream():
    H, D = 6, 64
    pool = filled(740, [333, 20], 2, D, 32, F8)
    rows = rand(741, (4, (H + 1) * D))
    q = rows[:, :H * D].unflatten(1, (H, D))
    args = pool.table, ints(0, 3, 4), ints(330, 19)
    want = dh.cache_attn(q.contiguous(), pool.cache, *args)
    wide = torch.zeros((4, H, 2 * D), dtype=BF16, device="cuda")
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = dh.cache_attn(q, pool.cache, *args, out=wide[..., D:])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want) and (wide[..., :D] == 0).all()


def test_attention_to_a_shared_prefix():
    """Two sequences whose tables begin with the same pages."""
    pool = filled(750, [64, 80, 96], 2, 64, 16, F8)
    table = pool.table.clone()
    table[1, :3] = table[0, :3]
    pool.rows[1][:3] = pool.rows[0][:3]
    q = rand(751, (3, 8, 64))
    check_attention(pool, q, (1, 1, 1), (60, 79, 95), dh.cache_attn(q, pool.cache, table, ints(0, 1, 2, 3), ints(60, 79, 95)))


def test_attention_far_into_a_large_pool():
    """Pages behind 4 GB of the pool."""
    P, KH, D = 256, 8, 128
    pages = (5 << 30) // (P * KH * D)
    c = dh.kv_cache(pages, KH, P, D, BF16)
    rows = [pages - 1, 3, pages - 2]
    n = 2 * P + 40
    k, v = rand(760, (n, KH, D)), rand(761, (n, KH, D))
    table = torch.tensor([rows], dtype=torch.int32, device="cuda")
    dh.cache_append(c, k, v, table, ints(0, n), ints(0))
    for j, p in enumerate(rows):
        m = min(P, n - j * P)
        assert torch.equal(c.k[p][:, :m], k[j * P:j * P + m].transpose(0, 1)) and torch.equal(c.v[p][:, :, :m], v[j * P:j * P + m].permute(1, 2, 0))
    q = rand(762, (1, KH, D))
    got = dh.cache_attn(q, c, table, ints(0, 1), ints(n - 1))
    want, tol = attended(q, k.to(F64), v.to(F64), n - 1, True, D ** -0.5)
    assert ((got.to(F64) - want).abs() <= tol).all()


BLOCKS = [  # heads, key heads, dim, page, (new tokens, past) of each sequence
    (4, 2, 128, 64, [(300, 3900)]),  # one long sequence: its keys in ranges
    (3, 3, 80, 128, [(70, 4200)]),
    (16, 16, 64, 64, [(2100, 2000)]),  # rows enough without
    (64, 8, 128, 64, [(1900, 2200), (1, 4096), (150, 3), (0, 9)]),
    (8, 2, 128, 64, [(100, 2500), (1, 3000), (40, 0), (1, 5), (0, 70)]),  # few rows beside many, keys in ranges
    (6, 1, 64, 256, [(3, 2100), (90, 1000), (1, 0)]),
    (4, 1, 112, 32, [(70, 2000)]),  # small pages
    (6, 2, 128, 16, [(90, 4100)]),
    (8, 4, 48, 16, [(150, 1200), (2, 900), (1, 3)]),
    (2, 1, 64, 64, [(1, 7 * b) for b in range(70)] + [(0, 3), (65, 64), (17, 1)]),  # more sequences than lanes
    (8, 2, 128, 64, [(1, 6000), (1, 0), (1, 4099)]),  # few rows, shared out
    (32, 32, 128, 64, [(1, 3000 - 70 * b) for b in range(40)]),  # few rows and blocks for every CU
    (64, 64, 64, 64, [(1, 6000 - 900 * b) for b in range(5)]),
]


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", BLOCKS)
def test_attention_of_many_rows_or_long_ones(dtype, heads, kv_heads, dim, page, seqs):
    new, past = zip(*seqs)
    pool = filled(770, [n + p for n, p in seqs], kv_heads, dim, page, dtype)
    q = rand(771, (sum(new) + 3, heads, dim))
    for causal in (True, False):
        out = dh.cache_attn(q, pool.cache, pool.table, starts(new, 2), ints(*past), causal=causal, out=torch.full_like(q, 7.0))
        assert (out[:2] == 7.0).all() and (out[2 + sum(new):] == 7.0).all()
        check_attention(pool, q, new, past, out, causal, front=2)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("page,new,past", [(64, (1, 1), (50, 200)), (64, (40, 3), (30, 64)), (128, (130, 1), (0, 9)), (64, (300,), (3900,)),
                                           (256, (150, 1), (2000, 2500)), (32, (150,), (4000,))])
def test_attention_of_later_tokens_in_pages_of_any_width(dtype, page, new, past):
    """NaN, and with bf16 an infinity, in the last token of a sequence: for its last row alone."""
    lens = [n + p for n, p in zip(new, past)]
    clean, pool = filled(780, lens, 2, 128, page, dtype), filled(780, lens, 2, 128, page, dtype)
    q = rand(781, (sum(new), 4, 128))
    args = pool.table, starts(new), ints(*past)
    base = dh.cache_attn(q, clean.cache, *args)
    t, last = lens[0] - 1, new[0] - 1
    p, off = pool.rows[0][t // page], t % page
    for x in [math.nan] + [math.inf] * (dtype == BF16):
        pool.cache.v[p, 1, 77, off] = x
        want = base.clone()
        want[last, 2:, 77] = x
        same(dh.cache_attn(q, pool.cache, *args), want, f"v {x}")
        pool.cache.v[p] = clean.cache.v[p]
    pool.cache.k[p, 0, off, 99] = math.nan
    want = base.clone()
    want[last, :2] = math.nan
    same(dh.cache_attn(q, pool.cache, *args), want, "k")


def test_append_to_more_sequences_than_lanes():
    new, past = zip(*[(b % 3, 5 * b % 40) for b in range(150)])
    pool = Pool(790, [n + p for n, p in zip(new, past)], 2, 32, 16, BF16)
    k, v, q = rand(791, (sum(new), 2, 32)), rand(792, (sum(new), 2, 32)), rand(793, (sum(new), 4, 32))
    r = dh.Rotary(dh.rotary_freqs(32), half=True)
    place = torch.cat([torch.arange(p, p + n, dtype=torch.int32) for n, p in zip(new, past)]).cuda()
    out = dh.cache_append(pool.cache, k, v, pool.table, starts(new), ints(*past), rot=r, q=q)
    check_turned(out, q, place, r.freq, True)
    want = turned(k, place, r.freq, True)
    for b, (n, p) in enumerate(zip(new, past)):
        a = sum(new[:b])
        got_k, got_v = (x[p:] for x in pool.held(b, n + p))
        same(got_k, round_bf16(want[a:a + n]), f"k of {b}")
        same(got_v, v[a:a + n].to(F64), f"v of {b}")


def test_calls_on_two_streams_at_once():
    """Two streams' calls on one cache, each with scratch of its own, hold what they do one after the other."""
    jobs = []
    for i, (new, past) in enumerate([((1, 1, 1), (3000, 50, 900)), ((100, 1, 40), (2500, 3000, 0))]):
        pool = filled(800 + i, [n + p for n, p in zip(new, past)], 2, 128, 64, F8)
        jobs.append((rand(810 + i, (sum(new), 8, 128)), pool, starts(new), ints(*past)))
    want = [dh.cache_attn(q, p.cache, p.table, s, n) for q, p, s, n in jobs]
    torch.cuda.synchronize()
    sides, got = [torch.cuda.Stream() for _ in jobs], [[], []]
    for _ in range(5):
        for i, (q, p, s, n) in enumerate(jobs):
            with torch.cuda.stream(sides[i]):
                got[i].append(dh.cache_attn(q, p.cache, p.table, s, n))
    torch.cuda.synchronize()
    assert all(torch.equal(g, want[i]) for i in range(2) for g in got[i])


# ----------------------------------------------------------------- together --
class Layer:
    """One layer of a text model on the operators: its projections' rows in, attention out."""

    def __init__(self, dtype, half):
        self.H, self.K, self.D, self.P, self.half = 8, 2, 64, 16, half
        self.pool = Pool(900, [200, 120, 64], self.K, self.D, self.P, dtype)
        self.rot = dh.Rotary(dh.rotary_freqs(self.D, 10000.0, 2.0, 64), half=half, attn_factor=1.0)
        self.tokens = [[], [], []]  # what each sequence got: (k, v) rows

    def step(self, rows, seq_start, past):
        q, k, v = rows.split([self.H * self.D, self.K * self.D, self.K * self.D], 1)
        q, k, v = (t.unflatten(1, (-1, self.D)) for t in (q, k, v))
        q = dh.cache_append(self.pool.cache, k, v, self.pool.table, seq_start, past, rot=self.rot, q=q)
        return dh.cache_attn(q, self.pool.cache, self.pool.table, seq_start, past)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("half", [True, False])
def test_prompts_then_tokens(dtype, half):
    """Prompts of three lengths, tokens one by one, a second piece of one prompt beside them."""
    layer = Layer(dtype, half)
    past = [0, 0, 0]
    for i, new in enumerate([(50, 17, 1), (1, 1, 1), (1, 0, 1), (70, 1, 0), (1, 1, 1), (2, 3, 1)]):
        rows = rand(910 + i, (sum(new), (layer.H + 2 * layer.K) * layer.D))
        o = layer.step(rows, starts(new), ints(*past))
        place = torch.cat([torch.arange(p, p + n) for p, n in zip(past, new)]).cuda()
        q = turned(rows[:, :layer.H * layer.D].unflatten(1, (-1, layer.D)), place, layer.rot.freq, half).to(BF16)
        for b in range(3):
            if new[b] == 0:
                continue
            a = sum(new[:b])
            held_k, held_v = layer.pool.held(b, past[b] + new[b])
            want, tol = attended(q[a:a + new[b]], held_k, held_v, past[b], True, layer.D ** -0.5)
            # beside the attention's own: q in the reference may round to the other side (a bf16 step of it, 2^-7)
            size = (q[a:a + new[b]].to(F64).abs().amax() * held_k.abs().amax() * layer.D ** 0.5 * 2.0 ** -7 * 2.0 ** -16)
            assert ((o[a:a + new[b]].to(F64) - want).abs() <= tol + size * held_v.abs().amax() + 2.0 ** -8 * want.abs()).all()
            # and what is held is the tokens, one rounding to the cache's type
            new_v = rows[a:a + new[b], (layer.H + layer.K) * layer.D:].unflatten(1, (-1, layer.D)).to(F64)
            step = 2.0 ** -4 if dtype == F8 else 0.0
            assert ((held_v[past[b]:] - new_v).abs() <= step * new_v.abs() + (2.0 ** -9 * 4.5 / 224 * 2 if dtype == F8 else 0.0)).all()
        past = [p + n for p, n in zip(past, new)]


@pytest.mark.parametrize("dtype", [F8, BF16])
def test_captured_steps_follow_the_lengths(dtype):
    """One captured step replayed while lengths, starts and tables change in place, eager work and waits between, and
    a second graph of the same operators beside it."""
    H, K, D, P, T = 4, 2, 64, 16, 5
    pool, ref = Pool(950, [90, 90, 90], K, D, P, dtype), Pool(950, [90, 90, 90], K, D, P, dtype)
    rot = dh.Rotary(dh.rotary_freqs(D), half=True)
    q, k, v = (torch.zeros((T, h, D), dtype=BF16, device="cuda") for h in (H, K, K))
    start, past, table = ints(0, 1, 2, 3), ints(0, 0, 0), pool.table.clone()

    def step(c, t):
        return dh.cache_attn(dh.cache_append(c.cache, k, v, t, start, past, rot=rot, q=q), c.cache, t, start, past)

    step(pool, table)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(step(pool, table))
        graphs.append(g)
    held = [0, 0, 0]
    for i, new in enumerate([(1, 1, 1), (3, 0, 2), (1, 2, 1), (5, 0, 0), (0, 4, 1), (1, 1, 1)]):
        for t, s in ((q, 960), (k, 970), (v, 980)):
            t.copy_(rand(s + i, t.shape))
        start.copy_(starts(new))
        past.copy_(ints(*held))
        if i == 3:  # a sequence moves to other pages
            free = [p for p in range(pool.pages) if p not in sum((r[:6] for r in pool.rows), [])][0]
            for c in (pool, ref):
                old = c.rows[0][0]
                for t in (c.cache.k, c.cache.v, c.cache.k_scale, c.cache.v_scale):
                    if t is not None:
                        t[free] = t[old]
                c.rows[0][0] = free
            table[0, 0] = free
        n = sum(new)
        want = step(ref, table)
        torch.cuda.synchronize()
        for g, o in zip(graphs, outs):
            o.fill_(9.0)
            g.replay()
            torch.cuda.synchronize()
            assert torch.equal(o[:n], want[:n]) and (o[n:] == 9.0).all()
        held = [p + m for p, m in zip(held, new)]


def test_prepared_launches_repeat():
    pool = filled(990, [77], 2, 64, 16, F8)
    q = rand(991, (2, 4, 64))
    start, past = ints(0, 2), ints(75)
    o, launch = dh.prepare(dh.cache_attn, q, pool.cache, pool.table, start, past)
    want = o.clone()
    o.zero_()
    launch()
    assert torch.equal(o, want)
    x = rand(992, (3, 2, 64))
    pos, rot = ints(1, 2, 3), dh.Rotary(dh.rotary_freqs(64))
    (y, _), launch = dh.prepare(dh.rotary, x, None, pos, rot)
    want = y.clone()
    y.zero_()
    launch()
    assert torch.equal(y, want)
