"""The text-serving operators where they can go wrong: at the ends of their types' ranges, among thousands of keys, and
behind tables wider than what is held.  Each against its definition in 64 bits."""
import gc
import math

import pytest
import torch

import dit_hip as dh
from test_gpu_text_serving import BF16, BLOCKS, F8, F32, F64, Pool, attended, check_attention, e4m3, filled, ints, power, rand, round_bf16, same, starts, turned

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


@pytest.mark.parametrize("T,heads,dim,half", [(22600000, 64, 6, True), (70000000, 1, 16, False)])
def test_rotary_of_more_threads_than_a_launch_holds(T, heads, dim, half):
    """2^32 threads and more (a thread a pair, or a wave a token), in place: the first tokens, the last and some between."""
    x = torch.ones((T, heads, dim), dtype=BF16, device="cuda")
    at = torch.cat((torch.arange(200), T - 1 - torch.arange(200), torch.randint(0, T, (3000,), generator=torch.Generator().manual_seed(3)))).cuda()
    rows = rand(4, (at.numel(), heads, dim))
    x[at] = rows
    rows = x[at]  # of a token drawn twice one of them
    pos = (torch.arange(T, dtype=torch.int32, device="cuda") * 7) % 100003
    freq = torch.rand(dim // 2, generator=torch.Generator().manual_seed(5)).cuda()
    dh.rotary(x, None, pos, dh.Rotary(freq, half=half), q_out=x)
    want = turned(rows, pos[at], freq, half)
    assert ((x[at].to(F64) - want).abs() <= 2.0 ** -8 * want.abs() + 8 * 2.0 ** -24 * 12).all()  # terms of at most 6 each


@pytest.mark.parametrize("half", [True, False])
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_rotary_of_one_token_of_each_of_a_batch(dtype, half):
    """[batch, 1, heads, dim] with a position each, k in the strides of a wider row: what the tokens side by side give."""
    B, H, K, D = 37, 6, 2, 64
    q, k = rand(7, (B, 1, H, D), dtype), rand(8, (B, 1, K, 2 * D), dtype)[..., D:]
    pos = torch.randint(0, 100000, (B,), dtype=torch.int32, generator=torch.Generator().manual_seed(9)).cuda()
    r = dh.Rotary(dh.rotary_freqs(D), half=half)
    got, want = dh.rotary(q, k, pos[:, None], r), dh.rotary(q[:, 0], k[:, 0], pos, r)
    assert torch.equal(got[0][:, 0], want[0]) and torch.equal(got[1][:, 0], want[1])


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


@pytest.mark.parametrize("dtype", [F8, BF16])
def test_prepared_appends_repeat(dtype):
    """prepare() keeps what the call points to: its description of the rotation, the sequences and the pages."""
    a, b = Pool(50, [40, 30], 2, 64, 16, dtype), Pool(50, [40, 30], 2, 64, 16, dtype)
    k, v, q, pos = rand(51, (25, 2, 64)), rand(52, (25, 2, 64)), rand(53, (25, 4, 64)), ints(*range(7, 32))
    freq, start, past = dh.rotary_freqs(64), ints(0, 20, 25), ints(3, 17)
    for pool in (a, b):
        for i, n in enumerate((3, 17)):
            pool.fill(i, rand(54 + i, (n, 2, 64), F64), rand(56 + i, (n, 2, 64), F64))
    out, launch = dh.prepare(dh.cache_append, a.cache, k, v, a.table, start, past, rot=dh.Rotary(freq, half=True, attn_factor=1.25), pos=pos, q=q)
    gc.collect()
    for i in range(3):
        for t in (k, v, q):
            t.copy_(rand(60 + i, t.shape))
        out.fill_(7.0)
        launch()
        want = dh.cache_append(b.cache, k, v, b.table, start, past, rot=dh.Rotary(freq, half=True, attn_factor=1.25), pos=pos, q=q)
        assert torch.equal(out, want)
        for s, n in ((0, 23), (1, 22)):
            for x, y in zip(a.held(s, n), b.held(s, n)):
                same(x[3 if s == 0 else 17:], y[3 if s == 0 else 17:], "pages")


# ---------------------------------------------------------------- attention --
def test_attention_reads_every_code_at_every_scale():
    """One token a sequence, so that o is its v: every code at every scale, as bf16 has it."""
    n, D = 254, 128
    c = dh.kv_cache(n, 2, 16, D)
    codes = torch.arange(256, dtype=torch.uint8, device="cuda")
    c.v.view(torch.uint8)[:, :, :, 0] = codes.view(2, D)
    scale = torch.arange(1, 255, dtype=torch.uint8, device="cuda")
    c.v_scale.copy_(scale[:, None].expand(n, 2))
    c.k_scale.fill_(127)
    table = torch.arange(n, dtype=torch.int32, device="cuda")[:, None]
    o = dh.cache_attn(rand(6, (n, 2, D)), c, table, torch.arange(n + 1, dtype=torch.int32, device="cuda"), torch.zeros(n, dtype=torch.int32, device="cuda"))
    x = codes.view(F8).to(F32).to(F64) * torch.exp2(scale.to(F64) - 127)[:, None]
    # from scale 3 on every code is a multiple of bf16's least value, from 247 on the largest are beyond its range
    want = torch.where(x.abs() >= 2.0 ** 128, torch.copysign(torch.full_like(x, math.inf), x), x)
    got = o.view(n, 256).to(F64)
    for i in range(n):
        if i + 1 >= 3:
            same(got[i], want[i], f"scale {i + 1}")
        else:
            bad = (got[i] - want[i]).abs() > 2.0 ** -133
            assert not bad.any(), f"scale {i + 1}: codes {bad.nonzero().flatten().tolist()}"


@pytest.mark.parametrize("page,new,past", [(64, (1, 1), (50, 200)), (16, (2, 1), (50, 200)), (64, (40, 3), (30, 64)), (16, (40, 3), (30, 64)), (64, (300,), (3900,)),
                                           (32, (150,), (4000,)), (64, (2, 3), (6000, 5000))])
def test_attention_of_later_tokens_beyond_bf16(page, new, past):
    """Codes of a token that their scale takes beyond bf16's range: infinite for the row that sees it, nothing to the others."""
    lens = [n + p for n, p in zip(new, past)]
    lens[0] = (lens[0] - 2) // page * page + 1  # the last token begins a page of its own
    past = (lens[0] - new[0],) + tuple(past[1:])
    clean, pool = filled(60, lens, 2, 128, page, F8), filled(60, lens, 2, 128, page, F8)
    q = rand(61, (sum(new), 4, 128))
    args = pool.table, starts(new), ints(*past)
    t, last = lens[0] - 1, new[0] - 1
    p, off = pool.rows[0][t // page], t % page
    for c in (clean, pool):
        c.cache.v[p, 1, :, off] = torch.zeros(128, device="cuda").to(F8)
    base = dh.cache_attn(q, clean.cache, *args)
    for scale, code, x in ((247, 256.0, math.inf), (250, -32.0, -math.inf), (254, 2.0, math.inf)):
        pool.cache.v_scale[p, 1] = scale
        pool.cache.v[p, 1, 77, off] = torch.tensor(code).to(F8)
        want = base.clone()
        want[last, 2:, 77] = x
        same(dh.cache_attn(q, pool.cache, *args), want, f"scale {scale}")
        pool.cache.v[p, 1, 77, off] = torch.tensor(code / 2).to(F8)
        got = dh.cache_attn(q, pool.cache, *args)
        assert torch.equal(got[:last], base[:last]), f"scale {scale}, code {code / 2}"


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("page,new,past", [(64, (1, 1), (50, 200)), (16, (1, 2), (130, 70)), (64, (1, 1, 3), (3000, 900, 64)), (16, (40, 3), (90, 64)),
                                           (64, (300,), (3900,)), (64, (2, 100), (700, 300)), (32, (1,), (4000,))])
def test_attention_to_values_that_are_infinite(dtype, wide, page, new, past):
    """An infinity that all rows see, alone in its page's dim: every row has it, and nothing else changes."""
    lens = [n + p for n, p in zip(new, past)]
    clean, pool = filled(62, lens, 2, 128, page, dtype), filled(62, lens, 2, 128, page, dtype)
    q = rand(63, (sum(new), 4, 128))
    table = torch.nn.functional.pad(pool.table, (0, wide), value=-1)
    args = table, starts(new), ints(*past)
    p, off = pool.rows[0][0], 7
    for c in (clean, pool):
        c.cache.v[p, 1] = torch.zeros((128, page), device="cuda").to(dtype)
    base = dh.cache_attn(q, clean.cache, *args)
    for x in (math.inf, -math.inf):
        if dtype == F8:  # 256 times 2^120
            pool.cache.v_scale[p, 1] = 247
        pool.cache.v[p, 1, 77, off] = torch.tensor(math.copysign(256.0, x)).to(F8) if dtype == F8 else x
        want = base.clone()
        want[:new[0], 2:, 77] = x
        same(dh.cache_attn(q, pool.cache, *args), want, f"{x}")


def key_dims(n, D):
    """Of each place a dim, neighbours' unlike."""
    j = torch.arange(n, device="cuda")
    return (j * 5 + j // D * 3) % D


@pytest.mark.parametrize("wide", [0, 200])
@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", BLOCKS)
def test_every_key_counts_once(dtype, heads, kv_heads, dim, page, seqs, wide):
    """Keys of 0 weigh alike, and each value is 1 in one dim: o is how many of a row's keys have that dim, over their number.
    One of N keys left out, or taken twice, changes a dim by D / N of it, where the result is rounded to 2^-8."""
    new, past = zip(*seqs)
    lens = [n + p for n, p in zip(new, past)]
    assert max(lens) / dim < 100
    pool = Pool(70, lens, kv_heads, dim, page, dtype)
    ones = [torch.nn.functional.one_hot(key_dims(n, dim), dim).to(F64) for n in lens]
    for b, n in enumerate(lens):
        pool.fill(b, torch.zeros((n, kv_heads, dim), dtype=F64, device="cuda"), ones[b][:, None].expand(n, kv_heads, dim))
    table = pool.table if not wide else torch.nn.functional.pad(pool.table, (0, wide), value=-1)
    q = rand(71, (sum(new), heads, dim))
    for causal in (True, False):
        got = dh.cache_attn(q, pool.cache, table, starts(new), ints(*past), causal=causal).to(F64)
        for b, (n, p) in enumerate(seqs):
            if n == 0:
                continue
            seen = p + 1 + torch.arange(n, device="cuda") if causal else torch.full((n,), p + n, device="cuda")
            want = (torch.cumsum(ones[b], 0)[seen - 1] / seen[:, None].to(F64))[:, None]
            a = sum(new[:b])
            # 1 / N and its product in fp32 (2^-24 each), the result's rounding; the counts are exact
            over = (got[a:a + n] - want).abs() - (2.0 ** -8 + 4 * 2.0 ** -24) * want
            assert over.max().item() <= 0, f"sequence {b}, row {int(over.amax((1, 2)).argmax())}"


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", BLOCKS)
def test_a_row_finds_its_key(dtype, heads, kv_heads, dim, page, seqs):
    """Keys of signs, and queries that are one key's each: o is that key's value, wherever it lies.  The first and the last key
    that a row sees, those on both sides of the borders of pages and tiles, others anywhere."""
    new, past = zip(*seqs)
    lens = [n + p for n, p in zip(new, past)]
    pool = Pool(80, lens, kv_heads, dim, page, dtype)
    q, at = torch.zeros((sum(new), heads, dim), dtype=BF16, device="cuda"), []
    g = torch.Generator().manual_seed(81)
    for b, (n, p) in enumerate(seqs):
        k = torch.where(torch.rand((n + p, kv_heads, dim), generator=g) < 0.5, 1.0, -1.0).to(F64).cuda()
        pool.fill(b, k, rand(82 + b, (n + p, kv_heads, dim), F64))
        if n == 0:
            at.append(None)
            continue
        sees = (p + 1 + torch.arange(n))[:, None].expand(n, heads)
        i = torch.arange(n * heads).view(n, heads)
        edge = torch.randint(0, 10 ** 6, (n, heads), generator=g) % (-(-sees // page)) * page - (i // 4) % 2
        edge = torch.where(edge < 0, 0, edge)
        far = torch.randint(0, 10 ** 6, (n, heads), generator=g) % sees
        j = torch.where(i % 4 == 0, sees - 1, torch.where(i % 4 == 1, edge, far)).clamp_max(sees - 1)
        j[:, -1] = torch.where(torch.arange(n) % 3 == 0, 0, j[:, -1])
        at.append(j.cuda())
        kv = (torch.arange(heads, device="cuda") // (heads // kv_heads))[None].expand(n, heads)
        q[sum(new[:b]):sum(new[:b]) + n] = k[at[b], kv].to(BF16)
    # A key's own score is dim, others' a sum of dim signs: dim / 2 behind it is 28 standard deviations (4 at dim 64) ... times 4
    got = dh.cache_attn(q, pool.cache, pool.table, starts(new), ints(*past), scale=4.0)
    for b, (n, p) in enumerate(seqs):
        if n == 0:
            continue
        a, (k, v) = sum(new[:b]), pool.held(b, n + p)
        kv = (torch.arange(heads, device="cuda") // (heads // kv_heads))[None].expand(n, heads)
        want = v[at[b], kv]
        # equal keys share the weight: rows whose key is another's too are left out
        x = 4.0 * torch.stack([q[a:a + n, h].to(F64) @ k[:, h * kv_heads // heads].t().contiguous() for h in range(heads)], 1)
        x = x.masked_fill((torch.arange(n + p, device="cuda")[None] > p + torch.arange(n, device="cuda")[:, None])[:, None], -math.inf)
        alone = (torch.exp(x - 4.0 * dim).sum(-1) - 1) <= 1e-6
        assert alone.float().mean().item() > 0.9
        # the weight's rounding to bf16 and the result's, beside what the others weigh (1e-6, of values up to 6)
        over = ((got[a:a + n].to(F64) - want).abs() - (2 * 2.0 ** -8 + 2.0 ** -16 + 2.0 ** -20) * want.abs() - 2e-5).amax(-1)
        assert over[alone].max().item() <= 0, f"sequence {b}: {(over * alone).argmax().item()}"


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", BLOCKS + [(8, 2, 128, 64, [(1, 1000), (1, 3)]), (40, 1, 96, 16, [(1, 70), (5, 0)]), (4, 4, 64, 32, [(9, 1500)])])
def test_attention_onto_its_queries(dtype, heads, kv_heads, dim, page, seqs):
    """o may be q, here inside wider rows: the bits of a call with a tensor of its own, and nothing else touched."""
    new, past = zip(*seqs)
    pool = filled(95, [n + p for n, p in seqs], kv_heads, dim, page, dtype)
    rows = rand(96, (sum(new) + 3, heads * dim + 64))
    q = rows[:, :heads * dim].unflatten(1, (heads, dim))
    args = pool.cache, pool.table, starts(new, 2), ints(*past)
    for causal in (True, False):
        before = rows.clone()
        want = dh.cache_attn(q, *args, causal=causal, out=q.clone())
        assert dh.cache_attn(q, *args, causal=causal, out=q) is q
        assert torch.equal(q, want) and torch.equal(rows[:, heads * dim:], before[:, heads * dim:])
        rows.copy_(before)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", [
    (8, 2, 128, 64, [(1, 1000)]), (8, 2, 128, 64, [(1, 1000), (1, 3), (1, 64)]), (8, 2, 128, 64, [(512, 0)]), (8, 2, 64, 16, [(100, 0), (1, 50), (3, 7)]),
    (4, 4, 80, 128, [(64, 100)]), (4, 1, 128, 32, [(40, 700), (90, 0)]),
])
def test_tables_wider_than_what_is_held(dtype, heads, kv_heads, dim, page, seqs):
    """A table made for the longest context: whatever it makes of the work, the results stay within their bounds."""
    new, past = zip(*seqs)
    pool = filled(90, [n + p for n, p in seqs], kv_heads, dim, page, dtype)
    q = rand(91, (sum(new), heads, dim))
    for wide in (0, 30, 500, 4000):
        table = torch.nn.functional.pad(pool.table, (0, wide), value=3)  # pages of others behind
        for causal in (True, False):
            check_attention(pool, q, new, past, dh.cache_attn(q, pool.cache, table, starts(new), ints(*past), causal=causal), causal)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("wide", [0, 300])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs", [
    (8, 2, 128, 64, [(0, 10)] * 30 + [(70, 500)] + [(0, 3)] * 39), (8, 2, 64, 16, [(0, 9), (3, 6000), (0, 0)]), (6, 6, 80, 32, [(9, 0)] + [(0, 0)] * 8),
    (4, 1, 128, 128, [(2, 3000), (0, 5), (1, 2000), (0, 4000), (3, 1), (0, 0)]),
])
def test_as_many_rows_as_sequences_shared_unevenly(dtype, heads, kv_heads, dim, page, seqs, wide):
    """What a step of one token each may become when it is replayed: the same numbers of rows and sequences, other lengths."""
    new, past = zip(*seqs)
    assert sum(new) == len(new)
    pool = filled(97, [n + p for n, p in seqs], kv_heads, dim, page, dtype)
    table = torch.nn.functional.pad(pool.table, (0, wide), value=-1)
    q = rand(98, (sum(new), heads, dim))
    for causal in (True, False):
        check_attention(pool, q, new, past, dh.cache_attn(q, pool.cache, table, starts(new), ints(*past), causal=causal), causal)


@pytest.mark.parametrize("dtype", [F8, BF16])
@pytest.mark.parametrize("heads,kv_heads,dim,page,seqs,wide", [
    (32, 8, 128, 64, [(1, 1000)], 0), (8, 2, 128, 64, [(1, 1000), (1, 37), (1, 640)], 100), (16, 16, 64, 32, [(1, 2300 - 70 * b) for b in range(24)], 0),
    (8, 1, 80, 16, [(1, 5000), (2, 300), (0, 7)], 0), (32, 8, 128, 64, [(1, 3000), (300, 0), (4, 2000), (1, 17)], 0), (4, 4, 112, 256, [(1, 4095)], 0),
])
def test_weights_of_few_rows_are_not_rounded_to_eight_bits(dtype, heads, kv_heads, dim, page, seqs, wide):
    """Rows of sequences of up to 32 a key head take their weights as two bf16: 2^-15 of a weight is lost, not 2^-8."""
    new, past = zip(*seqs)
    pool = filled(99, [n + p for n, p in seqs], kv_heads, dim, page, dtype)
    table = torch.nn.functional.pad(pool.table, (0, wide), value=-1)
    q = rand(100, (sum(new), heads, dim))
    got = dh.cache_attn(q, pool.cache, table, starts(new), ints(*past)).to(F64)
    for b, (n, p) in enumerate(seqs):
        if n == 0 or n * heads // kv_heads > 32:
            continue
        a, (k, v) = sum(new[:b]), pool.held(b, n + p)
        want, tol = attended(q[a:a + n], k, v, p, True, dim ** -0.5)
        size, _ = attended(q[a:a + n], k, v.abs(), p, True, dim ** -0.5)
        # the sums over keys have twice the terms
        tol = tol - (2.0 ** -8 - 2.0 ** -15 - 2.0 ** -23 - (n + p) * 2.0 ** -24) * size * (1 + 2.0 ** -7)
        err = (got[a:a + n] - want).abs()
        assert (err <= tol).all(), f"sequence {b}: {int((err > tol).sum())} of {err.numel()}, worst {(err / tol).max().item():.3g}"
