"""CPU-side checks of rotary positions and the paged cache: what the C entries and the
Python wrappers refuse, the scaled frequencies against their definition, and the cache's
index arithmetic (which pages a call writes, for any contents of the device arrays)
built for the host.  No kernel is launched here."""
import ctypes
import itertools
import math
import os
import random
import subprocess

import pytest
import torch

import dit_hip as dh
from conftest import PKG

ADDR = 1 << 20  # a 16-byte aligned address: no call here gets as far as reading it
BAD_ARG = 1  # DT_ERR_INVALID_ARG


def put(struct, **kw):
    for k, v in kw.items():
        if isinstance(v, tuple):
            getattr(struct, k)[:] = v
        elif "." in k:
            setattr(getattr(struct, k.split(".")[0]), k.split(".")[1], v)
        else:
            setattr(struct, k, v)
    return struct


def refused(fn, *args):
    assert fn(*args) == BAD_ARG
    return dh.load().dt_last_error().decode()


# ------------------------------------------------------------------- rotary --
def rotary_args(**kw):
    """A good call: 2 x 5 tokens, 4 and 2 heads of 64, bf16."""
    a = dh.RotaryArgs()
    put(a, q=ADDR, k=ADDR, q_out=ADDR, k_out=ADDR, q_strides=(1280, 256, 64), q_out_strides=(1280, 256, 64),
        k_strides=(640, 128, 64), k_out_strides=(640, 128, 64), batch=2, seq=5, heads=4, kv_heads=2, head_dim=64, pos=ADDR, pos_stride=5,
        io_type=dh.BF16)
    put(a.rotary, freq=ADDR, rot_dims=64, half=1, attn_factor=1.0)
    for k, v in kw.items():
        put(a.rotary if k in ("freq", "rot_dims", "half", "attn_factor") else a, **{k: v})
    return a


@pytest.mark.parametrize("change,says", [
    (dict(io_type=dh.F16), "io_type"), (dict(batch=-1), "negative"), (dict(seq=-1), "negative"), (dict(heads=-1), "negative"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=4098), "head_dim"), (dict(batch=1 << 20, seq=1 << 20), "too large"),
    (dict(heads=1 << 16), "too large"), (dict(rot_dims=66), "rotated dims"), (dict(rot_dims=7), "rotated dims"), (dict(rot_dims=-2), "rotated dims"),
    (dict(freq=None), "null freq"), (dict(freq=ADDR + 2), "freq"), (dict(attn_factor=math.inf), "attn_factor"),
    (dict(attn_factor=math.nan), "attn_factor"), (dict(q_out=None), "null q_out"), (dict(k_out=None), "null k_out"), (dict(q=ADDR + 1), "aligned"),
    (dict(q_strides=(1280, -256, 64)), "stride"), (dict(k_strides=(1 << 41, 128, 64)), "stride"),
    (dict(q_out_strides=(1280, 256, 0)), "overlap"), (dict(q_out_strides=(1280, 0, 64)), "overlap"), (dict(k_out_strides=(0, 128, 64)), "overlap"),
    (dict(k_out_strides=(640, 64, 64)), "overlap"), (dict(q_out_strides=(1280, 256, 63)), "overlap"),
    (dict(pos=None), "pos"), (dict(pos=ADDR + 2), "pos"), (dict(pos_stride=-1), "pos_stride"),
])
def test_rotary_refuses(change, says):
    a = rotary_args(**change)
    assert says in refused(dh.load().dt_rotary_apply, ctypes.addressof(a), None)


def test_rotary_of_nothing():
    lib = dh.load()
    assert "null arguments" in refused(lib.dt_rotary_apply, None, None)
    for change in (dict(batch=0), dict(seq=0), dict(q=None, k=None), dict(heads=0, kv_heads=0)):
        assert lib.dt_rotary_apply(ctypes.addressof(rotary_args(**change)), None) == 0


@pytest.mark.parametrize("dims,base,factor,context,lo,hi", [
    (128, 10000.0, 1.0, 0, 1.0, 32.0), (64, 10000.0, 4.0, 0, 1.0, 32.0), (128, 1e6, 8.0, 4096, 1.0, 32.0),
    (32, 500000.0, 32.0, 8192, 1.0, 4.0), (2, 10000.0, 2.0, 1, 0.0, 1.0), (0, 10000.0, 2.0, 100, 1.0, 32.0),
])
def test_frequencies(dims, base, factor, context, lo, hi):
    got = dh.rotary_freqs(dims, base, factor, context, lo, hi, device="cpu")
    for i in range(dims // 2):
        f = base ** (-2 * i / dims)
        turns = context * f / (2 * math.pi)
        keep = min(1.0, max(0.0, (turns - lo) / (hi - lo))) if context else 0.0
        want = f * keep + f / factor * (1 - keep)
        # one rounding to 32 bits, beside what 64 bits leave
        assert abs(got[i].item() - want) <= want * (2.0 ** -24 + 1e-14)


@pytest.mark.parametrize("args,says", [
    ((3, 1e4, 1.0, 0, 1.0, 2.0), "even"), ((-2, 1e4, 1.0, 0, 1.0, 2.0), "even"), ((4, 0.0, 1.0, 0, 1.0, 2.0), "positive"),
    ((4, math.inf, 1.0, 0, 1.0, 2.0), "positive"), ((4, 1e4, -1.0, 0, 1.0, 2.0), "positive"), ((4, 1e4, math.nan, 0, 1.0, 2.0), "positive"),
    ((4, 1e4, 2.0, -1, 1.0, 2.0), "context"), ((4, 1e4, 2.0, 10, 2.0, 2.0), "turns"), ((4, 1e4, 2.0, 10, -1.0, 2.0), "turns"),
])
def test_frequencies_refused(args, says):
    buf = (ctypes.c_float * 8)()
    assert says in refused(dh.load().dt_rotary_freq_fill, ctypes.addressof(buf), *args)
    assert "list" in refused(dh.load().dt_rotary_freq_fill, None, 4, 1e4, 1.0, 0, 1.0, 2.0)


# -------------------------------------------------------------------- cache --
def cache(**kw):
    c = dh.KVCacheStruct()
    put(c, k=ADDR, v=ADDR, k_scale=ADDR, v_scale=ADDR, pages=9, kv_heads=2, page=32, head_dim=64, type=dh.F8_E4M3)
    return put(c, **kw)


def seqs(**kw):
    s = dh.KVSeqs()
    put(s, table=ADDR, table_stride=400, table_pages=400, seq_start=ADDR, past=ADDR, seqs=3, rows=7)
    return put(s, **kw)


def append_args(rotary=True, **kw):
    a = dh.KVAppendArgs()
    put(a, k=ADDR, v=ADDR, q=ADDR, q_out=ADDR, k_strides=(128, 64), v_strides=(128, 64), q_strides=(256, 64), q_out_strides=(256, 64),
        heads=4, io_type=dh.BF16)
    r = put(dh.RotaryStruct(), freq=ADDR, rot_dims=64, half=1, attn_factor=1.0)
    if rotary:
        for k in ("freq", "rot_dims", "half", "attn_factor"):
            if k in kw:
                setattr(r, k, kw.pop(k))
        a.rotary = ctypes.addressof(r)
    put(a, **kw)
    a.keep = r
    return a


BAD_CACHE = [
    (dict(type=dh.F32), {}, "cache type"), (dict(type=dh.F16), {}, "cache type"), (dict(head_dim=0), {}, "head_dim"), (dict(head_dim=40), {}, "head_dim"),
    (dict(head_dim=144), {}, "head_dim"), (dict(page=8), {}, "pages of"), (dict(page=48), {}, "pages of"), (dict(page=512), {}, "pages of"),
    (dict(pages=0), {}, "unsupported"), (dict(pages=1 << 31), {}, "unsupported"), (dict(kv_heads=0), {}, "unsupported"),
    (dict(k=None), {}, "k and v"), (dict(v=ADDR + 8), {}, "k and v"), (dict(k_scale=None), {}, "k_scale"), (dict(v_scale=None), {}, "v_scale"),
    ({}, dict(seqs=-1), "out of range"), ({}, dict(rows=1 << 28), "out of range"), ({}, dict(seqs=1 << 20), "out of range"),
    ({}, dict(table_pages=-1), "table"), ({}, dict(table_pages=1 << 26), "table"), ({}, dict(table=None), "table"),
    ({}, dict(table=ADDR + 2), "table"), ({}, dict(table_stride=-4), "table_stride"), ({}, dict(seq_start=None), "seq_start"),
    ({}, dict(past=None), "past"), ({}, dict(seq_start=ADDR + 1), "seq_start"), ({}, dict(past=ADDR + 2), "past"),
]


def attn_call(c, s, q=ADDR, qs=(256, 64), heads=4, causal=1, scale=0.125, o=ADDR, os_=(256, 64), ws=ADDR, n=1 << 40):
    st = [None if t is None else dh._I64x2(*t) for t in (qs, os_)]
    return (ctypes.addressof(c), ctypes.addressof(s), q, st[0], heads, causal, scale, o, st[1], ws, n, None)


@pytest.mark.parametrize("in_cache,in_seqs,says", BAD_CACHE)
def test_cache_refused(in_cache, in_seqs, says):
    lib, c, s, a = dh.load(), cache(**in_cache), seqs(**in_seqs), append_args()
    assert says in refused(lib.dt_kv_append, ctypes.addressof(c), ctypes.addressof(s), ctypes.addressof(a), None)
    assert says in refused(lib.dt_kv_attn, *attn_call(c, s))
    assert lib.dt_kv_attn_workspace_bytes(ctypes.addressof(c), ctypes.addressof(s), 4) == 0


@pytest.mark.parametrize("page", [16, 32, 256])
@pytest.mark.parametrize("more", [0, 1, 5])
def test_tables_of_any_number_of_pages_are_measured(page, more):
    """Pages whose tokens pass 64 bits are too many, like any above 2^30 tokens; 2^30 are not."""
    lib, a = dh.load(), append_args()
    for n in ((1 << 30) // page + 1 + more, (1 << 64) // page + more, (1 << 63) // page - 1 - more, (1 << 63) - 1 - more):
        if n >= 1 << 63:
            continue
        c, s = cache(page=page), seqs(table_pages=n)
        assert "too long" in refused(lib.dt_kv_append, ctypes.addressof(c), ctypes.addressof(s), ctypes.addressof(a), None)
        assert "too long" in refused(lib.dt_kv_attn, *attn_call(c, s))
    c, s = cache(page=page), seqs(table_pages=(1 << 30) // page)
    assert "workspace" in refused(lib.dt_kv_attn, *attn_call(c, s, ws=None))


@pytest.mark.parametrize("change,says", [
    (dict(io_type=dh.F16), "io_type"), (dict(k=None), "null k"), (dict(v=None), "null v"), (dict(k=ADDR + 4), "aligned"),
    (dict(k_strides=(129, 64)), "aligned"), (dict(v_strides=(128, -64)), "stride"), (dict(q_out=None), "null q_out"),
    (dict(q_out_strides=(0, 64)), "overlap"), (dict(q_out_strides=(256, 56)), "overlap"), (dict(q_out_strides=(192, 64)), "overlap"),
    (dict(heads=-1), "out of range"), (dict(freq=None), "null freq"), (dict(rot_dims=80), "rotated dims"), (dict(rot_dims=24), "halves"),
    (dict(attn_factor=math.inf), "attn_factor"), (dict(pos=ADDR + 1), "pos"), (dict(rotary=False), "rotation"),
])
def test_append_refuses(change, says):
    lib, c, s, a = dh.load(), cache(), seqs(), append_args(**change)
    assert says in refused(lib.dt_kv_append, ctypes.addressof(c), ctypes.addressof(s), ctypes.addressof(a), None)


@pytest.mark.parametrize("change,says", [
    (dict(heads=3), "share"), (dict(heads=-2), "share"), (dict(scale=-1.0), "scale"), (dict(scale=math.nan), "scale"),
    (dict(scale=math.inf), "scale"), (dict(q=None), "null q"), (dict(o=None), "null o"), (dict(qs=None), "null q"), (dict(q=ADDR + 8), "aligned"),
    (dict(os_=(256, 60)), "aligned"), (dict(os_=(256, 0)), "overlap"), (dict(qs=(-256, 64)), "stride"), (dict(ws=None), "workspace"),
    (dict(n=16), "workspace"), (dict(ws=ADDR + 4), "workspace"),
])
def test_attention_refuses(change, says):
    assert says in refused(dh.load().dt_kv_attn, *attn_call(cache(), seqs(), **change))


def test_nothing_to_do():
    lib, a = dh.load(), append_args()
    for change in (dict(rows=0), dict(seqs=0)):
        c, s = cache(), seqs(**change, table=None, seq_start=None, past=None)
        assert lib.dt_kv_append(ctypes.addressof(c), ctypes.addressof(s), ctypes.addressof(a), None) == 0
        assert lib.dt_kv_attn(*attn_call(c, s, ws=None, n=0)) == 0
        assert lib.dt_kv_attn_workspace_bytes(ctypes.addressof(c), ctypes.addressof(s), 4) == 0
    assert lib.dt_kv_attn(*attn_call(cache(), seqs(), heads=0, ws=None, n=0)) == 0
    for args in ((None, ctypes.addressof(seqs())), (ctypes.addressof(cache()), None)):
        assert "null arguments" in refused(lib.dt_kv_append, *args, ctypes.addressof(a), None)
    assert "null arguments" in refused(lib.dt_kv_append, ctypes.addressof(cache()), ctypes.addressof(seqs()), None, None)


def test_workspace_goes_by_sizes():
    """The lengths are on the device: the same sizes ask for the same bytes whatever is held."""
    lib = dh.load()
    ask = lambda c, s, heads: lib.dt_kv_attn_workspace_bytes(ctypes.addressof(c), ctypes.addressof(s), heads)  # noqa: E731
    n = ask(cache(), seqs(), 4)
    assert n > 0 and n % 8 == 0
    assert ask(cache(pages=1 << 20), seqs(table_pages=1 << 15), 4) == n
    assert ask(cache(), seqs(table_pages=10), 4) == 0  # short tables: nothing is shared out
    # more rows than sequences: the row blocks' key ranges too, more of them for longer tables
    assert 0 < ask(cache(), seqs(rows=100), 4) < ask(cache(), seqs(rows=100, table_pages=1000), 4)


def test_launches_of_too_many_threads_are_refused():
    """2^32 threads and more in one dimension would be cut short without an error."""
    lib = dh.load()
    rows = (1 << 28) - 1
    c, s = cache(page=16, kv_heads=8), seqs(rows=rows, table_stride=1 << 26, table_pages=1 << 26)
    a = append_args(q=None, k_strides=(512, 64), v_strides=(512, 64))
    assert "grid too large" in refused(lib.dt_kv_append, ctypes.addressof(c), ctypes.addressof(s), ctypes.addressof(a), None)
    c, n = cache(kv_heads=8), (1 << 20) - 1
    for table_pages in (4, 4000):  # blocks of rows whole, and shared out
        s = seqs(seqs=n, rows=n, table_stride=table_pages, table_pages=table_pages)
        wide = (512 * 64, 64)
        assert "grid too large" in refused(lib.dt_kv_attn, *attn_call(c, s, qs=wide, os_=wide, heads=512))


# ---------------------------------------------------------- wrappers' refusals --
def meta(dtype, *shape):
    t = torch.empty(shape, dtype=dtype)
    return t.dtype, t.shape, t.stride(), 0


def test_wrapper_plans_refuse(monkeypatch):
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    bf, f32, i32, u8, f8 = torch.bfloat16, torch.float32, torch.int32, torch.uint8, torch.float8_e4m3fn
    q, k = meta(bf, 5, 4, 64), meta(bf, 5, 2, 64)
    pos, freq = meta(i32, 5), meta(f32, 32)

    def says(text, fn, *args):
        with pytest.raises(dh.DtError, match=text):
            fn(*args)

    plan = dh._rotary_plan.__wrapped__
    says("q or k", plan, None, None, None, None, pos, freq, True, 0)
    says("bf16 or fp32", plan, meta(torch.float16, 5, 4, 64), None, q, None, pos, freq, True, 0)
    says("dim", plan, meta(bf, 5, 64), None, meta(bf, 5, 64), None, pos, freq, True, 0)
    says("share", plan, q, meta(bf, 4, 2, 64), q, k, pos, freq, True, 0)
    says("share", plan, q, meta(f32, 5, 2, 64), q, k, pos, freq, True, 0)
    says("output", plan, q, k, q, meta(bf, 5, 2, 32), pos, freq, True, 0)
    says("pos", plan, q, k, q, k, meta(torch.int64, 5), freq, True, 0)
    says("pos", plan, q, k, q, k, meta(i32, 4), freq, True, 0)
    says("freq", plan, q, k, q, k, pos, meta(torch.float64, 32), True, 0)
    ck, cv, sc = meta(f8, 9, 2, 32, 64), meta(f8, 9, 2, 64, 32), meta(u8, 9, 2)
    table, start, past = meta(i32, 3, 4), meta(i32, 4), meta(i32, 3)
    plan = lambda *a: dh._cache_plan(*a)  # noqa: E731
    says("contiguous", plan, ck, ck, sc, sc, table, start, past, 5)
    says("scale", plan, ck, cv, None, sc, table, start, past, 5)
    says("scale", plan, ck, cv, sc, meta(f32, 9, 2), table, start, past, 5)
    says("e4m3fn or bf16", plan, meta(f32, 9, 2, 32, 64), meta(f32, 9, 2, 64, 32), None, None, table, start, past, 5)
    says("table", plan, ck, cv, sc, sc, meta(torch.int64, 3, 4), start, past, 5)
    says("seq_start", plan, ck, cv, sc, sc, table, meta(i32, 3), past, 5)
    says("past", plan, ck, cv, sc, sc, table, start, meta(i32, 4), 5)
    attn = dh._cache_attn_plan.__wrapped__
    says("q must be", attn, ck, cv, sc, sc, table, start, past, meta(f32, 5, 4, 64), meta(f32, 5, 4, 64), 0)
    says("q must be", attn, ck, cv, sc, sc, table, start, past, meta(bf, 5, 4, 32), meta(bf, 5, 4, 32), 0)
    says("out must", attn, ck, cv, sc, sc, table, start, past, q, meta(bf, 5, 4, 32), 0)
    app = dh._append_plan.__wrapped__
    says("of the cache", app, ck, cv, sc, sc, table, start, past, meta(bf, 5, 3, 64), meta(bf, 5, 3, 64), None, None, None, freq, True, 0)
    says("share a dtype", app, ck, cv, sc, sc, table, start, past, k, meta(f32, 5, 2, 64), None, None, None, freq, True, 0)
    says("rotation", app, ck, cv, sc, sc, table, start, past, k, k, q, q, None, None, None, 0)
    says("q must be", app, ck, cv, sc, sc, table, start, past, k, k, meta(bf, 4, 4, 64), q, None, freq, True, 0)


def test_tensors_elsewhere_are_refused(monkeypatch):
    """The launch goes to the current device: tensors elsewhere never reach it."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    q, pos, freq = meta(torch.bfloat16, 5, 4, 64), meta(torch.int32, 5), meta(torch.float32, 32)
    dh._rotary_plan.__wrapped__(q, None, q, None, pos, freq, True, 0)
    for at, says in ((-1, "the host"), (1, "device 1")):
        with pytest.raises(dh.DtError, match=says):
            dh._rotary_plan.__wrapped__(q, None, q, None, (*pos[:3], at), freq, True, 0)


# ------------------------------------------------------------------- indexes --
INDEX = r"""
#include <stdio.h>
#include <stdlib.h>
#include "kv_index.hpp"
using namespace dit::kv;
// stdin: seqs rows table_pages pages page_log2, seq_start, past, table; stdout: one line per item that exists
int main() {
    Seqs s{};
    if (scanf("%d %d %d %d %d", &s.seqs, &s.rows, &s.table_pages, &s.pages, &s.page_log2) != 5) return 1;
    int32_t *start = new int32_t[s.seqs + 1], *past = new int32_t[s.seqs], *table = new int32_t[s.seqs * s.table_pages + 1];
    for (int i = 0; i <= s.seqs; ++i) scanf("%d", start + i);
    for (int i = 0; i < s.seqs; ++i) scanf("%d", past + i);
    for (int i = 0; i < s.seqs * s.table_pages; ++i) scanf("%d", table + i);
    s.seq_start = start; s.past = past; s.table = table; s.table_stride = s.table_pages;
    for (int64_t item = 0; item < items(s); ++item) {
        int b = -1;  // as the kernels' search: how many sequences begin at or before the item, less one
        for (int i = 0; i < s.seqs; ++i) b += first_item(s, start_of(s, i), i) <= item;
        if (b < 0) continue;
        const Seq q(s, b);
        PageItem it;
        if (!page_item(s, q, b, item, &it)) continue;
        const int page = page_of(s, b, it.begin);
        if (page < 0) continue;
        printf("%d %d %d %d %d %d\n", b, page, it.begin, it.first, it.last, q.row + it.begin - q.past);
    }
}
"""


@pytest.fixture(scope="module")
def index(tmp_path_factory):
    d = tmp_path_factory.mktemp("kv_index")
    src, exe = d / "index.cpp", d / "index"
    src.write_text(INDEX)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(PKG, "csrc"), str(src),
                           "-o", str(exe)])

    def run(rows, pages, log2, start, past, table):
        n = len(past)
        text = [n, rows, len(table[0]) if table else 0, pages, log2, *start, *past, *itertools.chain(*table)]
        out = subprocess.run([str(exe)], input=" ".join(map(str, text)), stdout=subprocess.PIPE, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


@pytest.mark.parametrize("seed", range(12))
def test_every_new_token_is_written_once(index, seed):
    rng = random.Random(seed)
    log2 = rng.choice([4, 5, 6, 8])
    P, n = 1 << log2, rng.choice([1, 2, 7, 65])
    new = [rng.choice([0, 1, 1, 2, P - 1, P, P + 1, 3 * P + rng.randint(0, P)]) for _ in range(n)]
    past = [rng.choice([0, 1, P - 1, P, 2 * P + rng.randint(0, P)]) for _ in range(n)]
    width = max((a + b + P - 1) // P for a, b in zip(new, past)) + 1
    pages = n * width
    order = rng.sample(range(pages), pages)
    table = [order[b * width:(b + 1) * width] for b in range(n)]
    front = rng.choice([0, 3])  # rows before the first sequence belong to none
    start = [front + sum(new[:b]) for b in range(n + 1)]
    rows = start[-1] + rng.choice([0, 5])
    got = index(rows, pages, log2, start, past, table)
    seen = {}
    for b, page, begin, first, last, row0 in got:
        assert begin % P == 0 and 0 <= first < last <= P and table[b][begin // P] == page
        for t in range(first, last):
            assert (b, begin + t) not in seen
            seen[b, begin + t] = row0 + t
    want = {(b, past[b] + i): start[b] + i for b in range(n) for i in range(new[b])}
    assert seen == want


@pytest.mark.parametrize("seed", range(12))
def test_any_device_arrays_stay_in_bounds(index, seed):
    rng = random.Random(100 + seed)
    log2, n, width, pages, rows = rng.choice([4, 8]), rng.choice([1, 5, 70]), rng.choice([1, 3]), rng.choice([1, 6]), rng.choice([1, 40, 700])
    odd = [-2 ** 31, -1, 0, 1, 5, rows, rows + 1, 2 ** 30, 2 ** 31 - 1, rng.randint(0, rows), rng.randint(0, 900)]
    start, past = [rng.choice(odd) for _ in range(n + 1)], [rng.choice(odd) for _ in range(n)]
    table = [[rng.choice([-2 ** 31, -1, 0, pages - 1, pages, 2 ** 31 - 1]) for _ in range(width)] for _ in range(n)]
    for b, page, begin, first, last, row0 in index(rows, pages, log2, start, past, table):
        assert 0 <= b < n and 0 <= page < pages and 0 <= begin < width << log2 and 0 <= first < last <= 1 << log2
        assert 0 <= row0 + first and row0 + last <= rows
        assert table[b][begin >> log2] == page


def test_pages_that_are_none(index):
    # the middle page is missing, the last one lies past the pool
    got = index(64, 4, 4, [0, 64], [0], [[3, -1, 2, 4]])
    assert [(page, begin) for _, page, begin, *_ in got] == [(3, 0), (2, 32)]
    # a table too short for the tokens: those past it are not stored
    got = index(40, 4, 4, [0, 40], [10], [[1, 0]])
    assert [(page, begin, first, last) for _, page, begin, first, last, _ in got] == [(1, 0, 10, 16), (0, 16, 0, 16)]
    assert index(40, 4, 4, [0, 40], [32], [[1, 0]]) == []


# ------------------------------------------------------------------- overlaps --
OVERLAP = r"""
#include <stdio.h>
#include "overlap.hpp"
using namespace dit;
// stdin: pairs of operands, each: address, element bytes, dims, their sizes and strides, width; stdout: 1 or 0 a pair, each way
int main() {
    for (;;) {
        long long at[2], n[2][3], st[2][3], width[2];
        int es[2], dims[2];
        for (int k = 0; k < 2; ++k) {
            if (scanf("%lld %d %d", &at[k], &es[k], &dims[k]) != 3) return 0;
            for (int i = 0; i < dims[k]; ++i) scanf("%lld %lld", &n[k][i], &st[k][i]);
            scanf("%lld", &width[k]);
        }
        int64_t sizes[2][3], strides[2][3];
        for (int k = 0; k < 2; ++k)
            for (int i = 0; i < dims[k]; ++i) sizes[k][i] = n[k][i], strides[k][i] = st[k][i];
        const Strided a((void*)at[0], es[0], dims[0], sizes[0], strides[0], width[0]), b((void*)at[1], es[1], dims[1], sizes[1], strides[1], width[1]);
        printf("%d %d\n", share_memory(a, b), share_memory(b, a));
    }
}
"""


@pytest.fixture(scope="module")
def overlap(tmp_path_factory):
    d = tmp_path_factory.mktemp("overlap")
    src, exe = d / "overlap.cpp", d / "overlap"
    src.write_text(OVERLAP)
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover", "-I", os.path.join(PKG, "csrc"), str(src),
                           "-o", str(exe)])

    def run(pairs):
        text = "\n".join(" ".join(map(str, [at, es, len(n), *itertools.chain(*zip(n, st)), width])) for pair in pairs for at, es, n, st, width in pair)
        out = subprocess.run([str(exe)], input=text, stdout=subprocess.PIPE, text=True, check=True).stdout
        return [tuple(map(int, line.split())) for line in out.splitlines()]

    return run


def touched(at, es, n, st, width):
    return {at + es * sum(i * s for i, s in zip(index, st)) + w for index in itertools.product(*map(range, n)) for w in range(width * es)}


def test_operands_that_share_memory(overlap):
    """Against every byte of either, over layouts of up to three dimensions in any order."""
    rng = random.Random(7)
    pairs = []
    for _ in range(3000):
        one = []
        for _ in range(2):
            width, n, st = rng.randint(1, 6), [rng.randint(1, 4) for _ in range(rng.randint(0, 3))], []
            step = width + rng.choice([0, 0, rng.randint(0, 8), -width])
            for k in n:
                st.append(step)
                step = step * k + rng.choice([0, 0, rng.randint(0, 20)])
            order = rng.sample(range(len(n)), len(n))
            one.append((rng.randint(0, 60), rng.choice([2, 4]), [n[i] for i in order], [st[i] for i in order], width))
        if rng.random() < 0.5:  # one layout, at two places
            one[1] = (one[1][0], *one[0][1:])
        pairs.append(one)
    want = [bool(touched(*a) & touched(*b)) for a, b in pairs]
    assert 500 < sum(want) < 2500
    assert overlap(pairs) == [(w, w) for w in want]


def test_large_operands_that_share_memory(overlap):
    T, H, K, D = 1 << 20, 40, 8, 128
    R = (H + 2 * K) * D
    q, k, v = (0, 2, [T, H], [R, D], D), (2 * H * D, 2, [T, K], [R, D], D), (2 * (H + K) * D, 2, [T, K], [R, D], D)
    flat = (0, 2, [T, H], [H * D, D], D)
    gaps = [(2 * D * i, 2, [T, H], [2 * H * D, 2 * D], D) for i in range(2)]  # two tensors' heads in turn
    batch = [(2 * i * D, 2, [4, T, H], [3 * T * 2 * H * D, 2 * H * D, 2 * D], D) for i in range(2)]
    pairs = [((q, k), 0), ((k, v), 0), ((q, q), 1), ((q, flat), 1), ((k, flat), 1), ((gaps[0], gaps[1]), 0), ((gaps[0], gaps[0]), 1),
             ((gaps[0], flat), 1), ((batch[0], batch[1]), 0), ((batch[0], (2, *batch[1][1:])), 1), ((q, (2 * T * R, *flat[1:])), 0)]
    # sizes and strides at their limits, whose products pass 64 bits
    huge = [(at, 4, [1 << 29, 1 << 16], [(1 << 40) - 4, 1 << 35], 128) for at in (0, 4 * 128, 4 * 64)]
    pairs += [((huge[0], huge[0]), 1), ((huge[0], huge[2]), 1), ((huge[0], (0, 4, [2, 1 << 29], [1 << 39, (1 << 40) - 4], 128)), 1)]
    assert overlap([p for p, _ in pairs]) == [(w, w) for _, w in pairs]


def test_outputs_that_are_partly_inputs_are_refused():
    lib = dh.load()
    # 10 rows of 4 heads of 64 (bf16, 512 bytes); far: another buffer
    far = ADDR + (1 << 20)
    for change, says in ((dict(q_out=ADDR + 512), "q_out is partly q"), (dict(q_out_strides=(2560, 512, 64)), "q_out is partly q"),
                         (dict(k=far, k_out=far + 128), "k_out is partly k"), (dict(k_out=far), "q_out is partly k"),
                         (dict(k=far, k_out=ADDR), "k_out is partly q"),
                         (dict(k=far, k_out=far + 2 ** 18, q_out=far + 2 ** 18), "q_out is partly k_out")):
        assert says in refused(lib.dt_rotary_apply, ctypes.addressof(rotary_args(**change)), None)
    for change, says in ((dict(q_out=ADDR + 512, k=far, v=far), "q_out is partly q"), (dict(v=far), "q_out is partly k"), (dict(k=far), "q_out is partly v"),
                         (dict(q_out_strides=(512, 64), k=far, v=far), "q_out is partly q")):
        assert says in refused(lib.dt_kv_append, ctypes.addressof(cache()), ctypes.addressof(seqs()), ctypes.addressof(append_args(**change)), None)
    for change in (dict(o=ADDR + 512), dict(os_=(512, 64)), dict(o=ADDR + 128)):
        assert "o is partly q" in refused(lib.dt_kv_attn, *attn_call(cache(), seqs(), **change))
