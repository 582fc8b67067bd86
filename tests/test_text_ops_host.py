"""CPU-side checks of masked attention, its gradients and the adapters' product: what
the C entries refuse, what the Python wrappers refuse, and the buckets of a relative
position against their definition in whole numbers.  No kernel is launched here."""
import ctypes
import math

import pytest
import torch

import dit_hip as dh

ADDR = 1 << 20  # a 16-byte aligned address: no call here gets as far as reading it
BAD_ARG = 1  # DT_ERR_INVALID_ARG


def attn_args(**kw):
    """A good call: 2 entries, 4 heads on 2, 5 queries, 9 keys, width 64, bf16."""
    a = dh.AttnArgs()
    a.q = a.k = a.v = ADDR
    a.batch, a.heads, a.kv_heads, a.seq_q, a.seq_kv, a.head_dim = 2, 4, 2, 5, 9, 64
    a.q_strides[:], a.k_strides[:], a.v_strides[:] = (5 * 256, 256, 64), (9 * 128, 128, 64), (9 * 128, 128, 64)
    a.io_type, a.scale = dh.BF16, 0.125
    for k, v in kw.items():
        if k.endswith("strides"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return a


def rel_args(**kw):
    base = dict(rel_table=ADDR, rel_table_stride=4, rel_buckets=32, rel_distance=128, rel_two_sided=1)
    base.update(kw)
    return attn_args(**base)


def grads(**kw):
    y = dh.AttnGrads()
    y.d_o = y.o = y.lse = y.dq = y.dk = y.dv = ADDR
    for n in ("d_o", "o", "dq"):
        getattr(y, n + "_strides")[:] = (5 * 256, 256, 64)
    y.dk_strides[:] = y.dv_strides[:] = (9 * 128, 128, 64)
    y.d_rel_table_stride = 4
    for k, v in kw.items():
        if k.endswith("_strides"):
            getattr(y, k)[:] = v
        else:
            setattr(y, k, v)
    return y


def refused(fn, *args):
    assert fn(*args) == BAD_ARG
    return dh.load().dt_last_error().decode()


BAD_SHARED = [
    (dict(io_type=dh.F16), "io_type"), (dict(batch=-1), "negative"), (dict(seq_q=-1), "negative"), (dict(seq_kv=-5), "negative"),
    (dict(head_dim=0), "head_dim"), (dict(head_dim=60), "head_dim"), (dict(head_dim=136), "head_dim"),
    (dict(kv_heads=3), "share"), (dict(kv_heads=0), "share"), (dict(heads=1), "share"),
    (dict(batch=1 << 20), "too large"), (dict(heads=1 << 16, kv_heads=1 << 16), "too large"), (dict(seq_q=1 << 28), "too large"),
    (dict(seq_kv=1 << 28), "too large"), (dict(heads=1 << 15, kv_heads=1, seq_q=1 << 16), "too large"),
    (dict(scale=-1.0), "scale"), (dict(scale=math.inf), "scale"), (dict(scale=math.nan), "scale"),
    (dict(q=None), "null q"), (dict(k=None), "null k"), (dict(v=None), "null v"),
    (dict(q=ADDR + 8), "aligned"), (dict(k=ADDR + 2), "aligned"),
    (dict(q_strides=(5 * 256, 257, 64)), "aligned"), (dict(v_strides=(9 * 128, 128, 60)), "aligned"),
    (dict(k_strides=(9 * 128, -128, 64)), "unsupported"), (dict(q_strides=(-1280, 256, 64)), "unsupported"),
    (dict(k_strides=(1 << 30, (1 << 23) - 128, 64)), "unsupported"),
    (dict(io_type=dh.F32, k_strides=(1 << 30, (1 << 22) - 64, 64)), "unsupported"),
    (dict(kv_len=ADDR + 2), "aligned"), (dict(q_pos=ADDR + 1), "aligned"),
    (dict(kv_mask=ADDR, kv_mask_stride=-1), "kv_mask_stride"),
]


@pytest.mark.parametrize("change,says", BAD_SHARED)
def test_attention_refuses(change, says):
    lib, a = dh.load(), attn_args(**change)
    p, o = ctypes.addressof(a), dh._i64x3(5 * 256, 256, 64)
    assert says in refused(lib.dt_attn_fwd, p, ADDR, o, None, None, 0, None)
    y = grads()
    assert says in refused(lib.dt_attn_bwd, p, ctypes.addressof(y), ADDR, 1 << 40, None)
    assert lib.dt_attn_fwd_workspace_bytes(p) == 0 and lib.dt_attn_bwd_workspace_bytes(p) == 0


@pytest.mark.parametrize("change,says", [
    (dict(rel_buckets=1), "buckets"), (dict(rel_buckets=33), "buckets"), (dict(rel_buckets=130), "buckets"),
    (dict(rel_buckets=2), "buckets"), (dict(rel_buckets=65, rel_two_sided=0), "buckets"),
    (dict(rel_distance=8), "distance"), (dict(rel_distance=1025), "distance"), (dict(rel_distance=-1), "distance"),
    (dict(rel_table=ADDR + 2), "rel_table"), (dict(rel_table_stride=3), "rel_table"),
])
def test_bias_refuses(change, says):
    lib, a = dh.load(), rel_args(**change)
    p, o = ctypes.addressof(a), dh._i64x3(5 * 256, 256, 64)
    assert says in refused(lib.dt_attn_fwd, p, ADDR, o, None, None, 0, None)
    y = grads(d_rel_table=ADDR)
    assert says in refused(lib.dt_attn_bwd, p, ctypes.addressof(y), ADDR, 1 << 40, None)
    assert lib.dt_attn_fwd_workspace_bytes(p) == 0 and lib.dt_attn_bwd_workspace_bytes(p) == 0


def test_forward_refuses_its_outputs():
    lib, a = dh.load(), attn_args()
    p, good = ctypes.addressof(a), dh._i64x3(5 * 256, 256, 64)
    assert "null o" in refused(lib.dt_attn_fwd, p, None, good, None, None, 0, None)
    assert "null o" in refused(lib.dt_attn_fwd, p, ADDR, None, None, None, 0, None)
    assert "aligned" in refused(lib.dt_attn_fwd, p, ADDR + 4, good, None, None, 0, None)
    assert "lse" in refused(lib.dt_attn_fwd, p, ADDR, good, ADDR + 2, None, 0, None)
    for s in ((0, 256, 64), (5 * 256, 0, 64), (5 * 256, 256, 0), (5 * 256, 64, 64), (1000, 256, 64), (5 * 256, 248, 64)):
        assert "overlap" in refused(lib.dt_attn_fwd, p, ADDR, dh._i64x3(*s), None, None, 0, None)
    assert "null arguments" in refused(lib.dt_attn_fwd, None, ADDR, good, None, None, 0, None)
    # Nothing to compute: nothing is looked at.
    for n in ("batch", "heads", "seq_q"):
        e = attn_args(**{n: 0, "q": None})
        if n == "batch":
            e.k = e.v = None
        assert lib.dt_attn_fwd(ctypes.addressof(e), None, None, None, None, 0, None) == 0


def test_gradients_refuse():
    lib = dh.load()
    a, r = attn_args(), rel_args()
    need = lib.dt_attn_bwd_workspace_bytes(ctypes.addressof(a))
    assert need >= 2 * 2 * 4 * 5 * 4

    def says(y, x=a, ws=ADDR, n=1 << 40):
        return refused(lib.dt_attn_bwd, ctypes.addressof(x), ctypes.addressof(y), ws, n, None)

    for n in ("d_o", "o", "dq", "dk", "dv"):
        assert "null " + n in says(grads(**{n: None}))
        assert "aligned" in says(grads(**{n: ADDR + 8}))
    for n in ("dq", "dk", "dv"):
        assert "overlap" in says(grads(**{n + "_strides": (0, 256, 64)}))
    assert "aligned" in says(grads(d_o_strides=(5 * 256, 256, 65)))
    assert "lse" in says(grads(lse=None)) and "lse" in says(grads(lse=ADDR + 1))
    assert "d_rel_table" in says(grads(d_rel_table=ADDR + 2), r)
    assert "d_rel_table" in says(grads(d_rel_table=ADDR, d_rel_table_stride=3), r)
    assert "workspace" in says(grads(), ws=None) and "workspace" in says(grads(), n=need - 1)
    assert "workspace" in says(grads(), ws=ADDR + 8)
    assert "null gradients" in refused(lib.dt_attn_bwd, ctypes.addressof(a), None, ADDR, 1 << 40, None)


def lora_call(c_type=dh.BF16, problem=None, lora=None, ws=ADDR, n=1 << 40):
    p = dh.GemmProblem()
    p.A, p.lda, p.B, p.ldb, p.C, p.ldc, p.M, p.N, p.K = ADDR, 64, ADDR, 64, ADDR, 32, 8, 32, 64
    l = dh.LoraArgs()
    l.a, l.lda, l.a_stride, l.b, l.ldb, l.b_stride = ADDR, 64, 64 * 16, ADDR, 16, 32 * 16
    l.scale, l.row_adapter, l.adapters, l.rank = ADDR, ADDR, 3, 16
    for k, v in (problem or {}).items():
        setattr(p, k, v)
    for k, v in (lora or {}).items():
        setattr(l, k, v)
    return refused(dh.load().dt_lora_gemm, ctypes.addressof(p), ctypes.addressof(l), c_type, ws, n, None)


def test_adapters_refuse():
    lib = dh.load()
    assert "c_type" in lora_call(c_type=dh.F16)
    for change in (dict(rank=513), dict(rank=-1), dict(adapters=-1), dict(adapters=1 << 24), dict(a=None), dict(b=None),
                   dict(row_adapter=None), dict(a=ADDR + 1), dict(b=ADDR + 1), dict(scale=ADDR + 2),
                   dict(row_adapter=ADDR + 2), dict(lda=63), dict(ldb=15), dict(a_stride=-1), dict(b_stride=-1)):
        assert "dt_lora_gemm" in lora_call(lora=change), change
    for change in (dict(A=None), dict(B=None), dict(C=None), dict(lda=63), dict(ldb=63), dict(ldc=31), dict(M=-1)):
        lora_call(problem=change)
    need = lib.dt_lora_gemm_workspace_bytes(8, 32, 64, 16)
    assert need > 0
    assert "workspace" in lora_call(ws=None) and "workspace" in lora_call(n=8) and "workspace" in lora_call(ws=ADDR + 8)
    assert lib.dt_lora_gemm_workspace_bytes(8, 32, 64, 513) == 0 and lib.dt_lora_gemm_workspace_bytes(-1, 32, 64, 16) == 0
    assert "null" in refused(lib.dt_lora_gemm, None, None, dh.BF16, None, 0, None)


# ---- buckets ---------------------------------------------------------------------------
def bucket(d, side, distance):
    """floor(log(d / near) / log(distance / near) * far) in whole numbers."""
    near = side // 2
    if d < near:
        return d
    far, j = side - near, 0
    while j + 1 < far and d ** far >= near ** (far - j - 1) * distance ** (j + 1):
        j += 1
    return near + j


@pytest.mark.parametrize("buckets,distance,two_sided", [
    (32, 128, True), (32, 128, False), (4, 2, True), (2, 2, False), (3, 2, False), (64, 1024, True), (64, 1024, False), (128, 1024, True),
    (8, 3, True), (20, 100, True), (7, 512, False), (48, 65, False),
])
def test_buckets_are_exact(buckets, distance, two_sided):
    n = 1200
    got = dh.rel_buckets(n, buckets, distance, two_sided).tolist()
    side = buckets // 2 if two_sided else buckets
    for d in range(n):
        t = bucket(d, side, distance)
        assert got[n - 1 - d] == t, -d
        assert got[n - 1 + d] == (t if d == 0 else side + t if two_sided else 0), d
    assert got[0] == side - 1


def test_bucket_list_refuses():
    for n, buckets, distance, two_sided in ((4, 1, 8, False), (4, 2, 8, True), (4, 9, 128, True), (4, 65, 128, False), (4, 130, 128, True),
                                            (4, 32, 8, True), (4, 32, 1025, True), (-1, 32, 128, True)):
        with pytest.raises(dh.DtError):
            dh.rel_buckets(n, buckets, distance, two_sided)
    assert dh.rel_buckets(0, 32, 128).numel() == 0


# ---- the wrappers ----------------------------------------------------------------------
@pytest.fixture
def here(monkeypatch):
    """As if the host were the current device: a wrapper's own checks run up to the launch."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: -1)
    monkeypatch.setattr(dh, "stream", lambda: None)


def z(*shape, dtype=torch.bfloat16):
    return torch.zeros(shape, dtype=dtype)


def test_attention_wrappers_refuse(here):
    q, k, v, f = z(2, 5, 4, 64), z(2, 9, 2, 64), z(2, 9, 2, 64), torch.float32
    n, mask = z(2, dtype=torch.int32), z(2, 9, dtype=torch.uint8)
    tab = z(32, 4, dtype=f)
    rel = dh.RelBias(tab, 128)
    for args, kw in (
            ((q[0], k, v), {}), ((q, k[:1], v[:1]), {}), ((q, k, v[:, :8]), {}), ((q, k[..., :32], v[..., :32]), {}),
            ((q.to(f), k, v), {}), ((q.half(), k.half(), v.half()), {}), ((q, k, v.to(f)), {}),
            ((q.transpose(1, 3).contiguous().transpose(1, 3), k, v), {}),
            ((q, k, v), dict(kv_len=n.long())), ((q, k, v), dict(kv_len=z(3, dtype=torch.int32))),
            ((q, k, v), dict(kv_len=z(2, 2, dtype=torch.int32)[:, 0])), ((q, k, v), dict(kv_mask=mask.float())),
            ((q, k, v), dict(kv_mask=mask[:, :8])), ((q, k, v), dict(kv_mask=z(9, 2, dtype=torch.uint8).t())),
            ((q, k, v), dict(out=z(2, 5, 4, 32))), ((q, k, v), dict(out=z(2, 5, 4, 64, dtype=f))),
            ((q, k, v), dict(scale=-1.0)), ((q, k, v), dict(scale=math.nan)),
            ((q, z(2, 9, 3, 64), z(2, 9, 3, 64)), {}), ((q[..., :60], k[..., :60], v[..., :60]), {}),
            ((q, k, v), dict(out=z(1, 5, 4, 64).expand(2, 5, 4, 64))), ((q[..., 1:57], k[..., 1:57], v[..., 1:57]), {})):
        with pytest.raises(dh.DtError):
            dh.cross_attn(*args, **kw)
    for bad, kw in ((dh.RelBias(tab[:, :3], 128), {}), (dh.RelBias(tab.bfloat16(), 128), {}), (dh.RelBias(tab.t().contiguous().t(), 128), {}),
                    (dh.RelBias(tab[:31], 128), {}), (dh.RelBias(tab, 7), {}), (dh.RelBias(tab, 2000), {}),
                    (rel, dict(q_pos=n.long())), (rel, dict(q_pos=n[:1]))):
        with pytest.raises(dh.DtError):
            dh.rel_attn(q, k, v, bad, **kw)
    o, lse = z(2, 5, 4, 64), z(2, 4, 5, dtype=f)
    for args in ((o[:1], q, k, v, o, lse), (o.to(f), q, k, v, o, lse), (o, q, k, v, o[:, :4], lse), (o, q, k, v, o, lse.double()),
                 (o, q, k, v, o, lse[:, :, :4]), (o, q, k, v, o, z(2, 5, 4, dtype=f).transpose(1, 2))):
        with pytest.raises(dh.DtError):
            dh.cross_attn_bwd(*args)


def test_adapter_wrapper_refuses(here):
    f = torch.float32
    x, w, rows = z(8, 64), z(32, 64), z(8, dtype=torch.int32)
    a, b, s = z(3, 16, 64), z(3, 32, 16), z(3, dtype=f)

    def call(x=x, w=w, a=a, b=b, s=s, rows=rows, **kw):
        dh.lora_gemm(x, w, dh.Lora(a, b, s), rows, **kw)

    q = dh.Q8Weight(z(32, 64, dtype=torch.uint8), z(2, 32, dtype=f))
    for kw in (dict(x=x.to(f)), dict(w=w.to(f)), dict(a=a.half()), dict(b=b.to(f)), dict(w=z(32, 48)), dict(a=z(3, 16, 48)),
               dict(b=z(2, 32, 16)), dict(b=z(3, 31, 16)), dict(b=z(3, 32, 8)), dict(rows=rows.long()), dict(rows=rows[:7]),
               dict(s=s[:2]), dict(s=s.double()), dict(x=z(64, 8).t()), dict(a=z(3, 64, 16).transpose(1, 2)), dict(x=x[0]),
               dict(a=a[0]), dict(bias=z(31, dtype=f)), dict(bias=z(32)), dict(addend=z(8, 32, dtype=f)), dict(addend=z(8, 31)),
               dict(out=z(32, 8).t()), dict(out=z(8, 31)), dict(out_dtype=torch.float16), dict(a=z(3, 600, 64), b=z(3, 32, 600)),
               dict(w=dh.Q8Weight(q.codes, z(1, 32, dtype=f))), dict(w=dh.Q8Weight(q.codes, z(2, 32)))):
        with pytest.raises(dh.DtError):
            call(**kw)


def test_tensors_on_another_device_are_refused(monkeypatch):
    """The launch goes to the current device: tensors elsewhere (here: the host's) are named."""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    monkeypatch.setattr(dh, "stream", lambda: None)
    q, k = z(2, 5, 4, 64), z(2, 9, 4, 64)
    with pytest.raises(dh.DtError, match="host"):
        dh.cross_attn(q, k, k)
    with pytest.raises(dh.DtError, match="host"):
        dh.lora_gemm(z(8, 64), z(32, 64), dh.Lora(z(3, 16, 64), z(3, 32, 16)), z(8, dtype=torch.int32))


def test_adapter_wrapper_refuses_no_rows(here):
    with pytest.raises(dh.DtError, match="row_adapter"):
        dh.lora_gemm(z(8, 64), z(32, 64), dh.Lora(z(3, 16, 64), z(3, 32, 16)), None)


def test_lse_of_one_entry_or_head_may_have_any_stride_there(here):
    """Contiguous as torch counts it: the stride of a dimension of one element is none."""
    for H, all_lse in ((1, z(1, 4, 5, dtype=torch.float32)), (4, z(1, 4, 1, 7, dtype=torch.float32)[..., 0])):
        lse = all_lse[:, :H]
        assert lse.is_contiguous() == (H == 1)
        Sq = lse.shape[2]
        q = z(1, Sq, H, 64)
        args = [dh._meta(q)] * 3 + [None] * 6 + [dh._meta(q), dh._meta(q), dh._meta(lse), -1]
        if H == 1:
            dh._grads_plan(*args)
        else:
            with pytest.raises(dh.DtError, match="lse"):
                dh._grads_plan(*args)
