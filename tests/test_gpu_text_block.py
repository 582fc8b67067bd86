"""The text-conditioning operators together, as a request batch runs them: an encoder's
self attention with its bias, then projections with each request's adapter around the
attention to the encoder's states, and the gradients of both attentions."""
import functools
import math

import pytest
import torch

import dit_hip as dh
from test_gpu_lora import q8

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
U16 = 2.0 ** -8  # half a bf16 step, relative


def rand(seed, shape, dtype=BF16, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(dtype).cuda()


class Block:
    """Three requests of 17 .. 70 text tokens, 40 image tokens each, two of them with adapters."""

    def __init__(self, quant):
        self.B, self.S, self.T, self.H, self.D = 3, 40, 70, 4, 64
        E = self.E = self.H * self.D
        self.text = rand(1, (self.B, self.T, 3, self.H, self.D))
        self.x = rand(2, (self.B * self.S, E))
        self.len = torch.tensor([70, 17, 33], dtype=torch.int32, device="cuda")
        self.rel = dh.RelBias(rand(3, (32, self.H), F32), 128, True)
        self.rows = torch.tensor([0] * self.S + [-1] * self.S + [1] * self.S, dtype=torch.int32, device="cuda")
        self.lora = [dh.Lora(rand(4 + 4 * i, (2, 12, E), std=E ** -0.5), rand(5 + 4 * i, (2, E, 12), std=12 ** -0.5),
                             rand(6 + 4 * i, (2,), F32)) for i in range(2)]
        self.w, self.plain = [], []
        for i in range(2):
            w = rand(12 + i, (E, E), std=E ** -0.5)
            qw, value = q8(w) if quant else (w, w)
            self.w.append(qw)
            self.plain.append(value)
        self.d_out = rand(20, (self.B, self.S, self.H, self.D))

    def run(self):
        q, k, v = self.text.unbind(2)
        states, lse_t = dh.rel_attn(q, k, v, self.rel, kv_len=self.len, return_lse=True)
        xq = dh.lora_gemm(self.x, self.w[0], self.lora[0], self.rows).view(self.B, self.S, self.H, self.D)
        o, lse = dh.cross_attn(xq, states, states, kv_len=self.len, return_lse=True)
        out = dh.lora_gemm(o.view(self.B * self.S, self.E), self.w[1], self.lora[1], self.rows, addend=self.x)
        dq, dk, dv = dh.cross_attn_bwd(self.d_out, xq, states, states, o, lse, kv_len=self.len)
        d_states = dk + dv
        grads = dh.rel_attn_bwd(d_states, q, k, v, states, lse_t, self.rel, kv_len=self.len)
        return out, dq, d_states, *grads

    def linear(self, x, i):
        y = x @ self.plain[i].double().t()
        lo = self.lora[i]
        for a in range(2):
            at = (self.rows == a)[:, None]
            y = y + torch.where(at, lo.scale[a].double() * ((x @ lo.a[a].double().t()) @ lo.b[a].double().t()), 0.0)
        return y

    def attend(self, q, k, v, bias):
        s = torch.einsum("bihd,bjhd->bhij", q, k) * self.D ** -0.5 + bias
        keep = torch.arange(self.T, device="cuda")[None, :] < self.len[:, None]
        return torch.einsum("bhij,bjhd->bihd", s.masked_fill(~keep[:, None, None, :], -math.inf).softmax(-1), v)

    def oracle(self):
        """The same in 64 bits by automatic differentiation, nothing rounded between the steps."""
        text = self.text.double().requires_grad_(True)
        table = self.rel.table.double().requires_grad_(True)
        off = torch.arange(self.T)[None, :] - torch.arange(self.T)[:, None]
        idx = dh.rel_buckets(self.T, 32, 128, True).cuda().long()[(off + self.T - 1).cuda()]
        q, k, v = text.unbind(2)
        states = self.attend(q, k, v, table[idx].permute(2, 0, 1)[None])
        states.retain_grad()
        xq = self.linear(self.x.double(), 0).view(self.B, self.S, self.H, self.D).requires_grad_(True)
        o = self.attend(xq, states, states, 0.0)
        out = self.linear(o.reshape(self.B * self.S, self.E), 1) + self.x.double()
        o.backward(self.d_out.double())
        t = text.grad
        return out.detach(), xq.grad, states.grad, t[:, :, 0], t[:, :, 1], t[:, :, 2], table.grad


# Every value between the steps is rounded to bf16, at most six in a row (the text's P, the states,
# the queries, P, o and out; the gradients' path is as long: the states, P, dS, dk, the sum, dS),
# each by u = 2^-8 of itself; through a softmax an error of a score is an error of
# the weights of that size, and the scores here are sums of 64 terms of up to
# 3 u each, random in sign: below 2 u of a typical weight.  16 u of the largest value of a
# row's tensor therefore bounds the whole.
@pytest.mark.parametrize("quant", [False, True])
def test_block_with_gradients(quant):
    blk = Block(quant)
    names = ("out", "dq", "d_states", "text dq", "text dk", "text dv", "dtable")
    for name, got, want in zip(names, blk.run(), blk.oracle()):
        assert got.shape == want.shape and torch.isfinite(got).all(), name
        err = (got.double() - want).abs().max().item()
        assert err <= 16 * U16 * want.abs().max().item(), f"{name}: {err / want.abs().max().item() / U16:.1f} u"
    # What lies behind a request's tokens reaches nothing, and gets no gradient.
    first = blk.run()
    blk.text[1, 17:, 1:] = math.nan
    for name, a, b in zip(names, first, blk.run()):
        if name in ("text dk", "text dv"):
            assert (b[1, 17:] == 0).all()
        if name == "out":
            assert torch.equal(a, b)


def test_block_captured_beside_eager_calls():
    blk, other = Block(False), Block(True)
    blk.run()
    want0 = other.run()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = blk.run()
    for i in range(4):
        blk.x.copy_(rand(30 + i, blk.x.shape))
        blk.len.copy_(torch.tensor([70 - i, 1 + i, 0 if i == 2 else 60], dtype=torch.int32))
        blk.rows.copy_(blk.rows.roll(13))
        want = blk.run()
        torch.cuda.synchronize()
        graph.replay()
        again = other.run()  # an eager run behind the replay, with workspaces of its own
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert torch.equal(a, b), f"replay {i}"
        for a, b in zip(again, want0):
            assert torch.equal(a, b)


def test_prepared_launches_repeat():
    """prepare() records the launch alone, and its repeats read the tensors as they are then."""
    q, k = rand(40, (2, 9, 4, 64)), rand(41, (2, 1000, 2, 64))
    n = torch.tensor([1000, 3], dtype=torch.int32, device="cuda")
    x, w, rows = rand(42, (19, 128)), rand(43, (72, 128)), torch.zeros(19, dtype=torch.int32, device="cuda")
    lora = dh.Lora(rand(44, (1, 24, 128)), rand(45, (1, 72, 24)))
    o, lse = dh.cross_attn(q, k, k, kv_len=n, return_lse=True)
    for wrapper, args, kw in ((dh.cross_attn, (q, k, k), dict(kv_len=n)), (dh.cross_attn_bwd, (q, q, k, k, o, lse), dict(kv_len=n)),
                              (dh.lora_gemm, (x, w, lora, rows), {})):
        for cache in (dh._attn_plan, dh._grads_plan, dh._lora_plan):
            cache.cache_clear()
        got, launch = dh.prepare(wrapper, *args, **kw)
        assert isinstance(launch, functools.partial)  # one call of the library
        got = got if isinstance(got, tuple) else (got,)
        want = [t.clone() for t in got]
        for t in got:
            t.zero_()
        launch()
        for a, b in zip(got, want):
            assert torch.equal(a, b)
