"""The text-conditioning operators as timed cases: low-rank adapters of many
requests beside a shared Linear, cross attention to an encoder's states, and
attention with a learned relative position bias.

listed() holds fixed cases, draw(rng) gives more of the same ranges;
prepare(case, seed) makes what a program has in hand before the call,
run(state) is one pass, work(case) its least bytes and operations,
exact(case, seed) the same outputs in 64 bits from the definition.

With `own` false run() computes the operators in their plain form (elementary
torch operations in 32 bits, rounded once at the end); with `own` true it
calls the library.

Kinds of case:
  lora   rows x [n, k] Linear, each row with the low-rank adapter of its request (or none)
  cross  attention of q tokens to the states of an encoder: their number differs by
         request (a length or a mask), query heads may share key heads;
         train adds the gradients of q, k and v
  rel    attention with the bias table[bucket(key - query)] per head; train adds the
         gradients of q, k, v and the table
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
ES = {"bf16": 2, "f32": 4}
WBYTES = {"bf16": 2.0, "q8_0": 1.125}


# ---------------------------------------------------------------- the cases --
def listed():
    return [
        # One token of one request through a projection: the smallest call, a
        # stream of the weight.
        {"name": "lora_1row", "kind": "lora", "rows": 1, "n": 4096, "k": 4096, "rank": 16, "adapters": 8,
         "requests": 1, "weights": "bf16"},
        # A decoding step of sixteen requests, nearly all with adapters of their own.
        {"name": "lora_16rows", "kind": "lora", "rows": 16, "n": 12288, "k": 4096, "rank": 64, "adapters": 32,
         "requests": 16, "weights": "bf16"},
        # Five prompts of ragged lengths through a text encoder's projection kept
        # as Q8_0, adapters of an odd rank.
        {"name": "lora_1628_q8", "kind": "lora", "rows": 1628, "n": 9216, "k": 2560, "rank": 20, "adapters": 6,
         "requests": 5, "weights": "q8_0"},
        # Two images of 2304 tokens, each with a style of its own: the largest product.
        {"name": "lora_4608", "kind": "lora", "rows": 4608, "n": 12288, "k": 4096, "rank": 32, "adapters": 4,
         "requests": 2, "weights": "bf16"},
        # The image tokens of two 1024 x 1024 images to prompts of up to 512 tokens.
        {"name": "cross_4096x512", "kind": "cross", "dtype": "bf16", "batch": 2, "heads": 24, "kv_heads": 24, "q": 4096,
         "kv": 512, "dim": 128, "mask": "len", "train": False},
        # One new token of sixteen requests to long encoded documents, four query
        # heads to a key head.
        {"name": "cross_1token", "kind": "cross", "dtype": "bf16", "batch": 16, "heads": 32, "kv_heads": 8, "q": 1,
         "kv": 6144, "dim": 128, "mask": "len", "train": False},
        # A training step of the image tokens of four 512 x 512 images against
        # 77 prompt tokens, some dropped by a mask.
        {"name": "cross_train_1024x77", "kind": "cross", "dtype": "bf16", "batch": 4, "heads": 16, "kv_heads": 16,
         "q": 1024, "kv": 77, "dim": 64, "mask": "mask", "train": True},
        # A training step with shared key heads and long sequences.
        {"name": "cross_train_2048x1500", "kind": "cross", "dtype": "bf16", "batch": 1, "heads": 16, "kv_heads": 4,
         "q": 2048, "kv": 1500, "dim": 128, "mask": "none", "train": True},
        # A training step in 32 bits at odd sizes.
        {"name": "cross_train_f32", "kind": "cross", "dtype": "f32", "batch": 2, "heads": 8, "kv_heads": 8, "q": 333,
         "kv": 154, "dim": 64, "mask": "len", "train": True},
        # A text encoder's own attention over four padded prompts.
        {"name": "rel_512", "kind": "rel", "dtype": "bf16", "batch": 4, "heads": 64, "q": 512, "kv": 512, "dim": 64,
         "buckets": 32, "distance": 128, "two_sided": True, "train": False},
        # One new token of eight requests to its own past, with the bias of its position.
        {"name": "rel_1token", "kind": "rel", "dtype": "bf16", "batch": 8, "heads": 32, "q": 1, "kv": 2000, "dim": 64,
         "buckets": 32, "distance": 128, "two_sided": False, "train": False},
        # A training step of a text encoder at an odd length.
        {"name": "rel_train_500", "kind": "rel", "dtype": "bf16", "batch": 8, "heads": 12, "q": 500, "kv": 500,
         "dim": 64, "buckets": 32, "distance": 128, "two_sided": True, "train": True},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["lora", "cross", "rel"])
    if kind == "lora":
        rows = _log(rng, 1, 4608)
        return {"kind": kind, "rows": rows, "n": rng.choice([2560, 4096, 9216, 4 * _log(rng, 32, 3000)]),
                "k": rng.choice([2560, 4096, 64 * rng.randint(4, 64)]), "rank": rng.choice([4, 8, 16, 32, 64, 128, rng.randint(1, 96)]),
                "adapters": rng.randint(1, 32), "requests": min(rows, _log(rng, 1, 32)),
                "weights": rng.choice(["bf16", "bf16", "q8_0"])}
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    train = rng.random() < 0.5
    one = not train and rng.random() < 0.4
    if kind == "cross":
        dim = rng.choice([64, 128, 128, 8 * rng.randint(4, 16)])
        shared = rng.choice([1, 1, 2, 4])
        kv_heads = rng.choice([2, 4, 8, 12]) // (2 if shared == 4 else 1)
        top = 400 if dtype == "f32" else 2048
        return {"kind": kind, "dtype": dtype, "batch": rng.randint(1, 16) if one else rng.randint(1, 2),
                "heads": kv_heads * shared, "kv_heads": kv_heads, "q": rng.choice([1, 1, 2, 5]) if one else _log(rng, 17, top),
                "kv": _log(rng, 64, 8192) if one else _log(rng, 9, min(top, 1024)), "dim": dim,
                "mask": rng.choice(["none", "len", "mask"]), "train": train}
    n = _log(rng, 24, 300 if dtype == "f32" else 700)
    buckets, distance = rng.choice([(32, 128), (32, 128), (16, 64), (64, 256)])
    return {"kind": kind, "dtype": dtype, "batch": rng.randint(1, 8), "heads": rng.choice([6, 8, 12, 16]),
            "q": 1 if one else n, "kv": _log(rng, 64, 4096) if one else n, "dim": rng.choice([64, 64, 128]),
            "buckets": buckets, "distance": distance, "two_sided": not one, "train": train}


def _lengths(c):
    """The encoder tokens of each request: from all down to a quarter."""
    return [c["kv"] - (b * 3 * c["kv"]) // (4 * c["batch"]) for b in range(c["batch"])]


def _requests(c):
    """Rows of each request: ragged, every one with a row at least."""
    n, left = c["requests"], c["rows"] - c["requests"]
    w = [1 + (5 * i) % 7 for i in range(n)]
    rows = [1 + left * x // sum(w) for x in w]
    rows[0] += c["rows"] - sum(rows)
    return rows


# ------------------------------------------------------------- prepare, run --
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def prepare(case, seed):
    c = case
    g = _gen(seed)
    s = {"case": c}
    if c["kind"] == "lora":
        s["x"] = _randn(g, (c["rows"], c["k"]), torch.bfloat16)
        w = torch.randn((c["n"], c["k"]), device="cuda", generator=g) * c["k"] ** -0.5
        if c["weights"] == "q8_0":  # uint8 codes and block scales, as a loaded checkpoint has them
            blocks = w.view(c["n"], c["k"] // 32, 32)
            d = (blocks.abs().amax(-1) / 127).half().float()
            q = torch.round(blocks / d.clamp_min(1e-8)[..., None]).clamp(-127, 127)
            s["codes"] = (q + 128).to(torch.uint8).view(c["n"], c["k"])
            s["scales"] = d.t().contiguous()
        else:
            s["w"] = w.to(torch.bfloat16)
        s["bias"] = torch.randn(c["n"], device="cuda", generator=g) * 0.1
        s["a"] = _randn(g, (c["adapters"], c["rank"], c["k"]), torch.bfloat16, c["k"] ** -0.5)
        s["b"] = _randn(g, (c["adapters"], c["n"], c["rank"]), torch.bfloat16, 0.3 * c["rank"] ** -0.5)
        s["scale"] = 0.5 + torch.rand(c["adapters"], device="cuda", generator=g)
        # Each request's adapter; about one of seven has none (-1).
        of = torch.randint(0, c["adapters"], (c["requests"],), device="cuda", generator=g)
        of = torch.where(torch.rand(c["requests"], device="cuda", generator=g) < 0.15, -1, of)
        of[0] = torch.clamp(of[0], min=0)
        s["row_adapter"] = torch.repeat_interleave(of, torch.tensor(_requests(c), device="cuda")).to(torch.int32)
        return s
    dt, B, H, D = DTYPES[c["dtype"]], c["batch"], c["heads"], c["dim"]
    kvh = c.get("kv_heads", H)
    rel = c["kind"] == "rel"
    # The relative form has no scale of its own: its queries are small already.
    s["scale"] = 1.0 if rel else D ** -0.5
    s["q"] = _randn(g, (B, c["q"], H, D), dt, D ** -0.5 if rel else 1.0)
    s["k"] = _randn(g, (B, c["kv"], kvh, D), dt)
    s["v"] = _randn(g, (B, c["kv"], kvh, D), dt)
    s["kv_len"] = s["kv_mask"] = s["q_pos"] = None
    if rel or c["mask"] == "len":
        order = torch.randperm(B, device="cuda", generator=g)
        s["kv_len"] = torch.tensor(_lengths(c), device="cuda", dtype=torch.int32)[order].contiguous()
    elif c["mask"] == "mask":  # a quarter of the tokens left out, at other places in each request
        keep = torch.rand((B, c["kv"]), device="cuda", generator=g).argsort(1) >= c["kv"] // 4
        s["kv_mask"] = keep.to(torch.uint8)
    if rel:
        s["table"] = torch.randn((c["buckets"], H), device="cuda", generator=g)
        if c["q"] == 1:  # the new token stands behind the past it reads
            s["q_pos"] = s["kv_len"] - 1
    if c["train"]:
        s["do"] = _randn(g, (B, c["q"], H, D), dt)
    return s


_dit_hip = None


def _library():
    global _dit_hip
    if _dit_hip is None:
        sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "diffusers-cpp_amd"))
        import dit_hip
        _dit_hip = dit_hip
    return _dit_hip


def run(state):
    if own:
        return _run_own(state)
    c = state["case"]
    return _plain_lora(state) if c["kind"] == "lora" else _plain_attn(state)


def _run_own(s):
    dh = _library()
    c = s["case"]
    if c["kind"] == "lora":
        w = dh.Q8Weight(s["codes"], s["scales"]) if c["weights"] == "q8_0" else s["w"]
        return dh.lora_gemm(s["x"], w, dh.Lora(s["a"], s["b"], s["scale"]), s["row_adapter"], bias=s["bias"])
    keys = {"kv_len": s["kv_len"], "scale": s["scale"]}
    if c["kind"] == "cross":
        keys["kv_mask"] = s["kv_mask"]
        if not c["train"]:
            return dh.cross_attn(s["q"], s["k"], s["v"], **keys)
        o, lse = dh.cross_attn(s["q"], s["k"], s["v"], return_lse=True, **keys)
        return (o, *dh.cross_attn_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, **keys))
    rel = dh.RelBias(s["table"], c["distance"], c["two_sided"])
    keys["q_pos"] = s["q_pos"]
    if not c["train"]:
        return dh.rel_attn(s["q"], s["k"], s["v"], rel, **keys)
    o, lse = dh.rel_attn(s["q"], s["k"], s["v"], rel, return_lse=True, **keys)
    return (o, *dh.rel_attn_bwd(s["do"], s["q"], s["k"], s["v"], o, lse, rel, **keys))


def _weights(s, dtype):
    """The shared weight: a Q8_0 one is worth its bf16 rounding, as the library defines it."""
    if "w" in s:
        return s["w"].to(dtype)
    w = (s["codes"].float().view(s["codes"].shape[0], -1, 32) - 128) * s["scales"].t()[..., None]
    return w.to(torch.bfloat16).to(dtype).view(s["codes"].shape)


def _plain_lora(s):
    """y = x W' + bias + scale (x A') B', the adapters side by side and each row's own kept."""
    n, r, k = s["a"].shape
    x = s["x"].float()
    y = x @ _weights(s, torch.float32).t() + s["bias"]
    t = (x @ s["a"].float().view(n * r, k).t()).view(-1, n, r)
    mine = (torch.arange(n, device=x.device) == s["row_adapter"][:, None]) * s["scale"]
    t = (t * mine[..., None]).view(-1, n * r)
    y += t @ s["b"].float().transpose(1, 2).reshape(n * r, -1)
    return y.to(torch.bfloat16)


def _kept(s):
    """[B, kv] truth values: the keys that are attended to."""
    B, n = s["k"].shape[:2]
    if s["kv_len"] is not None:
        return torch.arange(n, device=s["k"].device) < s["kv_len"][:, None]
    if s["kv_mask"] is not None:
        return s["kv_mask"] != 0
    return torch.ones((B, n), dtype=torch.bool, device=s["k"].device)


def _plain_buckets(s):
    """The bucket of every (batch, query, key): distances up to half of a side's
    buckets one by one, the others by the logarithm, in 64 bits next to a border."""
    c = s["case"]
    at = s["q_pos"] if s["q_pos"] is not None else torch.zeros(1, dtype=torch.int32, device=s["k"].device)
    off = torch.arange(c["kv"], device=at.device) - (at[:, None] + torch.arange(c["q"], device=at.device))[..., None]
    side = c["buckets"] // 2 if c["two_sided"] else c["buckets"]
    dist = off.abs() if c["two_sided"] else (-off).clamp_min(0)
    near = side // 2
    far = torch.log(dist.clamp_min(1).double() / near) / math.log(c["distance"] / near) * (side - near)
    far = (near + torch.floor(far + 1e-9).long()).clamp_max(side - 1)
    return torch.where(dist < near, dist, far) + (side * (off > 0) if c["two_sided"] else 0)


def _plain_attn(s):
    c = s["case"]
    B, S, H, D = s["q"].shape
    shared = H // s["k"].shape[2]
    keep = _kept(s)[:, None, None, :]
    here = keep[:, 0, 0, :, None, None]  # [B, kv, 1, 1]
    q = s["q"].float().transpose(1, 2)
    k = torch.where(here, s["k"].float(), 0.0).repeat_interleave(shared, 2).transpose(1, 2).contiguous()
    v = torch.where(here, s["v"].float(), 0.0).repeat_interleave(shared, 2).transpose(1, 2).contiguous()
    x = (q @ k.transpose(2, 3).contiguous()) * s["scale"]
    if c["kind"] == "rel":
        bucket = _plain_buckets(s)
        x = x + s["table"][bucket].permute(0, 3, 1, 2)
    x = x.masked_fill(~keep, -math.inf)
    p = torch.exp(x - x.amax(-1, keepdim=True))
    p = p / p.sum(-1, keepdim=True)
    o = (p @ v).transpose(1, 2).to(s["q"].dtype).contiguous()
    if not c["train"]:
        return o
    do = s["do"].float().transpose(1, 2)
    dp = do @ v.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True))
    dv = p.transpose(2, 3).contiguous() @ do
    dq = (ds @ k) * s["scale"]
    dk = (ds.transpose(2, 3).contiguous() @ q) * s["scale"]

    def own_heads(t):  # the gradients of the query heads that share a key head, summed
        return t.view(B, -1, shared, c["kv"], D).sum(2).transpose(1, 2).to(s["k"].dtype).contiguous()

    grads = (o, dq.transpose(1, 2).to(s["q"].dtype).contiguous(), own_heads(dk), own_heads(dv))
    if c["kind"] == "cross":
        return grads
    # Each query's pairs to their buckets, then the long sum over the queries in 64 bits.
    mine = (bucket[0][:, None, :] == torch.arange(c["buckets"], device=q.device)[:, None]).float()
    table = (mine @ ds.sum(0).permute(1, 2, 0).contiguous()).double().sum(0)
    return (*grads, table.float())


# --------------------------------------------------------------------- work --
def work(case):
    c = case
    if c["kind"] == "lora":
        used = min(c["adapters"], c["requests"])
        b = (c["n"] * c["k"] * WBYTES[c["weights"]] + 2 * c["rows"] * (c["k"] + c["n"]) +
             2 * used * c["rank"] * (c["k"] + c["n"]) + 4 * c["n"] + 4 * c["rows"])
        return {"bytes": b, "flops": 2.0 * c["rows"] * (c["n"] * c["k"] + c["rank"] * (c["k"] + c["n"]))}
    B, H, D, es = c["batch"], c["heads"], c["dim"], ES[c["dtype"]]
    kvh = c.get("kv_heads", H)
    keys = sum(_lengths(c)) if c["kind"] == "rel" or c["mask"] == "len" else \
        B * (c["kv"] - (c["kv"] // 4 if c["mask"] == "mask" else 0))
    rows, kv = B * c["q"] * H * D * es, keys * kvh * D * es
    pair = 2.0 * H * D * c["q"] * keys  # one product over the attended pairs
    table = 4 * c["buckets"] * H if c["kind"] == "rel" else 0
    if not c["train"]:
        return {"bytes": 2 * rows + 2 * kv + table, "flops": 2 * pair}
    whole = B * c["kv"] * kvh * D * es  # gradients are written for every key
    return {"bytes": 4 * rows + 2 * kv + 2 * whole + 2 * table, "flops": 7 * pair}


# -------------------------------------------------------------------- exact --
def exact(case, seed):
    """64 bits from the definition: each request's rows through its own merged
    product, attention by torch's softmax and its gradients by autograd."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "lora":
        x, w = s["x"].double(), _exact_weight(s)
        y = x @ w.t() + s["bias"].double()
        for a in sorted(set(s["row_adapter"].tolist()) - {-1}):
            rows = (s["row_adapter"] == a).nonzero()[:, 0]
            y[rows] += s["scale"][a].double() * ((x[rows] @ s["a"][a].double().t()) @ s["b"][a].double().t())
        return y
    leaves = [s[n].double().requires_grad_(c["train"]) for n in ("q", "k", "v")]
    if c["kind"] == "rel":
        leaves.append(s["table"].double().requires_grad_(c["train"]))
    q, k, v = leaves[:3]
    share = q.shape[2] // k.shape[2]
    with torch.set_grad_enabled(c["train"]):
        outs = []
        for b in range(q.shape[0]):
            if s["kv_len"] is not None:
                at = torch.arange(int(s["kv_len"][b]), device=q.device)
            elif s["kv_mask"] is not None:
                at = s["kv_mask"][b].nonzero()[:, 0]
            else:
                at = torch.arange(k.shape[1], device=q.device)
            kb = k[b][at].repeat_interleave(share, 1).permute(1, 2, 0).contiguous()  # [H, D, keys]
            vb = v[b][at].repeat_interleave(share, 1).permute(1, 0, 2).contiguous()
            x = torch.bmm(q[b].permute(1, 0, 2).contiguous(), kb) * s["scale"]
            if c["kind"] == "rel":
                first = int(s["q_pos"][b]) if s["q_pos"] is not None else 0
                x = x + leaves[3][_exact_buckets(c, first, at)].permute(2, 0, 1)
            outs.append(torch.bmm(torch.softmax(x, -1), vb).permute(1, 0, 2))
        o = torch.stack(outs)
        if not c["train"]:
            return o
        grads = torch.autograd.grad(o, leaves, s["do"].double())
    return (o.detach(), *grads)


def _exact_weight(s):
    if "w" in s:
        return s["w"].double()
    n, k = s["codes"].shape
    d = s["scales"].double().t().repeat_interleave(32, 1)
    return ((s["codes"].double() - 128) * d).to(torch.bfloat16).double().view(n, k)


def _exact_buckets(c, first, keys):
    """Buckets by whole numbers: distance n falls at least t buckets behind the
    near ones where n^far >= near^(far - t) distance^t."""
    side = c["buckets"] // 2 if c["two_sided"] else c["buckets"]
    near = side // 2
    far = side - near
    top = c["kv"] + c["q"] + c["distance"]
    of = []
    for n in range(top):
        t = n if n < near else near
        while n >= near and t < side - 1 and n ** far >= near ** (side - t - 1) * c["distance"] ** (t + 1 - near):
            t += 1
        of.append(t)
    of = torch.tensor(of, device=keys.device)
    off = keys[None, :] - (first + torch.arange(c["q"], device=keys.device))[:, None]
    if c["two_sided"]:
        return of[off.abs()] + side * (off > 0)
    return of[(-off).clamp_min(0)]
