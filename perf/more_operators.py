"""The operators that serve a causal text model as timed cases: rotary positions,
appending to a paged key/value cache, and attention over that cache.

listed() holds fixed cases, draw(rng) gives more of the same ranges;
prepare(case, seed) makes what a program has in hand before the call,
run(state) is one pass, work(case) its least bytes and operations,
exact(case, seed) the same outputs in 64 bits from the definition.

With `own` false run() computes the operators in their plain form (elementary
torch operations, rounded once at the end); with `own` true it calls the library.

Kinds of case:
  rotary  q and k [tokens, heads, dim] rotated by their positions, as pairs (2i, 2i + 1)
          or halves (i, i + rot / 2), the first rot dims of a head; train adds the
          rotation of the gradients
  append  the new tokens of every sequence to its pages, k (and q) rotated on the
          way; a page is held as e4m3 with a power-of-two scale per page and head, or as bf16
  attn    the new tokens' queries to everything their sequences hold
"""
import math
import os
import sys

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f32": torch.float32, "e4m3": torch.float8_e4m3fn}
ES = {"bf16": 2, "f32": 4, "e4m3": 1}
CONTEXT = 4096  # what the frequencies were made for, before they are scaled


# ---------------------------------------------------------------- the cases --
def listed():
    return [
        # The new tokens of eight requests, far into their contexts: the smallest call.
        {"name": "rotary_8tokens", "kind": "rotary", "tokens": 8, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "half": True, "dtype": "bf16", "factor": 1.0, "far": 4096, "train": False},
        # Two prompts of 4096 tokens with frequencies scaled for eight times the context.
        {"name": "rotary_8192", "kind": "rotary", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rot": 128,
         "half": True, "dtype": "bf16", "factor": 8.0, "far": 32768, "train": False},
        # A training step in 32 bits, interleaved, with a part of an odd head rotated.
        {"name": "rotary_train_f32", "kind": "rotary", "tokens": 1501, "heads": 20, "kv_heads": 20, "dim": 80, "rot": 32,
         "half": False, "dtype": "f32", "factor": 1.0, "far": 2048, "train": True},
        # One token of each of 32 requests into an 8-bit cache.
        {"name": "append_32tokens", "kind": "append", "seqs": 32, "ones": 32, "new": 1, "past": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "e4m3", "half": True},
        # Five prompts of ragged lengths, some behind a cached prefix, into an 8-bit cache.
        {"name": "append_prompts", "kind": "append", "seqs": 5, "ones": 0, "new": 2500, "past": 77, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "e4m3", "half": True},
        # Prompts of an odd width into small bf16 pages, interleaved rotation.
        {"name": "append_bf16", "kind": "append", "seqs": 7, "ones": 2, "new": 700, "past": 333, "heads": 12, "kv_heads": 12,
         "dim": 80, "page": 16, "cache": "bf16", "half": False},
        # One token of one request with a short past: latency.
        {"name": "attn_1token", "kind": "attn", "seqs": 1, "ones": 1, "new": 1, "past": 1000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "e4m3"},
        # One token of each of 32 requests with long pasts of their own lengths.
        {"name": "attn_32tokens", "kind": "attn", "seqs": 32, "ones": 32, "new": 1, "past": 8000, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "e4m3"},
        # One token of 24 requests over a bf16 cache without shared heads.
        {"name": "attn_24tokens_bf16", "kind": "attn", "seqs": 24, "ones": 24, "new": 1, "past": 2300, "heads": 16,
         "kv_heads": 16, "dim": 64, "page": 32, "cache": "bf16"},
        # Two prompts from their first token on: the most operations.
        {"name": "attn_prompts", "kind": "attn", "seqs": 2, "ones": 0, "new": 4096, "past": 0, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 64, "cache": "e4m3"},
        # 300 more tokens of one request behind a long document.
        {"name": "attn_chunk", "kind": "attn", "seqs": 1, "ones": 0, "new": 300, "past": 16000, "heads": 24, "kv_heads": 8,
         "dim": 128, "page": 128, "cache": "e4m3"},
        # A step that mixes fifteen single tokens with two pieces of prompts.
        {"name": "attn_mixed", "kind": "attn", "seqs": 17, "ones": 15, "new": 512, "past": 3500, "heads": 32, "kv_heads": 8,
         "dim": 128, "page": 16, "cache": "bf16"},
    ]


def _log(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 0.49)))))))


def draw(rng):
    kind = rng.choice(["rotary", "append", "attn", "attn"])
    dim = rng.choice([64, 128, 128, 16 * rng.randint(2, 8)])
    shared, kv_heads = rng.choice([(1, 16), (1, 12), (2, 8), (3, 8), (4, 8), (4, 4), (8, 4), (5, 2)])
    c = {"kind": kind, "heads": shared * kv_heads, "kv_heads": kv_heads, "dim": dim}
    if kind == "rotary":
        train = rng.random() < 0.4
        return {**c, "tokens": _log(rng, 1, 4000), "rot": rng.choice([dim, dim, dim // 2, 2 * rng.randint(1, dim // 2)]),
                "half": rng.random() < 0.5, "dtype": rng.choice(["bf16", "bf16", "f32"]), "factor": rng.choice([1.0, 4.0, 8.0]),
                "far": _log(rng, 2048, 200000), "train": train}
    c["page"] = rng.choice([16, 32, 64, 64, 128])
    c["cache"] = rng.choice(["e4m3", "e4m3", "bf16"])
    if kind == "append":
        c["half"] = rng.random() < 0.7
    what = rng.choice(["tokens", "prompts", "mixed"])
    if what == "tokens":
        c["seqs"] = c["ones"] = _log(rng, 1, 32)
        c["new"], c["past"] = 1, _log(rng, 1, 7000)
    else:
        c["seqs"] = rng.randint(1, 4) if what == "prompts" else rng.randint(2, 16)
        c["ones"] = 0 if what == "prompts" else rng.randint(1, c["seqs"] - 1)
        c["new"] = _log(rng, 2, 4000 // (c["seqs"] - c["ones"]))
        c["past"] = rng.choice([0, _log(rng, 1, 4000)])
    return c


def _news(c):
    """New tokens of each sequence: prompts from all down to a quarter of `new`, then `ones` single tokens."""
    n = c["seqs"] - c["ones"]
    return [max(1, c["new"] - (b * 3 * c["new"]) // (4 * n)) for b in range(n)] + [1] * c["ones"]


def _pasts(c):
    """What each sequence holds before: from all down to a quarter of `past`."""
    return [c["past"] - (b * 3 * c["past"]) // (4 * c["seqs"]) for b in range(c["seqs"])]


# ------------------------------------------------------------- prepare, run --
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _randn(g, shape, dtype, std=1.0):
    return (torch.randn(shape, device="cuda", generator=g) * std).to(dtype)


def _freqs(rot, factor):
    """Radians per position of each pair; with a factor those that turn rarely within
    the original context are slowed by it, those that turn often are kept."""
    f = 10000.0 ** (-torch.arange(0, rot, 2, device="cuda", dtype=torch.float64) / rot)
    turns = CONTEXT * f / (2 * math.pi)
    keep = ((turns - 1.0) / 31.0).clamp(0.0, 1.0)
    return (f * (keep + (1.0 - keep) / factor)).float()


def prepare(case, seed):
    c = case
    g = _gen(seed)
    s = {"case": c}
    H, KH, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rotary":
        T, dt = c["tokens"], DTYPES[c["dtype"]]
        s["freq"] = _freqs(c["rot"], c["factor"])
        s["mul"] = 0.1 * math.log(c["factor"]) + 1.0
        s["q"], s["k"] = _randn(g, (T, H, D), dt), _randn(g, (T, KH, D), dt)
        first = torch.randint(0, max(1, c["far"] - T), (1,), device="cuda", generator=g)
        s["pos"] = (first + torch.arange(T, device="cuda")).to(torch.int32)
        if c["train"]:
            s["dq"], s["dk"] = _randn(g, (T, H, D), dt), _randn(g, (T, KH, D), dt)
        return s
    news, pasts, P = _news(c), _pasts(c), c["page"]
    T, B = sum(news), c["seqs"]
    need = [-(-(n + p) // P) for n, p in zip(news, pasts)]
    pages, width = sum(need) + 3, max(need) + 2
    # Every sequence's pages lie anywhere in the pool; the rest of the table is unused.
    order = torch.randperm(pages, device="cuda", generator=g).to(torch.int32)
    at = [sum(need[:b]) + j if j < n else -1 for b, n in enumerate(need) for j in range(width)]
    at = torch.tensor(at, device="cuda").view(B, width)
    s["table"] = torch.where(at >= 0, order[at.clamp_min(0)], -1).to(torch.int32)
    s["seq_start"] = torch.tensor([sum(news[:b]) for b in range(B + 1)], device="cuda", dtype=torch.int32)
    s["past"] = torch.tensor(pasts, device="cuda", dtype=torch.int32)
    s["widest"] = max(news)
    # The pool as earlier steps left it: values of the pages' own sizes, keys' dims of unlike sizes.
    dt = DTYPES[c["cache"]]
    gain = torch.exp2(torch.rand((pages, KH, 1, 1), device="cuda", generator=g) * 2 - 1)
    k = torch.randn((pages, KH, P, D), device="cuda", generator=g) * gain * (0.5 + torch.rand(D, device="cuda", generator=g))
    v = torch.randn((pages, KH, D, P), device="cuda", generator=g) * gain
    s["k_scale"] = s["v_scale"] = None
    if c["cache"] == "e4m3":
        # 2^(scale - 127) is a page's power of two
        s["k_scale"], s["v_scale"] = (_scale_of(x.abs().amax((2, 3))) for x in (k, v))
        k, v = (x * torch.exp2(127.0 - n.float())[..., None, None] for x, n in ((k, s["k_scale"]), (v, s["v_scale"])))
    s["k_pages"], s["v_pages"] = k.to(dt), v.to(dt)
    s["q"] = _randn(g, (T, H, D), torch.bfloat16)
    if c["kind"] == "append":
        s["freq"] = _freqs(D, 1.0)
        s["k"], s["v"] = _randn(g, (T, KH, D), torch.bfloat16, 1.5), _randn(g, (T, KH, D), torch.bfloat16)
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
    return {"rotary": _plain_rotary, "append": _plain_append, "attn": _plain_attn}[state["case"]["kind"]](state)


def _run_own(s):
    dh = _library()
    c = s["case"]
    if c["kind"] == "rotary":
        rot = dh.Rotary(s["freq"], half=c["half"], attn_factor=s["mul"])
        out = dh.rotary(s["q"], s["k"], s["pos"], rot)
        return (*out, *dh.rotary_bwd(s["dq"], s["dk"], s["pos"], rot)) if c["train"] else out
    cache = dh.KVCache(s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"])
    if c["kind"] == "attn":
        return dh.cache_attn(s["q"], cache, s["table"], s["seq_start"], s["past"])
    rot = dh.Rotary(s["freq"], half=c["half"])
    q = dh.cache_append(cache, s["k"], s["v"], s["table"], s["seq_start"], s["past"], rot=rot, q=s["q"])
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_rotate(x, pos, freq, half, mul=1.0, sign=1.0):
    """x [T, H, D], in 32 bits; the angles in 64."""
    n = 2 * freq.numel()
    a = (pos.double()[:, None] * freq.double())[:, None, :]
    co, si = (torch.cos(a) * mul).float(), (torch.sin(a) * (mul * sign)).float()
    x = x.float()
    u = x[..., :n]
    if half:
        a, b = u[..., :n // 2], u[..., n // 2:]
        u = torch.cat((a * co - b * si, b * co + a * si), -1)
    else:
        a, b = u[..., 0::2], u[..., 1::2]
        u = torch.stack((a * co - b * si, b * co + a * si), -1).flatten(-2)
    return torch.cat((u, x[..., n:]), -1)


def _plain_rotary(s):
    c = s["case"]
    todo = [(s["q"], 1.0), (s["k"], 1.0)] + ([(s["dq"], -1.0), (s["dk"], -1.0)] if c["train"] else [])
    return tuple(_plain_rotate(x, s["pos"], s["freq"], c["half"], s["mul"], sign).to(x.dtype) for x, sign in todo)


def _rows(s):
    """Each new token's sequence and place in it."""
    row = torch.arange(s["q"].shape[0], device="cuda")
    b = torch.searchsorted(s["seq_start"], row, right=True) - 1
    return b, s["past"][b] + row - s["seq_start"][b]


def _scale_of(most):
    """The least power of two (plus 127, 1 at least) by which e4m3's 448 reaches `most`:
    448 2^e >= m 2^x (m in [0.5, 1)) from e = x - 9 on where m <= 0.875."""
    m, x = torch.frexp(most)
    return torch.where(most > 0, (x - 9 + (m > 0.875) + 127).clamp(1, 254), 1).to(torch.uint8)


def _plain_append(s):
    c = s["case"]
    b, at = _rows(s)
    P, KH = c["page"], c["kv_heads"]
    page, off = s["table"][b, at // P].long(), at % P
    q = _plain_rotate(s["q"], at, s["freq"], c["half"]).to(torch.bfloat16)
    k, v = _plain_rotate(s["k"], at, s["freq"], c["half"]), s["v"].float()
    # The pages that tokens are added to in their middle.
    edge = s["table"].gather(1, (s["past"] // P)[:, None].long())[:, 0].clamp_min(0).long()
    held = (s["past"] % P)[:, None, None, None]
    old = torch.arange(P, device="cuda") < held[..., 0]  # [B, 1, P]
    for name, x in (("k", k), ("v", v)):
        pages, scale = s[name + "_pages"], s[name + "_scale"]
        if scale is not None:
            most = torch.zeros((pages.shape[0], KH), device="cuda")
            most.scatter_reduce_(0, page[:, None].expand(-1, KH), x.abs().amax(-1), "amax")
            new = _scale_of(most)
            new[edge] = torch.where(held[..., 0, 0] > 0, torch.maximum(new[edge], scale[edge]), new[edge])
            keep = old[..., None] if name == "k" else old[:, :, None]  # [B, 1, P, 1] or [B, 1, 1, P]
            shift = torch.exp2(scale[edge].float() - new[edge].float())[..., None, None]
            again = (pages[edge].float() * shift).to(pages.dtype)
            pages[edge] = torch.where(keep, again.float(), pages[edge].float()).to(pages.dtype)
            scale[page] = new[page]
            x = x * torch.exp2(127.0 - new[page].float())[..., None]
        if name == "k":
            pages[page, :, off] = x.to(pages.dtype)
        else:
            pages[page, :, :, off] = x.to(pages.dtype)
    return q, s["k_pages"], s["v_pages"], s["k_scale"], s["v_scale"]


def _plain_attn(s):
    c = s["case"]
    B, P, H, KH, D = c["seqs"], c["page"], c["heads"], c["kv_heads"], c["dim"]
    G, W = H // KH, s["table"].shape[1]
    table = s["table"].clamp_min(0).long()
    k, v = s["k_pages"][table].float(), s["v_pages"][table].float()  # [B, W, KH, ...]
    if s["k_scale"] is not None:
        k = k * torch.exp2(s["k_scale"][table].float() - 127.0)[..., None, None]
        v = v * torch.exp2(s["v_scale"][table].float() - 127.0)[..., None, None]
    new = s["seq_start"][1:] - s["seq_start"][:-1]
    held = (s["past"] + new)[:, None, None, None]
    key = torch.arange(W * P, device="cuda")
    k = k.transpose(1, 2).reshape(B, KH, W * P, D)
    v = v.permute(0, 2, 1, 4, 3).reshape(B, KH, W * P, D)
    v = torch.where((key < held[..., 0])[..., None], v, 0.0)
    i = torch.arange(s["widest"], device="cuda")
    row = (s["seq_start"][:-1, None] + i).clamp_max(s["q"].shape[0] - 1).long()
    q = s["q"][row].float().view(B, -1, KH, G, D).permute(0, 2, 3, 1, 4).reshape(B, KH, -1, D)
    x = (q @ k.transpose(2, 3).contiguous()) * D ** -0.5  # rows: heads of a group, then tokens
    x = x.view(B, KH, G, -1, W * P)
    x = x.masked_fill(key > (s["past"][:, None] + i)[:, None, None, :, None], -math.inf)
    x = torch.exp(x - x.amax(-1, keepdim=True))
    x = x / x.sum(-1, keepdim=True)
    o = (x.view(B, KH, -1, W * P) @ v).view(B, KH, G, -1, D).permute(0, 3, 1, 2, 4).reshape(B, -1, H, D)
    b, at = _rows(s)
    return o[b, (at - s["past"][b]).long()].to(torch.bfloat16)


# --------------------------------------------------------------------- work --
def work(case):
    c = case
    H, KH, D = c["heads"], c["kv_heads"], c["dim"]
    if c["kind"] == "rotary":
        n, times = c["tokens"] * (H + KH), 2 if c["train"] else 1
        return {"bytes": times * (2.0 * n * D * ES[c["dtype"]] + 4 * c["tokens"]) + 2 * c["rot"], "flops": times * 3.0 * n * c["rot"]}
    news, pasts, es = _news(c), _pasts(c), ES[c["cache"]]
    T = sum(news)
    pages = sum((p + n - 1) // c["page"] - p // c["page"] + 1 for n, p in zip(news, pasts))
    if c["kind"] == "append":
        scales = 2 * pages * KH if c["cache"] == "e4m3" else 0
        return {"bytes": 4.0 * T * H * D + 2 * T * KH * D * (2 + es) + scales + 4 * pages + 8 * c["seqs"] + 2 * D,
                "flops": 3.0 * T * (H + KH) * D + 4.0 * T * KH * D}
    keys = sum(n + p for n, p in zip(news, pasts))
    pairs = sum(n * p + n * (n + 1) // 2 for n, p in zip(news, pasts))
    return {"bytes": 2.0 * keys * KH * D * es + 4 * T * H * D + 4 * keys // c["page"] + 8 * c["seqs"], "flops": 4.0 * H * D * pairs}


# -------------------------------------------------------------------- exact --
def exact(case, seed):
    """64 bits from the definition, a sequence (and a page) at a time; rotations as
    complex products, e4m3 by its steps."""
    c, s = case, prepare(case, seed)
    if c["kind"] == "rotary":
        out = [_exact_rotate(s[n], s["pos"], s["freq"], c["half"], s["mul"]) for n in ("q", "k")]
        return tuple(out + ([_exact_rotate(s[n], s["pos"], s["freq"], c["half"], s["mul"], True) for n in ("dq", "dk")] if c["train"] else []))
    start, pasts = s["seq_start"].tolist(), s["past"].tolist()
    if c["kind"] == "append":
        return _exact_append(c, s, start, pasts)
    P, KH, G, D = c["page"], c["kv_heads"], c["heads"] // c["kv_heads"], c["dim"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b in range(c["seqs"]):
        n, held = start[b + 1] - start[b], pasts[b] + start[b + 1] - start[b]
        mine = s["table"][b, :-(-held // P)].long()
        k, v = s["k_pages"][mine].double(), s["v_pages"][mine].double()
        if s["k_scale"] is not None:
            k = torch.ldexp(k, (s["k_scale"][mine].int() - 127)[..., None, None])
            v = torch.ldexp(v, (s["v_scale"][mine].int() - 127)[..., None, None])
        seen = torch.ones((n, held), dtype=torch.bool, device="cuda").tril(pasts[b])
        for h in range(KH):
            kh = k[:, h].reshape(-1, D)[:held].t().contiguous()
            vh = v[:, h].transpose(1, 2).reshape(-1, D)[:held].contiguous()
            for g in range(G):
                x = (s["q"][start[b]:start[b + 1], h * G + g].double() @ kh) / math.sqrt(D)
                out[start[b]:start[b + 1], h * G + g] = torch.softmax(torch.where(seen, x, -math.inf), -1) @ vh
    return out


def _exact_rotate(x, pos, freq, half, mul=1.0, back=False):
    n = 2 * freq.numel()
    x = x.double()
    turn = torch.polar(torch.full_like(pos[:, None] * freq.double(), mul), pos.double()[:, None] * freq.double() * (-1 if back else 1))
    pairs = torch.stack((x[..., :n // 2], x[..., n // 2:n]), -1) if half else x[..., :n].unflatten(-1, (-1, 2))
    y = torch.view_as_real(torch.view_as_complex(pairs.contiguous()) * turn[:, None])
    y = torch.cat((y[..., 0], y[..., 1]), -1) if half else y.flatten(-2)
    return torch.cat((y, x[..., n:]), -1)


def _exact_e4m3(x):
    """The nearest value of e4m3 (ties to even): steps of an eighth of the power of two below, 2^-9 at least."""
    step = torch.exp2(torch.floor(torch.log2(x.abs().clamp_min(2.0 ** -6))) - 3)
    return torch.round(x / step) * step


def _exact_append(c, s, start, pasts):
    P = c["page"]
    place = torch.cat([torch.arange(p, p + n, device="cuda") for p, n in zip(pasts, _news(c))])
    q = _exact_rotate(s["q"], place, s["freq"], c["half"])
    new = {"k": _exact_rotate(s["k"], place, s["freq"], c["half"]), "v": s["v"].double()}
    got, scales = {}, {}
    for name, x in new.items():
        pages = s[name + "_pages"].double()
        pages = pages if name == "k" else pages.transpose(2, 3).contiguous()
        scale = s[name + "_scale"]
        for b in range(c["seqs"]):
            at, end = pasts[b], pasts[b] + start[b + 1] - start[b]
            while at < end:
                p, first = int(s["table"][b, at // P]), at % P
                n = min(P - first, end - at)
                rows = x[start[b] + at - pasts[b]:][:n].transpose(0, 1)  # [KH, n, D]
                if scale is None:
                    pages[p, :, first:first + n] = rows
                else:
                    most = rows.abs().amax((1, 2))
                    power = torch.ceil(torch.log2(most / 448)).clamp_min(-126)
                    if first:
                        power = torch.maximum(power, scale[p].double() - 127)
                        back = torch.exp2(scale[p].double() - 127 - power)[:, None, None]
                        pages[p, :, :first] = _exact_e4m3(pages[p, :, :first] * back)
                    pages[p, :, first:first + n] = _exact_e4m3(rows * torch.exp2(-power)[:, None, None])
                    scale[p] = (power + 127).to(torch.uint8)
                at += n
        got[name] = pages if name == "k" else pages.transpose(2, 3).contiguous()
        scales[name] = None
    return q, got["k"], got["v"], scales["k"], scales["v"]
