"""Operators of a decoder layer that is served with activations in 8 bits and a paged cache in 4 bits: what is timed and compared.

  norm     residual sum, RMS norm and its rows in 8 bits with a scale per token
  product  product in 8-bit integers with scales per token and per output channel
  append   rotation of queries and keys, keys and values into the paged 4-bit cache, and the cached rows read back as values
  attend   attention over the paged 4-bit cache: single tokens of many sequences, long contexts, prompts

A page holds, for each kv head, page x head_dim / 2 bytes of keys, the same of values, page f32 key scales and page f32 value scales; channel 2i of a
row is in the low four bits of its byte i.  A value is scale * (n - 8).
"""
import math

import torch

own = False

HEADS = {"8b": (32, 8, 128), "70b": (64, 8, 128), "1b": (32, 4, 64), "0.5b": (14, 2, 64)}  # query heads, kv heads, head size of the shapes in presets.py
TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = torch.tensor(1e-5).item()
TINY = 2.0**-119  # rows whose largest magnitude is below this are zeros


def listed():
    return [
        # one decoded token of an 8B model: latency
        dict(name="norm_token", op="norm", rows=1, hidden=4096, type="bf16", residual=True),
        # a prompt chunk of an 8B model
        dict(name="norm_prompt", op="norm", rows=2048, hidden=4096, type="bf16", residual=True),
        # f32 activations as the GGUF contexts have them, a 0.5B model's width, an odd number of rows, the first norm (no sum)
        dict(name="norm_f32", op="norm", rows=333, hidden=896, type="f32", residual=False),
        # four sequences' step through an 8B model's up projection: the weights' bytes
        dict(name="product_step", op="product", rows=4, k=4096, n=14336, type="f16", bias=False),
        # a prompt chunk through the same: the tensor pipe
        dict(name="product_prompt", op="product", rows=2048, k=4096, n=14336, type="bf16", bias=False),
        # ragged sizes, bias, f32 results
        dict(name="product_ragged", op="product", rows=61, k=1999, n=1537, type="f32", bias=True),
        # a step of 32 sequences of an 8B model, neighbouring channels paired
        dict(name="append_step", op="append", heads="8b", tokens=32, page=16, rot=128, neox=False, type="bf16", skip=0),
        # prompts of a 1.1B model, a part of them padding that is not cached
        dict(name="append_prompt", op="append", heads="1b", tokens=4001, page=64, rot=64, neox=True, type="f16", skip=100),
        # one short chat of a 0.5B model in f32: latency
        dict(name="attend_chat", op="attend", heads="0.5b", seqs=1, q=1, longest=333, page=32, window=0, type="f32"),
        # a server's step: 32 sequences of all lengths, one of them empty
        dict(name="attend_step", op="attend", heads="8b", seqs=32, q=1, longest=8000, page=16, window=0, type="bf16"),
        # one long document with a 70B model's heads
        dict(name="attend_document", op="attend", heads="70b", seqs=1, q=1, longest=131072, page=64, window=0, type="bf16"),
        # the second chunk of a prompt: 2048 tokens behind 2048 cached ones
        dict(name="attend_prompt", op="attend", heads="8b", seqs=1, q=2048, longest=4096, page=64, window=0, type="bf16"),
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op, type_ = rng.choice(["norm", "product", "append", "attend", "attend"]), rng.choice(sorted(TYPES))
    if op == "norm":
        hidden = rng.choice([size(32, 16384), 64 * size(1, 256)])
        return dict(op=op, rows=size(1, min(4096, 2**24 // hidden)), hidden=hidden, type=type_, residual=rng.random() < 0.7)
    if op == "product":
        k, n = rng.choice([size(16, 16384), 64 * size(1, 256)]), rng.choice([size(1, 16384), 64 * size(1, 256)])
        return dict(op=op, rows=size(1, min(4096, 2**36 // (k * n))), k=k, n=n, type=type_, bias=rng.random() < 0.5)
    heads = rng.choice(sorted(HEADS))
    if op == "append":
        tokens, hd = size(1, 6000), HEADS[heads][2]
        return dict(op=op, heads=heads, tokens=tokens, page=rng.choice([16, 32, 64, 128]), rot=rng.choice([hd, hd, hd // 2]), neox=rng.random() < 0.5, type=type_,
                    skip=rng.choice([0, tokens // 3]))
    q = rng.choice([1, 1, size(2, 16), size(17, 700)])
    longest = size(max(16, q), 40000 if q == 1 else max(64, min(12000, 2**27 // (q * HEADS[heads][0]))))
    fits = 2**28 // (longest * max(q * HEADS[heads][0], 2 * HEADS[heads][1] * HEADS[heads][2]))  # scores and decoded rows of the plain form
    return dict(op=op, heads=heads, seqs=size(1, max(1, min(64, fits))), q=min(q, longest), longest=longest, page=rng.choice([16, 32, 64, 128]),
                window=rng.choice([0, 0, 0, size(16, 4096)]), type=type_)


# ------------------------------------------------------------------------------------------------------------------ inputs
def padded(t):
    """The same rows at a distance of whole 16 bytes (t: int8)."""
    rows, k = t.shape
    buf = torch.zeros(rows, (k + 15) // 16 * 16, dtype=t.dtype, device=t.device)
    buf[:, :k] = t
    return buf[:, :k]


def quantised(x):
    """Rows of f32 as (nibbles 0..15, scale): the value of the largest magnitude becomes -8."""
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    top = torch.where(hi >= -lo, hi, lo)
    scale = torch.where(top.abs() >= TINY, top / -8, 0.0)
    scale = torch.where(torch.isfinite(top), scale, math.nan)
    inverse = torch.where(scale == 0, 0.0, torch.ones_like(scale) / scale)
    return torch.nan_to_num(torch.round(x * inverse) + 8, nan=8.0).clamp(0, 15), scale


def sections(pages, page, hd):
    """Views into the pages: key bytes, value bytes [pages, kv heads, page, hd / 2], key scales, value scales [pages, kv heads, page]."""
    p, nkv, _ = pages.shape
    at = [0, page * hd // 2, page * hd, page * hd + 4 * page, page * hd + 8 * page]
    data = [pages[:, :, a:b].view(p, nkv, page, hd // 2) for a, b in zip(at[:2], at[1:3])]
    return data + [pages[:, :, a:b].view(torch.float32) for a, b in zip(at[2:4], at[3:])]


def packed(n):
    n = n.to(torch.uint8)
    return n[..., 0::2] | (n[..., 1::2] << 4)


def unpacked(b):
    return torch.stack([b & 15, b >> 4], -1).flatten(-2)


def filled_pages(n_pages, nkv, page, hd, rng):
    pages = torch.empty(n_pages, nkv, page * (hd + 8), dtype=torch.uint8, device="cuda")
    parts = sections(pages, page, hd)
    for i in (0, 1):
        n, d = quantised(torch.randn(n_pages, nkv, page, hd, device="cuda", generator=rng))
        parts[i].copy_(packed(n))
        parts[2 + i].copy_(d[..., 0])
    return pages


def prepare(case, seed):
    rng = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=rng)  # noqa: E731
    t = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "norm":
        # a residual stream with a few channels that stand out
        big = 1 + 20 * (torch.rand(case["hidden"], device="cuda", generator=rng) < 0.01).float()
        s.update(x=normal(case["rows"], case["hidden"]).to(t), w=1 + 0.1 * normal(case["hidden"]))
        s["r"] = (normal(case["rows"], case["hidden"]) * big).to(t) if case["residual"] else None
    elif case["op"] == "product":
        q = torch.round(normal(case["rows"], case["k"]) * 32).clamp(-127, 127).to(torch.int8)
        w = torch.round(normal(case["n"], case["k"]) * 32).clamp(-127, 127).to(torch.int8)
        s.update(q=padded(q), w=padded(w), s=0.01 + 0.02 * torch.rand(case["rows"], device="cuda", generator=rng),
                 ws=0.0005 + 0.001 * torch.rand(case["n"], device="cuda", generator=rng), b=normal(case["n"]) if case["bias"] else None)
    elif case["op"] == "append":
        nh, nkv, hd = HEADS[case["heads"]]
        n, page = case["tokens"], case["page"]
        qkv = normal(n, (nh + 2 * nkv) * hd).to(t)  # the projection's rows, as one product leaves them
        q, k, v = qkv[:, : nh * hd], qkv[:, nh * hd : (nh + nkv) * hd], qkv[:, (nh + nkv) * hd :]
        s.update(q=q.unflatten(1, (nh, hd)), k=k.unflatten(1, (nkv, hd)), v=v.unflatten(1, (nkv, hd)))
        places = 16384
        angle = torch.arange(places, dtype=torch.float64)[:, None] * 10000.0 ** (-torch.arange(0, case["rot"], 2, dtype=torch.float64) / case["rot"])
        s["table"] = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
        s["positions"] = torch.randint(0, places, (n,), generator=host, dtype=torch.int32).cuda()
        n_pages = n // page + 8
        slots = 1 + torch.randperm(n_pages * page - 1, generator=host)[:n]  # slot 0 stays unused
        slots[torch.randperm(n, generator=host)[: case["skip"]]] = -1
        s.update(slots=slots.cuda(), pages=filled_pages(n_pages, nkv, page, hd, rng))
    else:
        nh, nkv, hd = HEADS[case["heads"]]
        S, page, longest = case["seqs"], case["page"], case["longest"]
        lens = (torch.rand(S, generator=host) ** 2 * longest).long().clamp(min=min(case["q"], longest))
        if S > 1:
            lens[1] = 0  # a slot without a sequence: its rows are zeros
        lens[0] = longest
        q_lens = torch.full((S,), case["q"])
        if case["q"] > 1:
            q_lens[1:] = torch.randint(1, case["q"] + 1, (S - 1,), generator=host)
        need = (lens + page - 1) // page
        order = torch.randperm(int(need.sum()) + 3, generator=host)
        table = torch.zeros(S, (longest + page - 1) // page, dtype=torch.int32)
        used = torch.arange(table.shape[1])[None] < need[:, None]
        table[used] = order[: int(need.sum())].int()
        starts = torch.cat([torch.zeros(1, dtype=torch.long), q_lens.cumsum(0)]).int()
        s.update(q_tokens=(2 * normal(int(starts[-1]), nh, hd)).to(t), pages=filled_pages(len(order), nkv, page, hd, rng), table=table.cuda(),
                 lens=lens.int().cuda(), starts=starts.cuda() if case["q"] > 1 else None, scale=hd**-0.5)
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def plain_norm(s):
    t = s["x"].dtype
    x = s["x"].float()
    r = x if s["r"] is None else (x + s["r"].float()).to(t).float()
    mean = r.double().square().mean(-1, keepdim=True)
    y = r * (1 / torch.sqrt(mean + EPS)).float() * s["w"]
    top = y.abs().amax(-1, keepdim=True)
    live = top >= TINY
    q = torch.where(live, torch.round(y * torch.where(live, torch.full_like(top, 127) / top, 0.0)), 0.0)
    scale = torch.where(live, top / torch.full_like(top, 127), 0.0)
    return [(q * scale).bfloat16(), scale[:, 0]] + ([] if s["r"] is None else [r.to(t)])


def plain_product(s):
    y = (s["q"].float() @ s["w"].float().T) * s["s"][:, None] * s["ws"]
    return (y if s["b"] is None else y + s["b"]).to(TYPES[s["type"]])


def rotated(x, cos, sin, rot, neox):
    a, b = (x[..., : rot // 2], x[..., rot // 2 : rot]) if neox else (x[..., 0:rot:2], x[..., 1:rot:2])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.cat([a, b], -1) if neox else torch.stack([a, b], -1).flatten(-2)
    return torch.cat([turned, x[..., rot:]], -1)


def plain_append(s):
    t, rot, page, hd = s["q"].dtype, s["rot"], s["page"], s["q"].shape[-1]
    cs = s["table"][s["positions"]][:, None]
    cos, sin = cs[..., : rot // 2], cs[..., rot // 2 :]
    q, k = (rotated(s[n].float(), cos, sin, rot, s["neox"]) for n in ("q", "k"))
    live, slot = s["slots"] >= 0, s["slots"].clamp(min=0)
    at = (slot // page, slice(None), slot % page)
    parts = sections(s["pages"], page, hd)
    out = [q.to(t)]
    for i, x in ((0, k), (1, s["v"].float())):
        n, d = quantised(x)
        # (a token that is not cached writes what is there, to slot 0, which holds no token)
        parts[i][at] = torch.where(live[:, None, None], packed(n), parts[i][at])
        parts[2 + i][at] = torch.where(live[:, None], d[..., 0], parts[2 + i][at])
        value = (unpacked(parts[i][at]).float() - 8) * parts[2 + i][at][..., None]
        out.append(torch.where(live[:, None, None], value, 0.0).bfloat16())
    return out


def attention(s, real):
    """Padded to the longest sequence; `real` is the type that it is computed in."""
    q, page, window = s["q_tokens"], s["page"], s["window"]
    tokens, nh, hd = q.shape
    S, width = s["table"].shape
    nkv = s["pages"].shape[1]
    dev = q.device
    starts = torch.arange(S + 1, device=dev) if s["starts"] is None else s["starts"].long()
    rows = torch.arange(tokens, device=dev)
    seq = torch.searchsorted(starts, rows, right=True) - 1
    nth = rows - starts[seq]
    most = s["q"]
    take = (starts[:-1, None] + torch.arange(most, device=dev)).clamp(max=tokens - 1)
    qp = q.to(real)[take].view(S, most, nkv, nh // nkv, hd)
    L = width * page
    kb, vb, ks, vs = (p[s["table"].long()].transpose(2, 3).flatten(1, 2) for p in sections(s["pages"], page, hd))
    k, v = ((unpacked(b).to(real) - 8) * d.to(real)[..., None] for b, d in ((kb, ks), (vb, vs)))
    z = torch.einsum("sqkgd,slkd->skgql", qp, k) * s["scale"]
    lens = s["lens"].long()
    here = (lens[:, None] - (starts[1:] - starts[:-1])[:, None] + torch.arange(most, device=dev))[:, :, None]
    j = torch.arange(L, device=dev)
    seen = (j <= here) & (j < lens[:, None, None])
    if window:
        seen &= here - j < window
    z = z.masked_fill_(~seen[:, None, None], -math.inf)
    top = z.amax(-1, keepdim=True)
    z = z.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    total = z.sum(-1, keepdim=True)
    v = torch.where(seen.any(1)[:, :, None, None], v, 0.0)
    o = torch.einsum("skgql,slkd->sqkgd", z.div_(torch.where(total == 0, 1.0, total)), v)
    return o.reshape(S, most, nh, hd)[seq, nth]


def run(s):
    t = TYPES[s["type"]]
    if not own:
        if s["op"] == "norm":
            return plain_norm(s)
        if s["op"] == "product":
            return plain_product(s)
        if s["op"] == "append":
            return plain_append(s)
        return attention(s, torch.float32).to(t)
    from llama_gguf_b200 import device_ops as D

    if s["op"] == "norm":
        q, scale, r = D.add_rms_norm_q8(s["x"], s["w"], EPS, residual=s["r"])
        value = torch.mul(q, scale[:, None], out=torch.empty(q.shape, dtype=torch.bfloat16, device=q.device))
        return [value, scale] + ([] if r is None else [r])
    if s["op"] == "product":
        return D.mat_mat_i8(s["q"], s["s"], s["w"], s["ws"], bias=s["b"], dtype=t)
    if s["op"] == "append":
        q = D.rope_append_q4(s["q"], s["k"], s["v"], s["table"], s["positions"], s["pages"], s["slots"], use_neox=s["neox"])
        return [q, *D.read_q4(s["pages"], s["slots"], s["q"].shape[-1], torch.bfloat16)]
    return D.attention_paged_q4(s["q_tokens"], s["pages"], s["table"], s["lens"], s["scale"], q_starts=s["starts"], max_q=s["q"], window=s["window"])


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "norm":
        n = case["rows"] * case["hidden"]
        return {"bytes": n * (size * (3 if case["residual"] else 1) + 2) + 4 * (case["rows"] + case["hidden"]), "flops": 8 * n}
    if case["op"] == "product":
        t, k, n = case["rows"], case["k"], case["n"]
        return {"bytes": t * k + n * k + 4 * (t + n) + t * n * size + (4 * n if case["bias"] else 0), "flops": 2 * t * k * n}
    nh, nkv, hd = HEADS[case["heads"]]
    if case["op"] == "append":
        t, live = case["tokens"], case["tokens"] - case["skip"]
        # (the rows read back: nibbles and scales once more, and their values)
        return {"bytes": t * ((2 * nh + 2 * nkv) * hd * size + 4 * case["rot"] + 12) + 2 * live * nkv * (hd + 8) + t * nkv * 2 * hd * 2, "flops": t * hd * (3 * nh + 10 * nkv)}
    S, q, longest, window = case["seqs"], case["q"], case["longest"], case["window"]
    # lengths are longest, 0, then a third of longest on average; query tokens q, then half of it
    reach = lambda n, m: min(n, window + m) if window else n  # noqa: E731
    some, m = max(0, S - 2), (q + 1) // 2 if q > 1 else 1
    keys = reach(longest, q) + some * reach(max(q, longest // 3), m)
    rows = q + (S - 1) * m
    pairs = q * (min(longest, window) if window else longest - (q - 1) / 2) + some * m * (min(max(q, longest // 3), window) if window else max(m, longest // 3 - m / 2))
    return {"bytes": keys * nkv * (hd + 8) + 2 * rows * nh * hd * size + 4 * S * (longest // case["page"] + 2), "flops": 4 * pairs * nh * hd}


# ----------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    f = lambda n: s[n].double()  # noqa: E731
    if case["op"] == "norm":
        # (the residual sum as it is kept, in the activations' type: the norm is of that)
        r = f("x") if s["r"] is None else (f("x") + f("r")).to(s["x"].dtype).double()
        y = r * (r.pow(2).sum(1, keepdim=True) / case["hidden"] + EPS).rsqrt() * f("w")
        step = y.abs().max(1, keepdim=True).values / 127
        return [torch.where(step > 0, torch.round(y / step) * step, 0.0), step[:, 0]] + ([] if s["r"] is None else [r])
    if case["op"] == "product":
        y = torch.einsum("tk,nk,t,n->tn", f("q"), f("w"), f("s"), f("ws")) if case["rows"] * case["n"] < 4096 else (f("q") * f("s")[:, None]) @ (f("w") * f("ws")[:, None]).T
        return y if s["b"] is None else y + f("b")
    if case["op"] == "append":
        rot, half = case["rot"], case["rot"] // 2
        c = torch.complex(f("table")[:, :half], f("table")[:, half:])[s["positions"].long()][:, None]
        out = []
        for name in ("q", "k"):
            x = f(name).clone()
            ends = (slice(0, half), slice(half, rot)) if case["neox"] else (slice(0, rot, 2), slice(1, rot, 2))
            z = torch.complex(x[..., ends[0]].contiguous(), x[..., ends[1]].contiguous()) * c
            x[..., ends[0]], x[..., ends[1]] = z.real, z.imag
            out.append(x)
        out.append(f("v"))
        for i in (1, 2):
            x = out[i]
            ends = x.sort(-1).values
            d = torch.where(ends[..., -1:] + ends[..., :1] >= 0, ends[..., -1:], ends[..., :1]) / -8
            out[i] = torch.where((s["slots"] >= 0)[:, None, None] & (d != 0), torch.round(x / d).clamp(-8, 7) * d, 0.0)
        return out
    nh, nkv, hd = HEADS[case["heads"]]
    if case["seqs"] * case["q"] * case["longest"] * nh > 2**31:
        return None
    kb, vb, ks, vs = sections(s["pages"], case["page"], hd)
    starts = list(range(case["seqs"] + 1)) if s["starts"] is None else s["starts"].tolist()
    result = torch.zeros(starts[-1], nh, hd, dtype=torch.float64, device="cuda")
    for i, n in enumerate(s["lens"].tolist()):
        a, b = starts[i], starts[i + 1]
        if n == 0:
            continue
        ids = s["table"][i, : -(-n // case["page"])].long()
        for h in range(nkv):
            rows = []
            for bytes_, d in ((kb, ks), (vb, vs)):
                x = bytes_[ids, h].flatten(0, 1)[:n].long()
                m = torch.empty(n, hd, dtype=torch.float64, device="cuda")
                m[:, 0::2], m[:, 1::2] = (x % 16).double(), (x // 16).double()
                rows.append((m - 8) * d[ids, h].flatten()[:n, None].double())
            g = nh // nkv
            z = (s["q_tokens"][a:b, h * g : (h + 1) * g].double() @ rows[0].T) * s["scale"]
            far = torch.arange(n - (b - a), n, device="cuda")[:, None] - torch.arange(n, device="cuda")
            hide = (far < 0) | (far >= case["window"]) if case["window"] else far < 0
            z = z.masked_fill(hide[:, None], -math.inf)
            # (a token ahead of an empty cache sees nothing)
            result[a:b, h * g : (h + 1) * g] = torch.nan_to_num(torch.softmax(z, -1), nan=0.0) @ rows[1]
    return result
