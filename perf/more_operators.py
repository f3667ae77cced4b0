"""Operators of a feed-forward sublayer with routed experts that is served with activations in 8 bits and weights in 4 bits: what is timed and compared.

  route    a router's logits to each token's experts and their weights
  product  product of rows in 8 bits with 4-bit weights that have a scale per group of channels: one matrix, or each token's experts'
  glu      gated unit of a row's two halves, its result in 8 bits with a scale per row
  block    a block's output (or its experts' weighted sum), normed, gated and scaled, onto the residual stream, and the next norm's rows in 8 bits

4-bit weights lie in tiles of 16 rows x 64 channels of 512 bytes, [row tile][channel step][g 8][t 4][half 2][row half 2][4 bytes]: byte b there has channels
32 half + 8t + b (low four bits) and 32 half + 8t + 4 + b (high four bits) of row 8 row_half + g, in two's complement (-8 .. 7).  Their scales lie [row tile][group][g 8][row half 2].
"""
import math

import torch

own = False

TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
EPS = torch.tensor(1e-5).item()
TINY = 2.0**-119  # rows whose largest magnitude is below this are zeros in 8 bits


def listed():
    return [
        # one decoded token of an 8x7B model: latency
        dict(name="route_token", op="route", tokens=1, experts=8, top=2, score="softmax", correction=False, groups=1, top_groups=1, renormalise=True, padding=0, type="f32"),
        # prompts through a router of many experts, with a correction for balance and a choice among groups first
        dict(name="route_prompt", op="route", tokens=8192, experts=256, top=8, score="sigmoid", correction=True, groups=8, top_groups=4, renormalise=True, padding=0, type="bf16"),
        # a padded batch, an odd number of experts
        dict(name="route_ragged", op="route", tokens=777, experts=60, top=4, score="softmax", correction=False, groups=1, top_groups=1, renormalise=False, padding=100, type="f16"),
        # one token through an 8B model's query, key and value projection: latency, and the weights' bytes
        dict(name="product_token", op="product", rows=1, k=4096, n=6144, group=128, experts=0, top=0, scales="f16", type="bf16", bias=False),
        # a step of 33 sequences through its down projection
        dict(name="product_step", op="product", rows=33, k=14336, n=4096, group=64, experts=0, top=0, scales="bf16", type="f16", bias=False),
        # one token through two of eight experts' gate and up projections
        dict(name="experts_token", op="product", rows=1, k=4096, n=28672, group=32, experts=8, top=2, scales="f16", type="bf16", bias=False),
        # sixteen tokens through their experts' down projections: most of the weights are read, each for a few tokens
        dict(name="experts_step", op="product", rows=16, k=14336, n=4096, group=32, experts=8, top=2, scales="f16", type="f32", bias=False),
        # one token's two experts
        dict(name="glu_token", op="glu", rows=2, ff=14336, act="silu", type="bf16"),
        # a prompt chunk of 2048 tokens through two experts each
        dict(name="glu_prompt", op="glu", rows=4096, ff=14336, act="silu", type="bf16"),
        # one token behind its two experts, with a norm of the block's output
        dict(name="block_token", op="block", rows=1, hidden=4096, mix=2, post=True, gate="none", scale=1.0, type="bf16"),
        # a prompt chunk behind a dense block, with a learned gate per channel
        dict(name="block_prompt", op="block", rows=2048, hidden=4096, mix=0, post=True, gate="channel", scale=1.0, type="bf16"),
        # an odd number of rows of a 0.5B model's width, a gate per token, a residual scale
        dict(name="block_ragged", op="block", rows=333, hidden=896, mix=3, post=False, gate="token", scale=0.22, type="f32"),
    ]


def draw(rng):
    def size(lo, hi):
        return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))

    op, type_ = rng.choice(["route", "product", "product", "glu", "block"]), rng.choice(sorted(TYPES))
    if op == "route":
        groups = rng.choice([1, 1, 2, 4, 8])
        experts = groups * size(max(2, 4 // groups), 512 // groups)
        top_groups = rng.randint(1, groups)
        tokens = size(1, min(8192, 2**21 // experts))
        return dict(op=op, tokens=tokens, experts=experts, top=rng.randint(1, min(16, top_groups * experts // groups)), score=rng.choice(["softmax", "sigmoid"]),
                    correction=rng.random() < 0.5, groups=groups, top_groups=top_groups, renormalise=rng.random() < 0.7, padding=rng.choice([0, tokens // 3]), type=type_)
    if op == "product":
        group = rng.choice([32, 64, 128])
        experts = rng.choice([0, 0, size(4, 128)])
        k = group * size(1, 16384 // group)
        n = size(1, max(1, min(16384, 2**28 // (k * max(1, experts)))))
        top = rng.randint(1, min(8, experts)) if experts else 0
        return dict(op=op, rows=size(1, 64), k=k, n=n, group=group, experts=experts, top=top, scales=rng.choice(sorted(TYPES)), type=type_, bias=rng.random() < 0.3)
    if op == "glu":
        ff = rng.choice([size(32, 16384), 64 * size(1, 256)])
        return dict(op=op, rows=size(1, min(4096, 2**25 // ff)), ff=ff, act=rng.choice(["silu", "silu", "gelu", "relu"]), type=type_)
    hidden = rng.choice([size(32, 16384), 64 * size(1, 256)])
    mix = rng.choice([0, 1, 2, 8])
    return dict(op=op, rows=size(1, min(4096, 2**23 // (hidden * (mix + 1)))), hidden=hidden, mix=mix, post=rng.random() < 0.5, gate=rng.choice(["none", "token", "channel", "each"]),
                scale=rng.choice([1.0, 0.5, 0.22]), type=type_)


# ------------------------------------------------------------------------------------------------------------------ inputs
def padded(t):
    """The same rows at a distance of whole 16 bytes (t: int8)."""
    rows, k = t.shape
    buf = torch.zeros(rows, (k + 15) // 16 * 16, dtype=t.dtype, device=t.device)
    buf[:, :k] = t
    return buf[:, :k]


def tiled(v, s):
    """Values int8 [experts, n, k] and scales [experts, n, groups] as they are laid out in tiles."""
    e, n, k = v.shape
    down, right = -n % 16, -k % 64
    v = torch.nn.functional.pad(v, (0, right, 0, down)).bitwise_and_(15).view(torch.uint8).view(e, (n + down) // 16, 2, 8, (k + right) // 64, 2, 4, 2, 4)
    v = v.permute(0, 1, 4, 3, 6, 5, 2, 7, 8)  # experts, row tile, step, g, t, half, row half, (low, high), byte
    s = torch.nn.functional.pad(s, (0, 0, 0, down)).view(e, (n + down) // 16, 2, 8, -1).permute(0, 1, 4, 3, 2)
    return (v[..., 0, :] | v[..., 1, :] << 4).flatten(3), s.contiguous()


def prepare(case, seed):
    rng = torch.Generator("cuda").manual_seed(seed)
    host = torch.Generator().manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=rng)  # noqa: E731
    uniform = lambda *s: torch.rand(*s, device="cuda", generator=rng)  # noqa: E731
    t = TYPES[case["type"]]
    s = dict(case)
    if case["op"] == "route":
        logits = 2 * normal(case["tokens"], case["experts"])
        # places of a batch that hold no token: nothing is left to choose
        logits[torch.randperm(case["tokens"], generator=host)[: case["padding"]].cuda()] = -math.inf
        s.update(logits=logits.to(t), bias=0.1 * normal(case["experts"]) if case["correction"] else None)
    elif case["op"] == "product":
        rows, k, n, E, top = case["rows"], case["k"], case["n"], case["experts"], case["top"]
        v = (2.5 * normal(max(E, 1), n, k)).round_().clamp_(-8, 7).to(torch.int8)
        d = (0.002 + 0.004 * uniform(max(E, 1), n, k // case["group"])).to(TYPES[case["scales"]])
        w, ws = tiled(v, d)
        # (an up projection reads a token's row for each of its experts, a down projection a row of each)
        own_rows = E and k > n
        x = torch.round(32 * normal(rows * top if own_rows else rows, k)).clamp(-127, 127).to(torch.int8)
        s.update(x=padded(x), xs=0.01 + 0.02 * uniform(x.shape[0]), w=w if E else w[0], ws=ws if E else ws[0], chosen=None)
        s["b"] = (normal(E, n) if E else normal(n)) if case["bias"] else None
        if E:
            # some experts are chosen more often than others; a place without a token has none
            weight = torch.rand(E, generator=host) + 0.2
            chosen = torch.multinomial(weight.expand(rows, E), top, generator=host).int()
            chosen[torch.rand(rows, generator=host) < (0.1 if rows > 4 else 0.0)] = -1
            s["chosen"] = chosen.cuda()
    elif case["op"] == "glu":
        x = normal(case["rows"], 2 * case["ff"])
        s["x"] = (x * (1 + 10 * (uniform(2 * case["ff"]) < 0.002))).to(t)  # a few channels stand out
    else:
        rows, n = case["rows"], case["hidden"]
        s.update(y=(0.5 * normal(rows * max(1, case["mix"]), n)).to(t), r=(normal(rows, n) * (1 + 20 * (uniform(n) < 0.01))).to(t), w=1 + 0.1 * normal(n))
        s["mixing"] = torch.softmax(normal(rows, case["mix"]), 1) if case["mix"] else None
        s["post_w"] = 0.3 + 0.1 * uniform(n) if case["post"] else None
        shape = {"none": None, "token": (rows, 1), "channel": (1, n), "each": (rows, n)}[case["gate"]]
        s["g"] = None if shape is None else torch.sigmoid(normal(*shape)).to(t).expand(rows, n)
    return s


# ------------------------------------------------------------------------------------------------------------- plain forms
def first_places(c, many):
    """The `many` largest of each row in falling order, the lower place first among equals, and their places."""
    v, i = torch.sort(c, dim=-1, descending=True, stable=True)
    return v[..., :many], i[..., :many]


def plain_route(s):
    z = s["logits"].double()  # (scores next to one another decide, so they are made in 64 bits)
    t, E = z.shape
    live = z > -math.inf
    if s["score"] == "softmax":
        e = torch.where(live, torch.exp(z - z.amax(1, keepdim=True)), 0.0)
        p = torch.where(live, e / e.sum(1, keepdim=True), 0.0)
    else:
        p = torch.where(live, 1 / (1 + torch.exp(-z)), 0.0)
    c = z if s["bias"] is None else torch.where(live, p + s["bias"].double(), -math.inf)
    if s["groups"] > 1:
        # a group counts by its two best scores, as they stand in the choice
        of = (p if s["bias"] is None else c).view(t, s["groups"], -1)
        of = torch.where(live.view(of.shape), of, -math.inf)
        best = first_places(of, 2)[0]
        value = torch.where(best[..., 0] > -math.inf, torch.where(best > -math.inf, best, 0.0).sum(-1), -math.inf)
        kept = first_places(value, s["top_groups"])[1]
        stays = torch.zeros(t, s["groups"], dtype=torch.bool, device=z.device).scatter_(1, kept, True)
        c = torch.where(stays[..., None].expand(t, s["groups"], E // s["groups"]).reshape(t, E), c, -math.inf)
    v, i = first_places(c, s["top"])
    w = torch.where(v > -math.inf, p.gather(1, i), 0.0)
    if s["renormalise"]:
        total = w.sum(1, keepdim=True)
        w = w / torch.where(total > 0, total, 1.0)
    return [torch.where(v > -math.inf, i, -1).int(), w.float()]


def weights(w, ws, n, k, real):
    """[experts, n, k] of the values that tiled weights stand for."""
    e, R, K = w.shape[:3]
    w = w.view(e, R, K, 8, 4, 2, 2, 4)
    v = torch.stack([w << 4, w & 240], -2).view(torch.int8)  # (sixteen times the value)
    v = v.permute(0, 1, 6, 3, 2, 5, 4, 7, 8).reshape(e, R * 16, K * 64)[:, :n, :k].to(real)
    d = ws.permute(0, 1, 4, 3, 2).reshape(e, R * 16, 1, -1)[:, :n, 0].to(real)
    return v.unflatten(2, (d.shape[2], -1)).mul_(d[..., None] / 16).flatten(2)


def plain_product(s):
    n, k, top = s["n"], s["k"], s["top"]
    x = s["x"].float()
    if s["chosen"] is None:
        y = (x @ weights(s["w"][None], s["ws"][None], n, k, torch.float32)[0].T) * s["xs"][:, None]
        return (y if s["b"] is None else y + s["b"]).to(TYPES[s["type"]])
    chosen = s["chosen"].flatten().long()
    to = chosen.clamp(min=0)
    pairs = torch.arange(len(chosen), device=x.device)
    row = pairs if len(x) == len(chosen) else pairs // top
    if len(chosen) < len(s["w"]):  # the chosen experts' weights
        y = torch.einsum("pk,pnk->pn", x[row], weights(s["w"][to], s["ws"][to], n, k, torch.float32))
    else:  # all rows through all experts
        y = torch.einsum("rk,enk->ren", x, weights(s["w"], s["ws"], n, k, torch.float32))[row, to]
    y = y * s["xs"][row][:, None]
    y = y if s["b"] is None else y + s["b"][to]
    return torch.where(chosen[:, None] >= 0, y, 0.0).to(TYPES[s["type"]])


def in_8_bits(y):
    """Rows of y as [the values that their 8-bit numbers stand for, the scales]."""
    top = y.abs().amax(-1, keepdim=True)
    live = top >= TINY
    q = torch.where(live, torch.round(y * torch.where(live, torch.full_like(top, 127) / top, 0.0)), 0.0)
    scale = torch.where(live, top / torch.full_like(top, 127), 0.0).float()
    return [(q.float() * scale).bfloat16(), scale[:, 0]]


def plain_glu(s):
    g, u = s["x"].double().chunk(2, 1)  # (values next to the border between two 8-bit numbers)
    if s["act"] == "silu":
        a = g / (1 + torch.exp(-g))
    elif s["act"] == "gelu":
        a = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g * g * g)))
    else:
        a = g.clamp(min=0)
    return in_8_bits(a * u)


def normed(x, w):
    return x * (1 / torch.sqrt(x.double().square().mean(-1, keepdim=True) + EPS)).float() * w


def plain_block(s):
    t = TYPES[s["type"]]
    y = s["y"].float()
    if s["mixing"] is not None:
        y = (y.unflatten(0, s["mixing"].shape) * s["mixing"][..., None]).sum(1)
    if s["post_w"] is not None:
        y = normed(y, s["post_w"])
    if s["g"] is not None:
        y = y * s["g"].float()
    r = (s["r"].float() + y * torch.tensor(s["scale"], dtype=torch.float32, device=y.device)).to(t)
    return [*in_8_bits(normed(r.float(), s["w"])), r]


def run(s):
    if not own:
        return {"route": plain_route, "product": plain_product, "glu": plain_glu, "block": plain_block}[s["op"]](s)
    from llama_gguf_b200 import device_ops as D

    if s["op"] == "route":
        return list(D.route_experts(s["logits"], s["top"], score=s["score"], correction=s["bias"], groups=s["groups"], top_groups=s["top_groups"], renormalise=s["renormalise"]))
    if s["op"] == "product":
        return D.mat_mat_i4(s["x"], s["xs"], s["w"], s["ws"], n=s["n"], experts=s["chosen"], bias=s["b"], dtype=TYPES[s["type"]])
    if s["op"] == "glu":
        q, scale = D.glu_q8(s["x"], act=s["act"])
        return [D.read_q8(q, scale, torch.bfloat16), scale]
    q, scale, r = D.add_gated_norm_q8(s["y"], s["r"], s["w"], EPS, mix=s["mixing"], post_weight=s["post_w"], gate=s["g"], scale=s["scale"])
    return [D.read_q8(q, scale, torch.bfloat16), scale, r]


def work(case):
    size = 4 if case["type"] == "f32" else 2
    if case["op"] == "route":
        n = case["tokens"] * case["experts"]
        return {"bytes": n * size + 8 * case["tokens"] * case["top"] + 4 * case["experts"] * case["correction"], "flops": n * (4 + case["top"])}
    if case["op"] == "product":
        rows, k, n, E, top = case["rows"], case["k"], case["n"], case["experts"], case["top"]
        reached = E * (1 - (1 - top / E) ** rows) if E else 1  # experts that some token has chosen
        outs = rows * max(1, top)
        ins = outs if E and k > n else rows
        scale = 4 if case["scales"] == "f32" else 2
        return {"bytes": int(reached * n * (k // 2 + k // case["group"] * scale + 4 * case["bias"])) + ins * (k + 4) + outs * (n * size + 4 * (E > 0)), "flops": 2 * outs * k * n}
    if case["op"] == "glu":
        n = case["rows"] * case["ff"]
        return {"bytes": n * (2 * size + 1 + 2) + 4 * case["rows"], "flops": 10 * n}
    rows, n, mix = case["rows"], case["hidden"], case["mix"]
    gate = {"none": 0, "token": rows, "channel": n, "each": rows * n}[case["gate"]]
    return {"bytes": rows * n * (size * (max(1, mix) + 2) + 1 + 2) + gate * size + 4 * (rows * (mix + 1) + n * (1 + case["post"])), "flops": rows * n * (12 + 2 * mix)}


# ----------------------------------------------------------------------------------------------------------------- exact
def exact(case, seed):
    s = prepare(case, seed)
    f = lambda n: s[n].double()  # noqa: E731
    if case["op"] == "route":
        z = f("logits")
        live = torch.isfinite(z)
        p = torch.nan_to_num(torch.softmax(z, 1), nan=0.0) if case["score"] == "softmax" else torch.sigmoid(z)
        by = z if s["bias"] is None else p + f("bias")
        by = torch.where(live, by, -math.inf)
        if case["groups"] > 1:
            shape = (len(z), case["groups"], -1)
            two = torch.where(live, p if s["bias"] is None else by, -math.inf).view(shape).topk(2, -1).values
            value = two[..., 0] + two[..., 1].clamp(min=-1e300).where(two[..., 1] > -math.inf, torch.zeros_like(two[..., 1]))
            rank = (value[:, None, :] > value[:, :, None]).sum(-1) + ((value[:, None, :] == value[:, :, None]) & torch.ones(shape[1], shape[1], dtype=torch.bool, device="cuda").tril(-1)).sum(-1)
            by = torch.where((rank < case["top_groups"])[..., None], by.view(shape), -math.inf).view(z.shape)
        ids, left = [], by.clone()
        for _ in range(case["top"]):  # the first of the largest, again and again
            top = left.amax(1, keepdim=True)
            i = (left == top).int().argmax(1, keepdim=True)
            ids.append(torch.where(top > -math.inf, i, -1))
            left.scatter_(1, i, -math.inf)
        ids = torch.cat(ids, 1)
        w = p.gather(1, ids.clamp(min=0)) * (ids >= 0)
        if case["renormalise"]:
            w = torch.nan_to_num(w / w.sum(1, keepdim=True), nan=0.0)
        return [ids.int(), w]
    if case["op"] == "product":
        n, k, group = case["n"], case["k"], case["group"]
        w, ws = (s["w"], s["ws"]) if case["experts"] else (s["w"][None], s["ws"][None])
        chosen = torch.zeros(case["rows"], 1, dtype=torch.int64) if s["chosen"] is None else s["chosen"].long().cpu()
        flat = chosen.flatten()
        x = f("x") * f("xs")[:, None]
        y = torch.zeros(len(flat), n, dtype=torch.float64, device="cuda")
        row, ch = torch.arange(n, device="cuda"), torch.arange(k, device="cuda")
        # where each value's byte lies in its tile, and which half of it it is
        inner = ((row % 8)[:, None] * 4 + (ch % 32 // 8)) * 16 + (ch % 64 // 32) * 8 + (row % 16 // 8)[:, None] * 4 + ch % 4
        for e in sorted(set(flat.tolist()) - {-1}):
            at = (flat == e).nonzero()[:, 0].cuda()
            for a in range(0, n, 4096):  # (in parts: 64-bit indices of a whole matrix are large)
                r = row[a : a + 4096]
                nib = w[e][(r // 16)[:, None], ch // 64, inner[a : a + 4096]] >> (ch % 8 // 4 * 4).to(torch.uint8) & 15
                nib = nib.double()
                m = torch.where(nib > 7, nib - 16, nib) * ws[e][(r // 16)[:, None], ch // group, (r % 8)[:, None], (r % 16 // 8)[:, None]].double()
                y[at, a : a + 4096] = x[at if len(x) == len(flat) else at // max(1, case["top"])] @ m.T
            if s["b"] is not None:
                y[at] += f("b")[e] if case["experts"] else f("b")
        return y
    if case["op"] == "glu":
        x = f("x")
        g, u = x[:, : case["ff"]], x[:, case["ff"] :]
        a = {"silu": lambda v: v * torch.sigmoid(v), "gelu": lambda v: v * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (v + 0.044715 * v**3)), "relu": torch.relu}[case["act"]](g)
        y, kept = a * u, []
    else:
        y = f("y")
        if case["mix"]:
            y = torch.einsum("rm,rmn->rn", f("mixing"), y.view(case["rows"], case["mix"], -1))
        if case["post"]:
            y = y * (y.pow(2).mean(1, keepdim=True) + EPS).rsqrt() * f("post_w")
        if s["g"] is not None:
            y = y * f("g")
        r = f("r") + case["scale"] * y
        # (the norm is of the stream as it is kept, in the activations' type)
        kept = [r]
        r = r.float().to(s["r"].dtype).double()
        y = r * (r.pow(2).mean(1, keepdim=True) + EPS).rsqrt() * f("w")
    step = y.abs().amax(1, keepdim=True) / 127
    return [torch.where(step > 0, torch.round(y / torch.where(step > 0, step, 1.0)) * step, 0.0), step[:, 0], *kept]
