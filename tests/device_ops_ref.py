"""Plain restatements, in 64 bits, of the operators on device tensors, and the 4-bit cache's bytes in plain torch (tests only)."""
import math

import torch

TINY = 2.0**-119
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
FLOOR = {torch.float32: 2.0**-29, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-25}
COST = {torch.float32: 2.0**-16, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
LEAST = {torch.float32: 0.0, torch.float16: 2.0**-25, torch.bfloat16: 0.0}  # half a step of the subnormals


def quantise_f32(x):
    """(nibbles uint8, scale f32) of rows x f32: the operator's own arithmetic, step by step in f32."""
    hi, lo = x.amax(-1, keepdim=True), x.amin(-1, keepdim=True)
    top = torch.where(hi >= -lo, hi, lo)
    finite = torch.isfinite(x).all(-1, keepdim=True)
    live = finite & (top.abs() >= TINY)
    scale = torch.where(live, top * -0.125, torch.zeros_like(top))
    inv = torch.where(live, 1.0 / torch.where(live, scale, 1.0), 0.0)
    n = torch.where(live, (torch.round(torch.where(finite, x, 0.0) * inv) + 8).clamp(max=15), 8.0).to(torch.uint8)
    return n, torch.where(finite, scale, math.nan)[..., 0]


def sections(pages, page, hd):
    p, nkv, _ = pages.shape
    r = page * hd // 2
    view = lambda a, n: pages[:, :, a : a + n]  # noqa: E731
    return (view(0, r).view(p, nkv, page, hd // 2), view(r, r).view(p, nkv, page, hd // 2), view(2 * r, 4 * page).view(torch.float32),
            view(2 * r + 4 * page, 4 * page).view(torch.float32))


def put_rows(pages, page, hd, slots, k, v):
    """Rows k, v f32 [tokens, kv heads, hd] into the pages (in place)."""
    kb, vb, ks, vs = sections(pages, page, hd)
    for b, s, x in ((kb, ks, k), (vb, vs, v)):
        n, d = quantise_f32(x)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < pages.shape[0] * page:
                b[slot // page, :, slot % page] = n[t][:, 0::2] | (n[t][:, 1::2] << 4)
                s[slot // page, :, slot % page] = d[t]


def values(pages, page, hd):
    """(k, v) f64 [positions of the cache, kv heads, hd]."""
    kb, vb, ks, vs = sections(pages, page, hd)
    out = []
    for b, s in ((kb, ks), (vb, vs)):
        n = torch.stack([b & 15, b >> 4], -1).flatten(-2).double() - 8
        out.append((n * s.double()[..., None]).transpose(1, 2).flatten(0, 1))
    return out


def rotate(x, cos, sin, neox):
    """x [tokens, heads, hd] with cos, sin [tokens, 1, pairs], in the type of x."""
    h = cos.shape[-1]
    y = x.clone()
    a, b = (x[..., :h], x[..., h : 2 * h]) if neox else (x[..., 0 : 2 * h : 2], x[..., 1 : 2 * h : 2])
    u, w = a * cos - b * sin, b * cos + a * sin
    if neox:
        y[..., :h], y[..., h : 2 * h] = u, w
    else:
        y[..., 0 : 2 * h : 2], y[..., 1 : 2 * h : 2] = u, w
    return y


def attention(q, kv, table, lens, starts, page, scale, window, n_pages, dtype=torch.float32):
    """(o, bound) f64: the result, and how far f32 arithmetic may be off before the result is rounded.

    With Z the largest sum of |scale q_c k_c| of a row's scores: an f32 sum of a head's products by tensor-pipe steps of 16 is off by at most hd / 16 * 2^-22 Z (each step
    may cut its products off at the 23rd bit of the largest), the query's two halves add 2^-22 Z, the scale 2^-23 Z; a probability is then off by that times itself (twice: in the
    sum too), by 2^-21 from the exponential's argument and value and 2^-21 from its own two halves (bf16 results: 2^-11 from its one;
    f32 and f16 results of sequences of more than 32 rows of a kv head: two bf16 numbers, 2^-8 of 2^-8), and the sum over L keys by L / 16 * 2^-22 of sum p |v|.
    The two fp16 halves of a weight p d (d a value's scale) end at 2^-24 of a reference that the largest weight reaches: whatever its size, a weight is off by 2^-25 of the largest, and a
    value is at most 8 d, so that a channel whose large weights meet values of zero keeps L * 2^-25 * 8 max(p d) = L * 2^-25 * max(p max |v|).  (Many rows: the
    reference is the largest score of the first tile with the largest scale of a value there, whose own score may be small, and the weights there are 1, or 2^4 for f32:
    L * 2^-25 or 2^-29 * max |v| of the sequence; a block where that may be more than 2^-8, 2^-11 or 2^-16 (bf16, f16, f32) of a row's largest channel is done again without it.)"""
    k, v = kv
    o = torch.zeros(q.shape, dtype=torch.float64)
    off = torch.zeros(q.shape, dtype=torch.float64)
    nh, hd = q.shape[1:]
    g = nh // k.shape[1]
    for s in range(len(lens)):
        n, a, b = lens[s], starts[s], starts[s + 1]
        many = (b - a) * g > 32
        held = [table[s][j // page] * page + j % page for j in range(n) if 0 <= table[s][j // page] < n_pages]
        far = torch.nan_to_num(v[torch.tensor(held)]).abs().max() if held else 0.0
        for i, t in enumerate(range(a, b)):
            pos = n - (b - a) + i
            keys = [j for j in range(max(0, pos - window + 1) if window else 0, pos + 1)]
            keys = [j for j in keys if 0 <= table[s][j // page] < n_pages]
            if not keys:
                continue
            at = torch.tensor([table[s][j // page] * page + j % page for j in keys])
            for h in range(nh):
                kk, vv = k[at, h // g], v[at, h // g]
                z = (kk @ q[t, h]) * scale
                p = torch.softmax(z, 0)
                big = float(((kk.abs() @ q[t, h].abs()) * abs(scale)).max())
                o[t, h] = p @ vv
                dz = big * (hd / 16 * 2.0**-22 + 2.0**-22 + 2.0**-23 + 2.0**-22)
                off[t, h] = (p @ vv.abs()) * (2 * dz + (2.0**-11 if dtype == torch.bfloat16 else 2.0**-16 if many else 0) + 2.0**-20 + len(keys) / 16 * 2.0**-22) + max(len(keys) * 2.0**-25 * (p * vv.abs().amax(1)).max(), min(len(keys) * FLOOR[dtype] * far, 1.01 * COST[dtype] * o[t, h].abs().max()) if many else 0.0)
    return o, off
