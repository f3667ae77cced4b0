"""Attention over the 4-bit cache in 64 bits on the device, with a bound on what f32 arithmetic with pairs of fp16 numbers may be off by (tests only)."""
import torch

import device_ops_ref as R

DEVICE = "cuda"


def attention(q, pages, table, lens, starts, page, scale, window=0, again=False, exact_scores=False):
    """(o, off) f64 on the device: the result, and how far it may be off before it is rounded to the type of q.

    Z: the largest sum of |scale q_c k_c| of a row's scores.  A score is off by hd / 16 * 2^-22 Z (tensor-pipe steps of 16 that may cut products off at the 23rd bit of the largest), 2^-22 Z (the
    query's two halves), 2^-23 Z (the scale) and 2^-22 Z (the argument of the exponential); exact_scores: one channel makes them, in numbers that need no rounding: 2^-24 Z times 1.5 (the scale) and 1 (the
    argument).  That and 2^-20 from the exponential are errors of a probability, in the sum of weights too: o = sum p v changes by sum p e (v - o), at most max e times the deviation of v.
    The weights of values alone: 2^-22 from their two fp16 halves, 2^-24 from the product with d, the value's scale, or with 2^(log2 p + log2 d) in its place 2^-24 times these logarithms and the 16 of the
    reference's place.  A sum of products: 2^-22 of what is there, in each step of 16 keys from a key's own to the last, and 4 for what joins parts; the reciprocal and the end 2^-21 of the result.
    The halves end at 2^-25.  A reference that moves keeps the largest weight p d of a row (a value is at most 8 d) at 2^7 or above: L * 2^-32 * max(p max |v|).  A row of a sequence with more than 32 rows of
    a kv head may have one that stays: a weight of 2^3 (f32: 2^4) stands for the largest scale of a value in the first tile: L * 2^-28 (2^-29) * max |v| of the sequence, or what makes the block go over the keys again,
    2^-8, 2^-11 or 2^-16 (bf16, f16, f32) of the row's largest channel.  again: the inputs make it."""
    dev = torch.device(DEVICE)
    tokens, nh, hd = q.shape
    pages, table, qd, dtype = pages.to(dev), table.to(dev).long(), q.to(dev).double(), q.dtype
    n_pages, nkv = pages.shape[:2]
    g = nh // nkv
    kb, vb, ks, vs = R.sections(pages, page, hd)
    o, off = (torch.zeros(tokens, nh, hd, dtype=torch.float64, device=dev) for _ in range(2))
    for s, n in enumerate(lens):
        a, b = starts[s], starts[s + 1]
        if n == 0 or a == b:
            continue
        ids = table[s, : -(-n // page)]
        good = (ids >= 0) & (ids < n_pages)
        at = ids.clamp(0, n_pages - 1)
        here = good.repeat_interleave(page)[:n]
        pos = torch.arange(n - (b - a), n, device=dev)[:, None]
        j = torch.arange(n, device=dev)
        seen = (j <= pos) & here & ((j > pos - window) if window else True)
        many = (b - a) * g > 32
        for h in range(nkv):
            d = vs[at, h].double().flatten()[:n]
            k, v = (((torch.stack([x[at, h] & 15, x[at, h] >> 4], -1).flatten(-2).double() - 8) * y[at, h].double()[..., None]).flatten(0, 1)[:n] for x, y in ((kb, ks), (vb, vs)))
            k, v = (torch.where(here[:, None], x, 0.0) for x in (k, v))
            power = torch.where(here & (d != 0), d, 1.0).abs().log2().abs().max()
            x = qd[a:b, h * g : (h + 1) * g]
            z = torch.einsum("mgc,nc->mgn", x, k) * scale
            z = z.masked_fill(~seen[:, None], -torch.inf)
            big = (torch.einsum("mgc,nc->mgn", x.abs(), k.abs()) * abs(scale)).masked_fill(~seen[:, None], 0.0).amax(-1)
            p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            keys = seen.sum(-1).double()[:, None]
            r = p @ v
            o[a:b, h * g : (h + 1) * g] = r
            unit = v.abs().max().clamp(min=1e-300)      # (squares of values near the ends of f32)
            spread = ((p @ (v / unit).square() - (r / unit).square()).clamp(min=0)).sqrt() * unit
            dz = big * (2.5 * 2.0**-24 if exact_scores else hd / 16 * 2.0**-22 + 2.0**-22 + 2.0**-23 + 2.0**-22)
            steps = ((pos - j).clamp(min=0) / 16 + 5)[:, None]
            own = p * (2.0**-22 + 2.0**-24 * (1 + 16 + power - p.clamp(min=2.0**-300).log2()) + steps * 2.0**-22)
            low = keys * 2.0**-32 * (p * v.abs().amax(1)).amax(-1)
            if many and not again:
                low = torch.maximum(low, torch.minimum(keys * (2.0**-29 if dtype == torch.float32 else 2.0**-28) * v.abs().max(), 1.01 * R.COST[dtype] * r.abs().amax(-1)))
            off[a:b, h * g : (h + 1) * g] = spread * (dz + 2.0**-20)[..., None] + own @ v.abs() + 2.0**-21 * r.abs() + low[..., None]
    return o, off


def rounded(o, off, dtype):
    """The smallest and the largest number of `dtype` that results within off of o may be rounded to (through f32: half a step of that more)."""
    off = off + 1.01 * 2.0**-24 * o.abs()
    return tuple((o + s * off).float().to(dtype).double() for s in (-1, 1))
