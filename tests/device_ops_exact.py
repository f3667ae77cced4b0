"""Attention over the 4-bit cache in 64 bits on the device, with a bound on what f32 arithmetic with pairs of fp16 numbers may be off by (tests only)."""
import torch

import device_ops_ref as R

DEVICE = "cuda"


def attention(q, pages, table, lens, starts, page, scale, window=0, again=False, exact_scores=False):
    """(o, off) f64 on the device: the result, and how far it may be off before it is rounded to the type of q.

    Z: the largest sum of |scale q_c k_c| of a row's scores.  A score is off by hd / 16 * 2^-22 Z (tensor-pipe steps of 16 that may cut products off at the 23rd bit of the largest), 2^-22 Z (the
    query's two halves), 2^-23 Z (the scale) and 2^-22 Z (the argument of the exponential); exact_scores: one channel makes them, in numbers that need no rounding: 2^-24 Z times 1.5 (the scale) and 1 (the argument).
    A probability is off by that times itself, twice since the sum has it too; by 2^-20 of itself from the exponential's own steps, by 2^-22 from its two fp16 halves; the sum over L keys by L / 16 * 2^-22 of sum p |v|.
    The halves end at 2^-25.  A reference that moves keeps the largest weight p d of a row (d a value's scale, a value is at most 8 d) at 2^7 or above: L * 2^-32 * max(p max |v|).  A row of a sequence with
    more than 32 rows of a kv head may have one that stays: weights of 1 (f32: 2^4) stand for the largest scale of a value in the first tile; L * 2^-25 (2^-29) * max |v| of the sequence, or what makes
    the block take moving ones, 2^-8, 2^-11 or 2^-16 (bf16, f16, f32) of the row's largest channel.  again: the inputs make it take them."""
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
            k, v = (((torch.stack([x[at, h] & 15, x[at, h] >> 4], -1).flatten(-2).double() - 8) * d[at, h].double()[..., None]).flatten(0, 1)[:n] for x, d in ((kb, ks), (vb, vs)))
            k, v = (torch.where(here[:, None], x, 0.0) for x in (k, v))
            x = qd[a:b, h * g : (h + 1) * g]
            z = torch.einsum("mgc,nc->mgn", x, k) * scale
            z = z.masked_fill(~seen[:, None], -torch.inf)
            big = (torch.einsum("mgc,nc->mgn", x.abs(), k.abs()) * abs(scale)).masked_fill(~seen[:, None], 0.0).amax(-1)
            p = torch.nan_to_num(torch.softmax(z, -1), nan=0.0)
            keys = seen.sum(-1).double()[:, None]
            r = p @ v
            o[a:b, h * g : (h + 1) * g] = r
            dz = big * (2.5 * 2.0**-24 if exact_scores else hd / 16 * 2.0**-22 + 2.0**-22 + 2.0**-23 + 2.0**-22)
            low = keys * 2.0**-32 * (p * v.abs().amax(1)).amax(-1)
            if many and not again:
                low = torch.maximum(low, torch.minimum(keys * R.FLOOR[dtype] * v.abs().max(), 1.01 * R.COST[dtype] * r.abs().amax(-1)))
            off[a:b, h * g : (h + 1) * g] = (p @ v.abs()) * (2 * dz + 2.0**-22 + 2.0**-20 + keys / 16 * 2.0**-22)[..., None] + low[..., None]
    return o, off


def rounded(o, off, dtype):
    """The smallest and the largest number of `dtype` that results within off of o may be rounded to (through f32: half a step of that more)."""
    off = off + 1.01 * 2.0**-24 * o.abs()
    return tuple((o + s * off).float().to(dtype).double() for s in (-1, 1))
