"""Plain restatements, in 64 bits on the CPU, of the operators on device tensors for feed-forwards with 4-bit weights and routed experts (tests only)."""
import math

import torch

TINY = 2.0**-119
HALF_STEP = {torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
LEAST = {torch.float32: 2.0**-150, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}      # half a step of the subnormals


def route(logits, top, score="softmax", correction=None, groups=1, top_groups=1, renormalise=True, scale=1.0):
    """(experts, weights f64), row by row in Python numbers."""
    ids, ws = [], []
    for row in logits.double().tolist():
        n = len(row)
        nan = any(math.isnan(z) or (score == "softmax" and z == math.inf) for z in row)
        live = [z > -math.inf for z in row]
        if score == "softmax":
            most = max([z for z, a in zip(row, live) if a], default=0.0)
            e = [0.0 if not a else 1.0 if z == most else math.exp(z - most) for z, a in zip(row, live)] if not nan else [0.0] * n
            total = math.fsum(e)
            p = [v / total if total else 0.0 for v in e]
        else:
            p = [(1 / (1 + math.exp(-z)) if z > -700 else 0.0) if a else 0.0 for z, a in zip(row, live)]
        by = [(z if correction is None or nan else v + c) if a else -math.inf for z, v, a, c in zip(row, p, live, [0.0] * n if correction is None else correction.double().tolist())]
        by = [-math.inf if math.isnan(v) else v for v in by]
        left = list(range(n))
        if groups > 1:
            each = n // groups
            value = []
            for g in range(groups):
                ours = range(g * each, (g + 1) * each)
                if nan:
                    value.append(max(by[i] for i in ours))
                else:
                    best = sorted(((by[i] if correction is not None else p[i]) for i in ours if by[i] > -math.inf), reverse=True)[:2]
                    value.append(sum(best) if best else -math.inf)
            kept = [g for g in sorted(range(groups), key=lambda g: (-value[g], g))[:top_groups] if value[g] > -math.inf]
            left = [i for i in left if i // each in kept]
        chosen = sorted((i for i in left if by[i] > -math.inf), key=lambda i: (-by[i], i))[:top]
        w = [p[i] for i in chosen]
        total = math.fsum(w)
        if renormalise and total > 0:
            w = [v / total for v in w]
        more = top - len(chosen)
        ids.append(chosen + [-1] * more)
        ws.append([math.nan if nan else v * scale for v in w] + [0.0] * more)
    return torch.tensor(ids, dtype=torch.int32).view(-1, top), torch.tensor(ws, dtype=torch.float64).view(-1, top)


def product(a, s, values, scales, experts=None, bias=None):
    """(y f64, bound): values int8 [.., n, k], scales [.., n, groups]; bound: what the f32 sum over the groups, the row's scale and the bias may be off by, before the result is rounded.

    A group's sum is an integer below 2^24, exact; a product with its scale and a sum of G + 8 such (in any order) are off by at most (G + 9) half steps of the sum of magnitudes; the
    row's scale and the bias one each."""
    groups = scales.shape[-1]
    pairs = torch.zeros(len(a), 1, dtype=torch.int64) if experts is None else experts.long()
    flat = pairs.flatten()
    if experts is None:
        values, scales, bias = values[None], scales[None], None if bias is None else bias[None]
    n = values.shape[1]
    y, off = torch.zeros(len(flat), n, dtype=torch.float64), torch.zeros(len(flat), n, dtype=torch.float64)
    for p, e in enumerate(flat.tolist()):
        if not 0 <= e < len(values):
            continue
        row = p if len(a) == len(flat) else p // pairs.shape[1]
        inner = (values[e].unflatten(1, (groups, -1)).double() * a[row].double().view(groups, -1)).sum(-1)      # exact
        terms = inner * scales[e].double() * s[row].double()
        y[p] = terms.sum(-1)
        off[p] = terms.abs().sum(-1) * (groups + 10) * 2.0**-24
        if bias is not None:
            y[p] += bias[e].double()
            off[p] += 2.0**-24 * (y[p].abs() + off[p])
    return y, off


def glu(x, act):
    """y f64 of act(gate) * up."""
    g, u = x.double().chunk(2, 1)
    if act == "silu":
        g = torch.where(g < -700, g * torch.exp(g), g / (1 + torch.exp(-g)))
    elif act == "gelu":
        g = 0.5 * g * (1 + torch.tanh(math.sqrt(2 / math.pi) * (g + 0.044715 * g**3)))
    else:
        g = torch.where(g > 0, g, g * 0)
    return g * u


def gated(y, residual, eps, mix=None, post_weight=None, gate=None, scale=1.0):
    """(r f64 before it is rounded to the type, bound): a product or sum of f32 is off by half a step; the norm by three of them, its mean's share included."""
    h = 2.0**-24
    m, off = y.double(), torch.zeros(y.shape, dtype=torch.float64)
    if mix is not None:
        t = m.unflatten(0, mix.shape) * mix.double()[..., None]
        m, off = t.sum(1), t.abs().sum(1) * (mix.shape[1] + 1) * h
    if post_weight is not None:
        rms = (m.square().mean(1, keepdim=True) + float(torch.tensor(eps))).sqrt()
        slip = off.square().mean(1, keepdim=True).sqrt() / rms      # of the root mean square, relative
        w = post_weight.double()
        m, off = m / rms * w, (off / rms + (m / rms).abs() * (slip + 3.01 * h)) * w.abs()
    if gate is not None:
        m, off = m * gate.double(), off * gate.double().abs() + h * (m * gate.double()).abs()
    s = float(torch.tensor(scale))
    r = residual.double() + m * s
    return r, off * abs(s) + h * (m * s).abs() * 1.01 + h * r.abs() * 1.01
