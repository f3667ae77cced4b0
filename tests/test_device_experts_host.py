"""Refusals of the operators on device tensors for routed experts and 4-bit weights, and how those weights are laid out, without a GPU."""
import ctypes as C
import math

import pytest
import torch

BUF = (C.c_char * 4096)()
AT = (C.addressof(BUF) + 255) & ~255      # never followed: every call below is refused first


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    return device_ops


def refused(b200, rc, exc, words):
    assert rc == {v: k for k, v in b200._STATUS.items()}[exc], (rc, b200.lib().b200_last_error())
    assert words in b200.lib().b200_last_error().decode()


def test_layout_of_4_bit_weights(D):
    """Byte by byte, as the header describes it."""
    g = torch.Generator().manual_seed(1)
    for lead, n, k, group in (((), 17, 96, 32), ((3,), 16, 64, 64), ((2,), 40, 256, 128)):
        v = torch.randint(-8, 8, (*lead, n, k), generator=g, dtype=torch.int8)
        s = torch.rand(*lead, n, k // group, generator=g).half()
        w, ws = D.i4_weights(v, s)
        assert w.shape == (*lead, (n + 15) // 16, (k + 63) // 64, 512) and ws.shape == (*lead, (n + 15) // 16, k // group, 8, 2) and ws.dtype == s.dtype
        flat, fs, fv, sv = w.reshape(-1, *w.shape[-3:]), ws.reshape(-1, *ws.shape[-4:]), v.reshape(-1, n, k), s.reshape(-1, n, k // group)
        for e in range(len(flat)):
            for r in range(flat.shape[1] * 16):
                for c in range(flat.shape[2] * 64):
                    at = ((r % 8 * 4 + c % 32 // 8) * 2 + c % 64 // 32) * 8 + r % 16 // 8 * 4 + c % 4
                    b = int(flat[e, r // 16, c // 64, at]) >> (4 if c % 8 >= 4 else 0) & 15
                    assert b == (int(fv[e, r, c]) & 15 if r < n and c < k else 0)
            for r in range(n):
                assert torch.equal(fs[e, r // 16, :, r % 8, r % 16 // 8], sv[e, r])
        back = D.read_i4(w, ws, n, k)
        assert torch.equal(back, v.float() * s.float().repeat_interleave(group, -1))


def test_weights_from_blocks(D):
    """Q4_0: 18 bytes, an f16 scale and 32 numbers, element j in the low four bits of byte j, element 16 + j in its high four; a value is scale * (number - 8)."""
    g = torch.Generator().manual_seed(2)
    n, k = 20, 160
    blocks = torch.randint(0, 256, (n, k // 32, 18), generator=g, dtype=torch.uint8)
    blocks[..., :2] = torch.rand(n, k // 32, 1, generator=g).half().view(torch.uint8)
    want = torch.zeros(n, k)
    for r in range(n):
        for b in range(k // 32):
            d = blocks[r, b, :2].clone().view(torch.float16).float()
            for j in range(16):
                want[r, b * 32 + j] = d * (int(blocks[r, b, 2 + j]) % 16 - 8)
                want[r, b * 32 + 16 + j] = d * (int(blocks[r, b, 2 + j]) // 16 - 8)
    assert torch.equal(D.read_i4(*D.i4_from_q4_0(blocks.flatten(1), k), n, k), want)
    import numpy as np
    import oracle as O

    assert np.array_equal(O.dequantize(2, blocks.numpy(), n * k).reshape(n, k), want.numpy())


def test_quantised_weights(D):
    x = torch.tensor([[1.0, -2.0, 8.0, 4.0] * 8, [0.0] * 32, [-7.0, 3.5, 0.4, -0.5] * 8])
    w, s = D.quantise_i4(x, 32, torch.float32)
    back = D.read_i4(w, s, 3, 32)
    assert torch.equal(back[:2, :4], torch.tensor([[1.0, -2.0, 8.0, 4.0], [0.0] * 4])) and float(back[2, 0]) == -7.0
    for bad in (lambda: D.quantise_i4(x, 16), lambda: D.quantise_i4(x, 64), lambda: D.i4_weights(x.to(torch.int8), s[:1]), lambda: D.i4_from_q4_0(torch.zeros(2, 17, dtype=torch.uint8), 32)):
        with pytest.raises(Exception) as e:
            bad()
        assert type(e.value).__name__ == "ShapeMismatch"


def route(D, **kw):
    a = D.Route(device=0, type=0, logits=AT, ld=8, tokens=2, n=8, top=2, groups=1, top_groups=1, scale=1.0, experts=AT, weights=AT)
    for k, v in kw.items():
        setattr(a, k, v)
    return D._lib().b200_dev_route_experts(C.byref(a))


def test_routing_refusals(b200, D):
    for change, exc, words in [
            (dict(type=3), b200.UnsupportedDType, "type 3"), (dict(n=0), b200.ShapeMismatch, "experts"), (dict(n=1025), b200.ShapeMismatch, "experts"), (dict(tokens=-1), b200.ShapeMismatch, "tokens"),
            (dict(tokens=1 << 31), b200.ShapeMismatch, "tokens"), (dict(groups=0), b200.ShapeMismatch, "groups"), (dict(groups=3), b200.ShapeMismatch, "groups"),
            (dict(n=66, groups=33), b200.ShapeMismatch, "groups"), (dict(top_groups=2), b200.ShapeMismatch, "top_groups"), (dict(top_groups=0), b200.ShapeMismatch, "top_groups"),
            (dict(top=0), b200.ShapeMismatch, "top"), (dict(top=9), b200.ShapeMismatch, "top"), (dict(n=64, top=33), b200.ShapeMismatch, "top"), (dict(groups=4, top=3), b200.ShapeMismatch, "top"),
            (dict(ld=-1), b200.ShapeMismatch, "negative"), (dict(scale=math.inf), b200.InvalidArgument, "scale"), (dict(logits=None), b200.InvalidArgument, "null"),
            (dict(experts=None), b200.InvalidArgument, "null"), (dict(weights=None), b200.InvalidArgument, "null")]:
        refused(b200, route(D, **change), exc, words)
    refused(b200, D._lib().b200_dev_route_experts(None), b200.InvalidArgument, "null")
    assert route(D, tokens=0, logits=None) == 0


def product(D, **kw):
    a = D.I4Product(device=0, out_type=0, scale_type=1, group=32, a=AT, lda=64, a_scales=AT, w=AT, w_scales=AT, out=AT, ldo=8, tokens=2, k=64, n=8)
    for k, v in kw.items():
        setattr(a, k, v)
    return D._lib().b200_dev_mat_mat_i4(C.byref(a))


def test_product_refusals(b200, D):
    experts = dict(experts=AT, top=2, n_experts=4)
    for change, exc, words in [
            (dict(out_type=2), b200.UnsupportedDType, "type 2"), (dict(scale_type=8), b200.UnsupportedDType, "type 8"), (dict(group=16), b200.Unsupported, "group"), (dict(group=256), b200.Unsupported, "group"),
            (dict(group=128), b200.ShapeMismatch, "multiple"), (dict(k=0), b200.ShapeMismatch, "shape"), (dict(n=0), b200.ShapeMismatch, "shape"), (dict(tokens=-1), b200.ShapeMismatch, "shape"),
            (dict(n=(1 << 31) - 1, ldo=1 << 31), b200.ShapeMismatch, "shape"), (dict(tokens=(1 << 31) - 1), b200.ShapeMismatch, "rows"), (dict(lda=48), b200.ShapeMismatch, "overlap"),
            (dict(ldo=7), b200.ShapeMismatch, "overlap"), (dict(a=AT + 8), b200.InvalidArgument, "16 bytes"), (dict(w=AT + 1), b200.InvalidArgument, "16 bytes"), (dict(lda=72), b200.InvalidArgument, "16 bytes"),
            (dict(w_scales=AT + 8), b200.InvalidArgument, "16 bytes"), (dict(out=None), b200.InvalidArgument, "null"), (dict(w=None), b200.InvalidArgument, "null"), (dict(a_scales=None), b200.InvalidArgument, "null"),
            (dict(top=2), b200.InvalidArgument, "without experts"), (dict(rows_per_pair=1), b200.InvalidArgument, "without experts"), ({**experts, "top": 0}, b200.ShapeMismatch, "places"),
            ({**experts, "top": 33}, b200.ShapeMismatch, "places"), ({**experts, "n_experts": 0}, b200.ShapeMismatch, "places"), ({**experts, "n_experts": 1025}, b200.ShapeMismatch, "places"),
            ({**experts, "tokens": 1 << 30}, b200.ShapeMismatch, "rows")]:
        refused(b200, product(D, **change), exc, words)
    refused(b200, D._lib().b200_dev_mat_mat_i4(None), b200.InvalidArgument, "null")
    assert product(D, tokens=0, a=None) == 0 and product(D, **{**experts, "tokens": 0}) == 0


def test_glu_refusals(b200, D):
    good = dict(device=0, stream=None, type=0, act=0, x=AT, ldx=128, q=AT, ldq=64, scales=AT, rows=2, ff=64)
    for change, exc, words in [(dict(type=9), b200.UnsupportedDType, "type 9"), (dict(act=3), b200.InvalidArgument, "act"), (dict(act=-1), b200.InvalidArgument, "act"), (dict(rows=-1), b200.ShapeMismatch, "rows"),
                               (dict(ff=0), b200.ShapeMismatch, "ff"), (dict(ff=65537, ldq=65537), b200.ShapeMismatch, "ff"), (dict(ldx=-1), b200.ShapeMismatch, "negative"), (dict(ldq=63), b200.ShapeMismatch, "overlap"),
                               (dict(x=None), b200.InvalidArgument, "null"), (dict(scales=None), b200.InvalidArgument, "null")]:
        refused(b200, D._lib().b200_dev_glu_q8(*{**good, **change}.values()), exc, words)
    assert D._lib().b200_dev_glu_q8(*{**good, "rows": 0, "x": None}.values()) == 0


def gated(D, **kw):
    a = D.GatedNorm(device=0, type=0, y=AT, residual=AT + 256, sum=AT + 512, weight=AT, q=AT, scales=AT, ldy=64, ldr=64, lds=64, ldq=64, rows=2, hidden=64, scale=1.0, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return D._lib().b200_dev_add_gated_norm_q8(C.byref(a))


def test_gated_norm_refusals(b200, D):
    for change, exc, words in [
            (dict(type=8), b200.UnsupportedDType, "type 8"), (dict(rows=-1), b200.ShapeMismatch, "rows"), (dict(hidden=0), b200.ShapeMismatch, "hidden"), (dict(hidden=65537, lds=70000, ldq=70000), b200.ShapeMismatch, "hidden"),
            (dict(mix=AT, top=0), b200.ShapeMismatch, "per row"), (dict(mix=AT, top=33), b200.ShapeMismatch, "per row"), (dict(ldy=-1), b200.ShapeMismatch, "negative"), (dict(gate=AT, gate_row=-1), b200.ShapeMismatch, "negative"),
            (dict(lds=63), b200.ShapeMismatch, "overlap"), (dict(ldq=63), b200.ShapeMismatch, "overlap"), (dict(eps=-1.0), b200.InvalidArgument, "eps"), (dict(eps=math.nan), b200.InvalidArgument, "eps"),
            (dict(scale=math.nan), b200.InvalidArgument, "scale"), (dict(y=None), b200.InvalidArgument, "null"), (dict(residual=None), b200.InvalidArgument, "null"), (dict(sum=None), b200.InvalidArgument, "null"),
            (dict(q=None), b200.InvalidArgument, "null"), (dict(sum=AT + 256, lds=65), b200.InvalidArgument, "in place"), (dict(sum=AT), b200.InvalidArgument, "must not be")]:
        refused(b200, gated(D, **change), exc, words)
    refused(b200, D._lib().b200_dev_add_gated_norm_q8(None), b200.InvalidArgument, "null")
    assert gated(D, rows=0, y=None) == 0


def test_python_refusals(b200, D):
    z, f = torch.zeros(4, 8), torch.zeros(4, 64)
    for call, exc in [
            (lambda: D.route_experts(z, 2), b200.InvalidArgument), (lambda: D.route_experts(z.double(), 2), b200.UnsupportedDType), (lambda: D.route_experts(z[0], 2), b200.ShapeMismatch),
            (lambda: D.route_experts(z.T, 2), b200.ShapeMismatch), (lambda: D.route_experts(z, 0), b200.ShapeMismatch), (lambda: D.route_experts(z, 2, score="relu"), b200.InvalidArgument),
            (lambda: D.route_experts(z, 2, score=1), TypeError), (lambda: D.route_experts(z, 2, correction=z[0].half()), b200.DTypeMismatch), (lambda: D.route_experts(z, 2, correction=torch.zeros(7)), b200.ShapeMismatch),
            (lambda: D.route_experts(z, 2, experts=torch.zeros(4, 2)), b200.DTypeMismatch), (lambda: D.route_experts(z, 2, weights=torch.zeros(4, 3)), b200.ShapeMismatch),
            (lambda: D.route_experts(z.clone().requires_grad_(), 2), b200.Unsupported), (lambda: D.route_experts(torch.zeros(1, 2000), 2), b200.ShapeMismatch),
            (lambda: D.glu_q8(f), b200.InvalidArgument), (lambda: D.glu_q8(f[:, :63]), b200.ShapeMismatch), (lambda: D.glu_q8(f, "tanh"), b200.InvalidArgument), (lambda: D.glu_q8(f.int()), b200.UnsupportedDType),
            (lambda: D.glu_q8(f, out=torch.zeros(4, 64, dtype=torch.int8)), b200.ShapeMismatch), (lambda: D.glu_q8(f, scales=torch.zeros(3)), b200.ShapeMismatch)]:
        with pytest.raises(exc):
            call()
    a, s, (w, ws) = torch.zeros(3, 64, dtype=torch.int8), torch.ones(3), D.i4_weights(torch.zeros(20, 64, dtype=torch.int8), torch.ones(20, 2))
    e, we, wse = torch.zeros(3, 2, dtype=torch.int32), w[None].expand(4, *w.shape).contiguous(), ws[None].expand(4, *ws.shape).contiguous()
    for change, exc in [
            (dict(), b200.InvalidArgument), (dict(a=a.float()), b200.DTypeMismatch), (dict(a=a[:, :32]), b200.Unsupported), (dict(a_scales=s[:2]), b200.ShapeMismatch), (dict(w=w.to(torch.int8)), b200.DTypeMismatch),
            (dict(w=w[:, :, :256]), b200.ShapeMismatch), (dict(w=w[:1]), b200.ShapeMismatch), (dict(w_scales=ws[:1]), b200.ShapeMismatch), (dict(w_scales=ws.double()), b200.UnsupportedDType),
            (dict(w_scales=ws.repeat(1, 2, 1, 1)), b200.Unsupported), (dict(n=33), b200.ShapeMismatch), (dict(n=16), b200.ShapeMismatch), (dict(bias=torch.zeros(19)), b200.ShapeMismatch),
            (dict(experts=e), b200.ShapeMismatch), (dict(experts=e.long(), w=we, w_scales=wse), b200.DTypeMismatch), (dict(experts=e[:2], w=we, w_scales=wse), b200.ShapeMismatch),
            (dict(experts=e, w=we, w_scales=wse[:3]), b200.ShapeMismatch), (dict(experts=e.T, w=we, w_scales=wse), b200.ShapeMismatch), (dict(dtype=torch.int8), b200.UnsupportedDType),
            (dict(out=torch.zeros(3, 21)), b200.ShapeMismatch)]:
        with pytest.raises(exc):
            D.mat_mat_i4(**{**dict(a=a, a_scales=s, w=w, w_scales=ws, n=20), **change})
    one = torch.ones(64)
    for change, exc in [
            (dict(), b200.InvalidArgument), (dict(y=f[:3]), b200.ShapeMismatch), (dict(y=f.half()), b200.DTypeMismatch), (dict(weight=one[:63]), b200.ShapeMismatch), (dict(mix=torch.ones(4, 2)), b200.ShapeMismatch),
            (dict(mix=torch.ones(4, 33)), b200.ShapeMismatch), (dict(mix=torch.ones(4)), b200.ShapeMismatch), (dict(post_weight=one.half()), b200.DTypeMismatch), (dict(gate=one), b200.ShapeMismatch),
            (dict(gate=f.half()), b200.DTypeMismatch), (dict(gate=f[:2]), b200.ShapeMismatch), (dict(weight=None, scales=torch.ones(4)), b200.InvalidArgument), (dict(sum_out=f[:, :63]), b200.ShapeMismatch),
            (dict(post_weight=one.clone().requires_grad_()), b200.Unsupported)]:
        with pytest.raises(exc):
            D.add_gated_norm_q8(**{**dict(y=f, residual=f, weight=one, eps=1e-5), **change})
