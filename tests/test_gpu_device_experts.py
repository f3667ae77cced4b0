"""Operators on device tensors for feed-forwards with routed experts and 4-bit weights, against plain forms in 64 bits: routing, 4-bit products, the gated unit, a block's norms."""
import math

import pytest
import torch

import device_experts_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    return device_ops


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


def same_bits(a, b):
    return all(torch.equal(x.contiguous().view(torch.uint8), y.contiguous().view(torch.uint8)) for x, y in zip(a, b))


# ---------------------------------------------------------------------------------------------------------------- routing
def check_route(D, z, top, **kw):
    e, w = D.route_experts(z.cuda() if not z.is_cuda else z, top, **{k: v.cuda() if torch.is_tensor(v) else v for k, v in kw.items()})
    want, ww = R.route(z.cpu(), top, **kw)
    assert e.dtype == torch.int32 and w.dtype == torch.float32
    assert torch.equal(e.cpu(), want)
    assert torch.equal(torch.isnan(w.cpu()), torch.isnan(ww))
    # in 64 bits (2^-45 of it left for exponentials and sums), then rounded once
    assert (torch.nan_to_num((w.cpu().double() - ww).abs()) <= torch.nan_to_num(ww.abs() * (2.0**-24 + 2.0**-45) + 2.0**-150)).all()
    return e, w


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("tokens,n,top", [(1, 1, 1), (1, 8, 2), (3, 2, 2), (5, 31, 4), (7, 32, 32), (2, 33, 8), (9, 60, 4), (6, 64, 6), (5, 100, 7), (3, 128, 8), (4, 200, 10), (5, 256, 8), (3, 257, 5),
                                          (2, 512, 8), (2, 1000, 16), (3, 1024, 32)])
def test_routing(D, dtype, score, tokens, n, top):
    z = (2 * normal(n + tokens, tokens, n)).to(dtype)
    for correction in (None, 0.1 * normal(5, n)):
        for renormalise in (False, True):
            check_route(D, z, top, score=score, correction=correction, renormalise=renormalise, scale=2.5 if renormalise else 1.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("n,groups,top_groups,top", [(8, 8, 3, 3), (8, 2, 1, 4), (16, 4, 4, 16), (60, 12, 5, 6), (64, 8, 3, 6), (96, 3, 2, 5), (160, 8, 3, 6), (256, 8, 4, 8), (256, 32, 5, 8), (252, 4, 2, 9),
                                                     (512, 16, 4, 12), (1024, 32, 32, 32), (1024, 2, 1, 8), (992, 31, 7, 8)])
def test_routing_by_groups(D, dtype, n, groups, top_groups, top):
    z = (2 * normal(n + groups, 6, n)).to(dtype)
    for score in ("softmax", "sigmoid"):
        for correction in (None, 0.2 * normal(5, n)):
            check_route(D, z, top, score=score, correction=correction, groups=groups, top_groups=top_groups)


@pytest.mark.parametrize("n,groups", [(24, 1), (24, 4), (300, 1), (300, 6), (256, 8)])
def test_routing_among_equals(D, n, groups):
    """Few different logits: the lower number first, among experts and among groups."""
    z = normal(1, 40, n).round()
    z[3] = 0
    z[4, ::2] = -0.0
    z[5] = 1.5
    for score in ("softmax", "sigmoid"):
        for correction in (None, normal(2, n).round() / 4, torch.zeros(n)):
            if score == "softmax" and correction is not None and correction.any():
                continue      # (sums of unlike scores: equal only up to rounding)
            check_route(D, z, 7, score=score, correction=correction, groups=groups, top_groups=max(1, groups // 2))


def test_routing_of_scores_next_to_one_another(D):
    """Scores that f32 does not tell apart: 64 bits do.  Sigmoids near 1, corrections that differ in their last bits, groups whose sums are that near."""
    z = torch.full((4, 64), 17.0)
    z[0] += torch.arange(64) * 2.0**-19
    z[1] -= torch.arange(64) * 2.0**-19
    z[2] = torch.where(torch.arange(64) % 2 == 0, 18.0, 18.0 + 2.0**-19)
    z[3] = 20 + normal(3, 64)
    check_route(D, z, 8, score="sigmoid")
    check_route(D, z, 8, score="sigmoid", correction=torch.full((64,), 0.25))
    check_route(D, z, 8, score="sigmoid", correction=torch.full((64,), 0.25), groups=8, top_groups=3)
    check_route(D, z, 8, score="sigmoid", groups=8, top_groups=3)
    check_route(D, z, 8, correction=torch.full((64,), 1000.0), groups=8, top_groups=3)


@pytest.mark.parametrize("groups", [1, 5])
def test_routing_where_little_is_left(D, groups):
    z = normal(7, 12, 40)
    z[0] = -math.inf
    z[1, 1:] = -math.inf
    z[2, :38] = -math.inf
    z[3, 5] = math.nan
    z[4] = math.nan
    z[5, 7] = math.inf
    z[6, 8:] = -math.inf
    z[7] = -1e30
    z[8] = 1e30 * normal(1, 40)
    z[9, :20] = 3e38
    for score in ("softmax", "sigmoid"):
        for renormalise in (False, True):
            check_route(D, z, 6, score=score, groups=groups, top_groups=max(1, groups - 2), renormalise=renormalise)
    c = normal(8, 40)
    c[0], c[3], c[11] = -math.inf, math.nan, math.inf
    z = z[[0, 1, 2, 6, 7, 10, 11]]
    for score in ("softmax", "sigmoid"):
        check_route(D, z, 6, score=score, groups=groups, top_groups=max(1, groups - 2), correction=c)


def test_routing_of_rows_apart_and_into_tensors(D):
    wide = normal(1, 9, 300).cuda()
    e, w = torch.full((9, 3), 77, dtype=torch.int32).cuda(), torch.zeros(9, 3).cuda()
    got = D.route_experts(wide[:, 11:99], 3, experts=e, weights=w)
    assert got[0].data_ptr() == e.data_ptr() and got[1].data_ptr() == w.data_ptr()
    want = D.route_experts(wide[:, 11:99].contiguous(), 3)
    assert same_bits(got, want)
    assert same_bits(D.route_experts(wide[:1, 11:99].expand(4, 88), 3), [v[:1].expand(4, 3) for v in want])
    e, w = D.route_experts(wide[:0], 3)
    assert e.shape == (0, 3) and w.shape == (0, 3)


def test_routing_of_many_tokens(D):
    z = 2 * normal(3, 3001, 72)
    check_route(D, z.bfloat16(), 6, score="sigmoid", correction=0.1 * normal(4, 72), groups=9, top_groups=3)


# ----------------------------------------------------------------------------------------------------------------- product
def bytes_of(seed, rows, k, extra=0):
    g = torch.Generator().manual_seed(seed)
    return torch.randint(-128, 128, (rows, (k + 15) // 16 * 16 + extra), generator=g, dtype=torch.int8).cuda()[:, :k]      # (what lies behind a row is not zero)


def four_bits(seed, *shape):
    return torch.randint(-8, 8, shape, generator=torch.Generator().manual_seed(seed), dtype=torch.int8)


def check_product(D, a, values, scales, dtype, experts=None, bias=None, **kw):
    s = 0.01 + torch.rand(len(a), generator=torch.Generator().manual_seed(1))
    w, ws = D.i4_weights(values, scales)
    n = values.shape[-2]
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    y = D.mat_mat_i4(a, s.cuda(), w.cuda(), ws.cuda(), n=n, experts=cuda(experts), bias=cuda(bias), dtype=dtype, **kw)
    want, off = R.product(a.cpu(), s, values, scales, experts, bias)
    assert y.dtype == dtype and y.shape == want.shape
    tol = off + R.HALF_STEP[dtype] * 1.001 * (want.abs() + off) + R.LEAST[dtype]
    assert ((y.cpu().double() - want).abs() <= tol).all(), float(((y.cpu().double() - want).abs() - tol).max())
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,k,n,group", [(1, 32, 1, 32), (1, 64, 16, 64), (1, 128, 17, 128), (2, 96, 33, 32), (7, 192, 100, 64), (8, 384, 15, 128), (9, 4096, 48, 32), (1, 4096, 300, 128), (16, 1056, 64, 32),
                                            (17, 832, 130, 64), (33, 640, 65, 128), (40, 2048, 31, 64), (64, 288, 257, 32), (65, 512, 40, 32), (130, 256, 72, 128), (1, 14336, 40, 32), (3, 64, 2000, 32)])
def test_product(D, dtype, rows, k, n, group):
    scales = (0.001 + 0.01 * torch.rand(n, k // group, generator=torch.Generator().manual_seed(2))).to(TYPES[(rows + n) % 3])
    check_product(D, bytes_of(rows, rows, k), four_bits(k, n, k), scales, dtype, bias=normal(3, n) if n % 2 else None)


@pytest.mark.parametrize("k,group", [(224, 32), (32, 32), (96, 32), (160, 32), (192, 64), (64, 64), (384, 128), (480, 32), (1248, 32)])
@pytest.mark.parametrize("rows", [1, 2, 4, 8, 16, 20, 64])
@pytest.mark.parametrize("experts", [0, 3])
def test_product_reads_nothing_behind_its_operands(D, k, group, rows, experts):
    """NaN scales behind the last tile's, numbers behind the rows' channels and in a last tile's unused channels: none of them counts."""
    n, E = 21, max(1, experts)
    values, scales = four_bits(k, E, n, k), 0.01 * normal(2, E, n, k // group).abs() + 0.001
    w, ws = D.i4_weights(values, scales)
    if k % 64:
        w = w.unflatten(-1, (8, 4, 2, 2, 4)).clone()
        w[:, :, -1, :, :, 1] = 0x5A      # (channels 32 to 63 of the last tile)
        w = w.flatten(3)
    behind = lambda t, v: torch.cat([t.flatten(), torch.full((4096,), v, dtype=t.dtype)]).cuda()[: t.numel()].view(t.shape)  # noqa: E731
    w, ws = behind(w, 0x77), behind(ws, math.nan)
    a = bytes_of(3, rows, k, extra=16)
    s, e = torch.ones(rows), chosen(4, rows, 1, E) if experts else None
    y = D.mat_mat_i4(a, s.cuda(), w if experts else w[0], ws if experts else ws[0], n=n, experts=None if e is None else e.cuda(), dtype=torch.float32)
    want, off = R.product(a.cpu(), s, values if experts else values[0], scales if experts else scales[0], e)
    assert ((y.cpu().double() - want).abs() <= off + 2.0**-24 * want.abs()).all()


@pytest.mark.parametrize("scale", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [1, 12, 33, 70])
def test_product_of_every_kind_of_scale(D, scale, group, rows):
    scales = (0.01 * normal(5, 90, 768 // group)).to(scale)      # (of either sign)
    check_product(D, bytes_of(3, rows, 768), four_bits(4, 90, 768), scales, torch.float32)


@pytest.mark.parametrize("rows", [1, 8, 40])
def test_product_of_the_largest_numbers(D, rows):
    """128 products of -128 and -8: 2^17 in a group."""
    a = torch.full((rows, 512), -128, dtype=torch.int8).cuda()
    for group in (32, 64, 128):
        for v in (-8, 7):
            check_product(D, a, torch.full((20, 512), v, dtype=torch.int8), torch.ones(20, 512 // group), torch.float32)
    a[:, ::2] = 127
    check_product(D, a, four_bits(1, 20, 512), torch.ones(20, 4).half(), torch.float32)


@pytest.mark.parametrize("rows", [1, 8, 40])
def test_product_of_rows_with_the_smallest_scales(D, rows):
    """A row's scale of 2^-126 and a little more has all its bits; the weights' large ones bring the result back."""
    values, scales = four_bits(1, 20, 256), 2.0**100 * (1 + torch.rand(20, 8, generator=torch.Generator().manual_seed(2)))
    a, s = bytes_of(2, rows, 256), 2.0**-126 * (1 + torch.rand(rows, generator=torch.Generator().manual_seed(3)))
    w, ws = (v.cuda() for v in D.i4_weights(values, scales))
    y = D.mat_mat_i4(a, s.cuda(), w, ws, n=20, dtype=torch.float32)
    want, off = R.product(a.cpu(), s, values, scales)
    assert ((y.cpu().double() - want).abs() <= off + 2.0**-24 * want.abs()).all()


def test_product_of_many_rows(D):
    check_product(D, bytes_of(1, 1001, 160), four_bits(2, 200, 160), 0.01 * normal(3, 200, 5), torch.float32, bias=normal(4, 200))


def test_product_of_rows_apart_and_into_tensors(D):
    values, scales = four_bits(1, 50, 320), 0.01 * normal(2, 50, 10)
    a = bytes_of(3, 11, 320, extra=48)
    y = check_product(D, a, values, scales, torch.float16)
    into = torch.full((11, 77), 5.0, dtype=torch.float16).cuda()
    z = check_product(D, a, values, scales, torch.float16, out=into[:, 9:59])
    assert torch.equal(y, z) and (into[:, :9] == 5).all() and (into[:, 59:] == 5).all()
    w, ws = (v.cuda() for v in D.i4_weights(values, scales))
    one = D.mat_mat_i4(a, torch.ones(11).cuda(), w, ws, dtype=torch.float32)
    assert one.shape == (11, 64) and (one[:, 50:] == 0).all()      # (without n: all rows of the tiles)
    assert torch.equal(D.mat_mat_i4(a[:1].expand(5, 320).contiguous(), torch.ones(5).cuda(), w, ws, dtype=torch.float32), one[:1].expand(5, 64))
    assert D.mat_mat_i4(a[:0], torch.ones(0).cuda(), w, ws).shape == (0, 64)


def test_product_of_a_row_is_the_same_among_others(D):
    """A row's result does not depend on what is in the rows beside it, nor on its place (another number of rows may be another kernel, whose sums have another order)."""
    values, scales = four_bits(1, 70, 1024), (0.01 * normal(2, 70, 32)).half()
    w, ws = (v.cuda() for v in D.i4_weights(values, scales))
    for rows in (2, 4, 8, 16, 32, 64):
        a = bytes_of(3, rows, 1024)
        whole = D.mat_mat_i4(a, torch.ones(rows).cuda(), w, ws, dtype=torch.float32)
        for i in (0, rows // 2, rows - 1):
            b = bytes_of(4 + i, rows, 1024)
            b[rows - 1 - i] = a[i]
            assert torch.equal(D.mat_mat_i4(b, torch.ones(rows).cuda(), w, ws, dtype=torch.float32)[rows - 1 - i], whole[i])


def chosen(seed, tokens, top, n, empty=0.0):
    g = torch.Generator().manual_seed(seed)
    e = torch.stack([torch.randperm(n, generator=g)[:top] for _ in range(tokens)]).int()
    e[torch.rand(tokens, top, generator=g) < empty] = -1
    return e


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,top,experts,k,n,group", [(1, 2, 8, 256, 40, 32), (1, 1, 1, 64, 16, 64), (4, 2, 8, 384, 33, 128), (16, 2, 8, 512, 100, 32), (33, 4, 5, 128, 48, 64), (64, 2, 3, 96, 20, 32),
                                                          (20, 8, 64, 128, 17, 32), (150, 6, 10, 64, 24, 32), (9, 3, 300, 64, 16, 64), (5, 32, 40, 64, 8, 32)])
@pytest.mark.parametrize("own_rows", [False, True])
def test_product_of_experts(D, dtype, tokens, top, experts, k, n, group, own_rows):
    scales = (0.001 + 0.01 * torch.rand(experts, n, k // group, generator=torch.Generator().manual_seed(2))).to(TYPES[tokens % 3])
    check_product(D, bytes_of(tokens, tokens * top if own_rows else tokens, k), four_bits(k, experts, n, k), scales, dtype, experts=chosen(1, tokens, top, experts, 0.2 if tokens > 4 else 0.0),
                  bias=normal(4, experts, n) if n % 2 == 0 else None)


def test_product_of_experts_at_odd_places(D):
    values, scales = four_bits(1, 6, 30, 128), 0.01 * normal(2, 6, 30, 4)
    a = bytes_of(3, 10, 128)
    e = chosen(5, 10, 2, 6)
    e[:] = 5
    check_product(D, a, values, scales, torch.float32, experts=e)      # one expert, twice for each token
    e[:] = -1
    assert (check_product(D, a, values, scales, torch.float32, experts=e) == 0).all()
    e = chosen(5, 10, 2, 6)
    e[2, 0], e[3, 1], e[9, 0] = 6, -2, 2**31 - 1      # (no experts: zeros, and the status says so)
    status = torch.zeros(1, dtype=torch.int32).cuda()
    y = check_product(D, a, values, scales, torch.float32, experts=e, status=status)
    assert (y[[4, 7, 18]] == 0).all() and int(status) == D.STATUS_BAD_EXPERT
    status.zero_()
    check_product(D, a, values, scales, torch.float32, experts=chosen(5, 10, 2, 6, 0.5), status=status)
    assert int(status) == 0
    w, ws = (v.cuda() for v in D.i4_weights(values, scales))
    assert D.mat_mat_i4(a[:0], torch.ones(0).cuda(), w, ws, experts=e[:0].cuda()).shape == (0, 32)


@pytest.mark.parametrize("top,own_rows", [(3, False), (3, True), (1, False), (32, False)])
def test_product_of_experts_of_many_tokens(D, top, own_rows):
    """More pairs than a launch lists."""
    tokens = 9001 // top
    values, scales = four_bits(1, 40, 16, 64), 0.01 * normal(2, 40, 16, 2)
    check_product(D, bytes_of(3, tokens * top if own_rows else tokens, 64), values, scales, torch.float32, experts=chosen(5, tokens, top, 40, 0.1))


def test_product_of_weights_behind_two_gigabytes(D):
    n, k, E = 16384, 8192, 40      # 64 MiB for each expert's weights, 2.5 GiB for all
    w = torch.zeros(E, n // 16, k // 64, 512, dtype=torch.uint8, device="cuda")
    ws = torch.ones(E, n // 16, k // 128, 8, 2, device="cuda", dtype=torch.float16)
    values = four_bits(1, n, k)
    for e in (0, 39):
        w[e] = D.i4_weights(values.cuda(), torch.ones(n, k // 128, dtype=torch.float16).cuda())[0]
    a = bytes_of(2, 2, k)
    y = D.mat_mat_i4(a, torch.ones(2).cuda(), w, ws, experts=torch.tensor([[39, 3], [0, 39]], dtype=torch.int32).cuda(), dtype=torch.float32)
    want = a.double() @ values.double().cuda().T      # (below 2^24: exact)
    assert torch.equal(y.double(), torch.stack([want[0], 0 * want[0], want[1], want[1]]))


def test_weights_from_values_and_from_blocks(D):
    x = normal(1, 3, 50, 192)
    for group, dtype in ((32, torch.float16), (64, torch.bfloat16)):
        w, ws = D.quantise_i4(x.cuda(), group, dtype)
        back = D.read_i4(w, ws, 50, 192).cpu()
        step = x.unflatten(-1, (-1, group)).abs().amax(-1, keepdim=True) / 8
        # half a step, one where the value of the other sign is as large (7 for 8), and the scale's rounding of 8 of them
        assert ((back - x).unflatten(-1, (-1, group)).abs() <= step * (1 + 8 * R.HALF_STEP[dtype] * 1.01)).all()
    a = bytes_of(2, 4, 192)
    y = D.mat_mat_i4(a, torch.ones(4).cuda(), w[1], ws[1], n=50, dtype=torch.float32)
    want = a.double().cpu() @ back[1].double().T
    assert ((y.cpu().double() - want).abs() <= (a.double().cpu().abs() @ back[1].double().abs().T) * 20 * 2.0**-24).all()


# ------------------------------------------------------------------------------------------------------------- gated unit
def check_glu(D, x, act, **kw):
    q, s = D.glu_q8(x, act, **kw)
    y = R.glu(x.cpu(), act)
    top = y.abs().amax(1, keepdim=True)
    assert q.dtype == torch.int8 and s.dtype == torch.float32
    # one rounding of a number made in 64 bits; the numbers as if y were exact (2^-40: 64-bit exponentials)
    live = top >= R.TINY
    step = torch.where(live, top, 0.0)[:, 0] / 127
    assert ((s.cpu().double() - step).abs() <= step * (2.0**-24 + 2.0**-40)).all()
    t = torch.where(live, y * 127 / torch.where(live, top, 1.0), 0.0)
    assert ((q.cpu().double() - t).abs() <= 0.5 + 127 * 2.0**-40).all(), float((q.cpu().double() - t).abs().max())
    return q, s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("rows,ff", [(1, 1), (1, 14336), (3, 31), (5, 896), (2, 2001), (17, 2048), (4, 8192), (300, 136), (2, 16384), (1, 28672), (1, 40000), (2, 65536), (700, 64)])
def test_gated_unit(D, dtype, act, rows, ff):
    check_glu(D, (2 * normal(rows + ff, rows, 2 * ff)).to(dtype).cuda(), act)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_unit_of_rows_apart_and_into_tensors(D, dtype):
    wide = normal(1, 9, 700).to(dtype).cuda()
    for x in (wide[:, 100:612], wide[:, 3:517], wide[:1].expand(9, 700)[:, 8:520]):
        q, s = check_glu(D, x, "silu")
        into, scales = torch.full((9, 400), 77, dtype=torch.int8).cuda(), torch.zeros(9).cuda()
        n = q.shape[1]
        D.glu_q8(x, "silu", out=into[:, 5 : 5 + n], scales=scales)
        assert torch.equal(into[:, 5 : 5 + n], q) and torch.equal(scales, s) and (into[:, :5] == 77).all() and (into[:, 5 + n :] == 77).all()
    assert D.glu_q8(wide[:0, :64])[0].shape == (0, 32)


def test_gated_unit_of_rows_that_are_zero_tiny_or_not_finite(D):
    x = normal(1, 9, 520)
    x[1] = 0
    x[2, :260], x[2, 260:] = 2.0**-70, 2.0**-70
    x[3, 5] = math.inf
    x[4, 259] = math.nan
    x[5, 300] = -math.inf
    x[6] *= 1e19      # (products up to 1e38)
    x[7, :260] = -90 - 10 * normal(2, 260).abs()      # (exponentials beyond f32)
    x[8, :260] = -20 - 10 * normal(3, 260).abs()
    for act in ("silu", "gelu", "relu"):
        q, s = (v.cpu() for v in D.glu_q8(x.cuda(), act))
        assert (q[3:6] == 0).all() and torch.isnan(s[3:6]).all()
        assert (q[1:3] == 0).all() and (s[1:3] == 0).all()
        check_glu(D, x[[0, 6, 7, 8]].cuda(), act)
    with_nan = x[:1].clone()
    with_nan[0, 3] = math.nan
    assert torch.isnan(D.glu_q8(with_nan.cuda(), "relu")[1]).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_unit_halves_to_even(D, dtype):
    """Exact values half way between two numbers: relu(g) * u with a largest value of 127."""
    for ff in (256, 301):
        g = torch.ones(2, ff)
        u = (torch.arange(ff) % 253 - 126).float() + 0.5
        u[0] = 127
        x = torch.cat([g, u.expand(2, ff)], 1).to(dtype)      # (all of them bf16 numbers)
        assert torch.equal(x.float()[:, ff:], u.expand(2, ff))
        q, s = D.glu_q8(x.cuda(), "relu")
        assert torch.equal(q.cpu().float(), torch.round(u).expand(2, ff)) and (s == 1).all()


# ------------------------------------------------------------------------------------------------------------ gated norm
def check_gated(D, y, res, w, eps, mix=None, post_weight=None, gate=None, scale=1.0, **kw):
    cuda = lambda t: None if t is None else t.cuda()  # noqa: E731
    first = res.cpu().clone()
    q, s, r = D.add_gated_norm_q8(cuda(y), cuda(res), cuda(w), eps, mix=cuda(mix), post_weight=cuda(post_weight), gate=cuda(gate), scale=scale, **kw)
    t = res.dtype
    want, off = R.gated(y.cpu(), first, eps, mix, post_weight, gate, scale)
    assert r.dtype == t
    tol = off + R.HALF_STEP[t] * 1.001 * (want.abs() + off) + R.LEAST[t]
    assert ((r.cpu().double() - want).abs() <= tol).all(), float(((r.cpu().double() - want).abs() - tol).max())
    if w is None:
        assert q is None and s is None
        return q, s, r
    n = r.cpu().double()
    n = n * (1 / (n.square().mean(1, keepdim=True) + float(torch.tensor(eps))).sqrt()) * w.double()
    top = n.abs().amax(1)
    # rstd, two products: 3 half steps; the division 1
    assert ((s.cpu().double() - top / 127).abs() <= 4.01 * 2.0**-24 * top / 127).all()
    step = torch.where(top > 0, top / 127, 1.0)[:, None]
    # the quotient: 3 (y) + 4 (127 / m) + 1 half steps of at most 127, around the half that rounding takes
    assert ((q.cpu().double() - n / step).abs() <= 0.5 + 127 * 8.1 * 2.0**-24).all()
    return q, s, r


def gates(t, rows, n):
    g = torch.sigmoid(normal(9, rows, n)).to(t)
    return {"none": None, "each": g, "token": g[:, :1], "channel": g[:1], "expanded": g[:1].expand(rows, n), "one": g[:1, :1]}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 4096), (3, 31), (5, 896), (2, 2001), (17, 2048), (4, 8192), (300, 136), (2, 16384), (1, 40000), (1, 65536), (400, 1024)])
@pytest.mark.parametrize("mix,post,gate", [(0, True, "channel"), (2, True, "none"), (3, False, "token"), (8, True, "each"), (0, False, "none"), (1, True, "one")])
def test_gated_norm(D, dtype, rows, hidden, mix, post, gate):
    y, res = normal(1, rows * max(1, mix), hidden).to(dtype), (5 * normal(2, rows, hidden)).to(dtype)
    check_gated(D, y, res, 1 + 0.2 * normal(3, hidden), 1e-5, mix=torch.softmax(normal(4, rows, mix), 1) if mix else None, post_weight=1 + 0.2 * normal(5, hidden) if post else None,
                gate=gates(dtype, rows, hidden)[gate], scale=0.3 if rows % 2 else 1.0)


@pytest.mark.parametrize("dtype", TYPES)
def test_gated_norm_of_rows_apart_and_in_place(D, dtype):
    wide, res = normal(1, 18, 700).to(dtype).cuda(), normal(2, 9, 513).to(dtype).cuda()
    w, post, mix = 1 + 0.2 * normal(7, 513), 1 + 0.1 * normal(8, 513), torch.softmax(normal(4, 9, 2), 1)
    for gate in gates(dtype, 9, 513).values():
        a = check_gated(D, wide[:, 100:613], res, w, 1e-6, mix=mix, post_weight=post, gate=gate)
        keep = res.clone()
        b = D.add_gated_norm_q8(wide[:, 100:613], keep, w.cuda(), 1e-6, mix=mix.cuda(), post_weight=post.cuda(), gate=None if gate is None else gate.cuda(), sum_out=keep)
        assert b[2].data_ptr() == keep.data_ptr() and same_bits(a, b)
        into, out = torch.full((9, 600), 77, dtype=torch.int8).cuda(), torch.full((9, 600), 7.0, dtype=dtype).cuda()
        c = D.add_gated_norm_q8(wide[:, 100:613], res, w.cuda(), 1e-6, mix=mix.cuda(), post_weight=post.cuda(), gate=None if gate is None else gate.cuda(), out=into[:, 3:516], sum_out=out[:, 5:518])
        assert same_bits(a, c) and (into[:, :3] == 77).all() and (into[:, 516:] == 77).all() and (out[:, :5] == 7).all() and (out[:, 518:] == 7).all()
    wide_gate = torch.sigmoid(normal(6, 513, 9)).to(dtype)
    check_gated(D, wide[:9, 8:521], res, w, 1e-6, gate=wide_gate.T)      # (a gate whose channels are apart)
    check_gated(D, wide[:1, 8:521].expand(9, 513), res, w, 1e-6, post_weight=post)
    assert D.add_gated_norm_q8(wide[:0, :513], res[:0], w.cuda(), 1e-6)[0].shape == (0, 513)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hidden", [64, 1024, 33])
def test_gated_norm_without_the_next_norm(D, dtype, hidden):
    y, res = normal(1, 10, hidden).to(dtype), normal(2, 5, hidden).to(dtype)
    check_gated(D, y, res, None, 1e-5, mix=torch.rand(5, 2), post_weight=normal(3, hidden), gate=gates(dtype, 5, hidden)["each"], scale=-2.0)


@pytest.mark.parametrize("hidden", [260, 257])
def test_gated_norm_of_rows_that_are_zero_tiny_or_not_finite(D, hidden):
    y, res, one = normal(1, 6, hidden), normal(2, 6, hidden), torch.ones(hidden)
    y[1] = 0
    y[2] = res[2] = 2.0**-140
    y[3, 5] = math.inf
    res[4, hidden - 1] = math.nan
    y[5] *= 1e18
    q, s, r = (v.cpu() for v in D.add_gated_norm_q8(y.cuda(), res.cuda(), one.cuda(), 1e-6, post_weight=one.cuda()))
    assert (q[3:5] == 0).all() and torch.isnan(s[3:5]).all() and not torch.isnan(s[[0, 1, 2, 5]]).any()
    assert torch.equal(r[1], res[1])
    check_gated(D, y[[0, 1, 5]], res[[0, 1, 5]], one, 1e-6, post_weight=one)
    q, s, r = D.add_gated_norm_q8(torch.zeros(2, hidden).cuda(), torch.zeros(2, hidden).cuda(), one.cuda(), 1e-6, post_weight=one.cuda())
    assert (q == 0).all() and (s == 0).all() and (r == 0).all()


# ---------------------------------------------------------------------------------------------------------------- together
def sublayer(D, s):
    """A feed-forward sublayer with routed experts as a server runs it: norm, router, experts' gate and up, gated unit, experts' down, their sum onto the stream, the next norm."""
    a, sa, r = D.add_rms_norm_q8(s["x"], s["w1"], 1e-5, residual=s["r"])
    logits = D.mat_mat_i8(a, sa, s["wr"], s["sr"], dtype=torch.float32)
    experts, weights = D.route_experts(torch.where(s["live"][:, None], logits, -math.inf), 2, score="sigmoid", correction=s["correction"], scale=1.5)
    h = D.mat_mat_i4(a, sa, s["up"], s["sup"], experts=experts, dtype=s["x"].dtype)
    b, sb = D.glu_q8(h)
    y = D.mat_mat_i4(b, sb, s["down"], s["sdown"], experts=experts, dtype=s["x"].dtype)
    q, sq, r = D.add_gated_norm_q8(y, r, s["w2"], 1e-5, mix=weights, post_weight=s["w3"], gate=s["gate"], scale=0.5)
    return q, sq, r, experts, weights, h, y


def sublayer_state(D, dtype, tokens, hidden=256, ff=320, experts=8):
    up, sup = D.quantise_i4(0.05 * normal(1, experts, 2 * ff, hidden))
    down, sdown = D.quantise_i4(0.05 * normal(2, experts, hidden, ff), 64)
    s = dict(x=normal(3, tokens, hidden).to(dtype), r=(3 * normal(4, tokens, hidden)).to(dtype), w1=1 + 0.1 * normal(5, hidden), w2=1 + 0.1 * normal(6, hidden), w3=1 + 0.1 * normal(7, hidden),
             wr=torch.randint(-127, 128, (experts, hidden), dtype=torch.int8, generator=torch.Generator().manual_seed(8)), sr=torch.full((experts,), 0.001), correction=0.1 * normal(9, experts),
             up=up, sup=sup, down=down, sdown=sdown, gate=torch.sigmoid(normal(10, 1, hidden)).to(dtype), live=torch.arange(tokens) % 5 != 3)
    return {k: v.cuda() for k, v in s.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens", [1, 6, 40])
def test_a_sublayer(D, dtype, tokens):
    """The chain against its plain form, each step from the kernels' own inputs so that no rounding decides otherwise than theirs."""
    s = sublayer_state(D, dtype, tokens)
    c = {k: v.cpu() for k, v in s.items()}
    q, sq, r, experts, weights, h, y = (v.cpu() for v in sublayer(D, s))
    a, sa, r0 = (v.cpu() for v in D.add_rms_norm_q8(s["x"], s["w1"], 1e-5, residual=s["r"]))
    logits = (a.double() @ c["wr"].double().T * sa.double()[:, None] * c["sr"].double()).float()
    logits[~c["live"]] = -math.inf
    want, ww = R.route(logits, 2, score="sigmoid", correction=c["correction"], scale=1.5)
    assert torch.equal(experts, want) and (weights.double() - ww).abs().max() < 1e-5 and (experts[~c["live"]] == -1).all()
    pair = experts.flatten().long().clamp(min=0)
    none = experts.flatten() < 0
    wide = D.read_i4(c["up"], c["sup"], 640, 256).double()[pair]
    x = (a.double() * sa.double()[:, None]).repeat_interleave(2, 0)
    hh = torch.einsum("pnk,pk->pn", wide, x).masked_fill_(none[:, None], 0)
    room = torch.einsum("pnk,pk->pn", wide.abs(), x.abs()) * 20 * 2.0**-24
    assert ((h.double() - hh).abs() <= room + R.HALF_STEP[dtype] * 1.01 * (hh.abs() + room) + R.LEAST[dtype]).all()
    b, sb = (v.cpu() for v in D.glu_q8(h.cuda()))
    wide = D.read_i4(c["down"], c["sdown"], 256, 320).double()[pair]
    x = b.double() * sb.double()[:, None]
    yy = torch.einsum("pnk,pk->pn", wide, x).masked_fill_(none[:, None], 0)
    room = torch.einsum("pnk,pk->pn", wide.abs(), x.abs()) * 20 * 2.0**-24
    assert ((y.double() - yy).abs() <= room + R.HALF_STEP[dtype] * 1.01 * (yy.abs() + room) + R.LEAST[dtype]).all()
    rr, off = R.gated(y, r0, 1e-5, weights, c["w3"], c["gate"], 0.5)
    assert ((r.double() - rr).abs() <= off + R.HALF_STEP[dtype] * 1.001 * (rr.abs() + off) + R.LEAST[dtype]).all()
    assert torch.equal(r[~c["live"]], r0[~c["live"]])      # (places without a token: nothing is added)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_sublayer_captured_and_replayed(D, dtype):
    """Two graphs of different batches, captured one after the other, replayed in turn on two streams with new inputs: each as without a graph."""
    states = [sublayer_state(D, dtype, 3), sublayer_state(D, dtype, 40)]
    graphs, outs = [], []
    for s in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            sublayer(D, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(sublayer(D, s))
        graphs.append(g)
    for turn in range(3):
        for s in states:
            s["x"].copy_(normal(100 + turn, *s["x"].shape))
        want = [[v.clone() for v in sublayer(D, s)] for s in states]
        torch.cuda.synchronize()
        streams = [torch.cuda.Stream(), torch.cuda.Stream()]
        for _ in range(5):
            for g, st in zip(graphs, streams):
                with torch.cuda.stream(st):
                    g.replay()
        torch.cuda.synchronize()
        assert all(same_bits(o, w) for o, w in zip(outs, want))


def test_two_calls_at_once_on_other_streams(D):
    states = [sublayer_state(D, torch.bfloat16, 3), sublayer_state(D, torch.float32, 40)]
    want = [[v.clone() for v in sublayer(D, s)] for s in states]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in states], [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(sublayer(D, s))
    torch.cuda.synchronize()
    assert all(same_bits(r, w) for g, w in zip(got, want) for r in g)


def test_calls_from_two_threads(D):
    import threading

    s = sublayer_state(D, torch.float16, 20)
    want = [v.clone() for v in sublayer(D, s)]
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                r = sublayer(D, s)
                torch.cuda.current_stream().synchronize()
                if not same_bits(r, want):
                    wrong.append(1)

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


def test_a_device_that_is_not_the_current_one(D):
    if torch.cuda.device_count() < 2:
        pytest.skip("one GPU")
    s = {k: v.to("cuda:1") for k, v in sublayer_state(D, torch.bfloat16, 9).items()}
    with torch.cuda.device(1):
        want = [v.clone() for v in sublayer(D, s)]
    assert torch.cuda.current_device() == 0
    assert same_bits(sublayer(D, s), want) and torch.cuda.current_device() == 0


def test_the_same_bits_every_time(D):
    s = sublayer_state(D, torch.bfloat16, 40)
    one = [v.clone() for v in sublayer(D, s)]
    for _ in range(5):
        assert same_bits(one, sublayer(D, s))
