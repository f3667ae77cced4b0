"""Operators on device tensors for feed-forwards with routed experts and 4-bit weights where their kernels' places end: rings that go round, rows that fill no block of columns, magnitudes at the ends of f32."""
import pytest
import torch

import device_experts_ref as R
from test_gpu_device_experts import bytes_of, check_glu, check_route, four_bits, normal

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    return device_ops


def product64(a, s, values, scales, experts=None):
    """device_experts_ref.product's result and bound, in matrix products of 64 bits on the device (values [experts, n, k], a row of a for each pair)."""
    groups = scales.shape[-1]
    flat = torch.zeros(len(a), dtype=torch.int64) if experts is None else experts.flatten().long()
    y, off = (torch.zeros(len(flat), values.shape[1], dtype=torch.float64, device="cuda") for _ in range(2))
    for e in flat[flat >= 0].unique().tolist():      # (expert -1: zeros)
        rows = (flat == e).nonzero()[:, 0].cuda()
        w, d = values[e].cuda().unflatten(1, (groups, -1)).double(), scales[e].cuda().double()
        x = a[rows].unflatten(1, (groups, -1)).double()
        for g in range(groups):
            term = (x[:, g] @ w[:, g].T) * d[:, g] * s[rows].double()[:, None]      # (the product: integers below 2^24, exact)
            y[rows] += term
            off[rows] += term.abs() * (groups + 10) * 2.0**-24
    return y, off


def check_product(D, rows, k, n, group, scale=torch.float16, experts=None, n_experts=1):
    values = four_bits(k + n, n_experts, n, k)
    scales = (0.01 * normal(2, n_experts, n, k // group)).to(scale)
    w, ws = (v.cuda() for v in D.i4_weights(values.cuda(), scales.cuda()))
    a, s = bytes_of(rows, rows, k), (0.01 + torch.rand(rows, generator=torch.Generator().manual_seed(1))).cuda()
    y = D.mat_mat_i4(a, s, w if experts is not None else w[0], ws if experts is not None else ws[0], n=n, experts=None if experts is None else experts.cuda(), dtype=torch.float32)
    want, off = product64(a, s, values, scales, experts)
    assert y.shape == want.shape and ((y.double() - want).abs() <= off + 2.0**-24 * (want.abs() + off)).all()


@pytest.mark.parametrize("scale", TYPES)
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("rows", [49, 50, 55, 56, 57])
def test_product_of_rows_that_fill_seven_blocks_of_columns(D, scale, group, rows):
    """Eight blocks are computed for them, over more steps than a ring has."""
    check_product(D, rows, 14336, 200, group, scale)


@pytest.mark.parametrize("rows,one", [(50, 50), (56, 56), (60, 52), (114, 114)])
def test_product_of_an_expert_that_has_seven_blocks_of_rows(D, rows, one):
    experts = torch.zeros(rows, 1, dtype=torch.int32)
    experts[one:] = 1
    check_product(D, rows, 14336, 300, 64, experts=experts, n_experts=2)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("ff", [1024, 1023, 8200, 8199])
def test_gated_unit_of_gates_below_the_normal_numbers(D, dtype, act, ff):
    """Gates of some 2^-149 (bf16: 2^-133), whose halves have few bits, and ups that bring them back."""
    g = torch.Generator().manual_seed(ff)
    least = 2.0**-149 if dtype == torch.float32 else 2.0**-133
    for most, up in ((1023, 2.0**60), (31, 2.0**100), (3, 2.0**40), (2**20 - 1, 2.0**50)):
        most = most if dtype == torch.float32 else min(most, 127)
        gate = torch.randint(1, most + 1, (16, ff), generator=g).float() * (torch.randint(0, 2, (16, ff), generator=g) * 2 - 1) * least
        x = torch.cat([gate, up * torch.randn(16, ff, generator=g)], 1).to(dtype)
        assert (x[:, :ff] != 0).all()
        check_glu(D, x.cuda(), act)


@pytest.mark.parametrize("act", ["silu", "gelu"])
@pytest.mark.parametrize("ff", [4096, 4095])
def test_gated_unit_of_ups_below_the_normal_numbers(D, act, ff):
    """Rows next to the least ones that count: ups of up to 2^-123 and gates up to 16, which make the ups' products' roundings larger."""
    g = torch.Generator().manual_seed(ff)
    for place, up in enumerate((2.0**-128, 2.0**-126, 2.0**-124, 2.0**-122)):
        x = torch.cat([16 * (2 * torch.rand(64, ff, generator=g) - 0.5), up * torch.randn(64, ff, generator=g)], 1)
        check_glu(D, x.cuda(), act)


@pytest.mark.parametrize("act", ["silu", "gelu", "relu"])
@pytest.mark.parametrize("ff", [256, 257, 20000])
def test_gated_unit_next_to_the_largest_numbers(D, act, ff):
    """Largest values a step below 2^128 - 2^103, where f32 becomes infinite, and a step above: the exact one decides."""
    rows = 300
    g = torch.Generator().manual_seed(ff)
    x = torch.randn(rows, 2 * ff, generator=g)
    at = torch.randint(0, ff, (rows,), generator=g)
    every = torch.arange(rows)
    x[every, at] = 2 + 18 * torch.rand(rows, generator=g)
    x[every, ff + at] = 1.0
    per = R.glu(x, act)[every, at]      # act(gate)
    border = 2.0**128 - 2.0**103
    up = (border / per).float()
    y = per * up.double()
    assert torch.isfinite(up).all()
    above = torch.where(y >= border, up, torch.nextafter(up, torch.tensor(torch.inf)))
    below = torch.nextafter(above, torch.tensor(0.0))
    for u, live in ((below, True), (above, False)):
        x[every, ff + at] = u
        away = ((per * u.double() / border - 1).abs() > 2.0**-40) & torch.isfinite(u)      # (exact ones that 64 bits tell from the border)
        assert away.sum() > 250
        part = x[away].cuda()
        if live:
            check_glu(D, part, act)
        else:
            q, s = D.glu_q8(part, act)
            assert (q == 0).all() and torch.isnan(s).all()


@pytest.mark.parametrize("score", ["softmax", "sigmoid"])
@pytest.mark.parametrize("size", [64.0, 1000.0, 8000.0, 3e38])
@pytest.mark.parametrize("n,groups,top_groups", [(8, 4, 2), (64, 32, 8), (64, 16, 4), (256, 8, 4)])
def test_routing_by_groups_with_corrections_that_cancel(D, score, size, n, groups, top_groups):
    """A group's two best scores of opposite signs: their sum is small, the roundings of f32 are those of the scores."""
    rows = 400 if size < 1e30 else 20
    z = normal(n, rows, n) * (min(size, 1e4) * 2.0**-23 * 2.0 ** (torch.arange(rows) % 8))[:, None]      # (scores some of the corrections' roundings apart)
    place = torch.arange(n) % (n // groups)
    for first, second in ((size, -size), (-size, -size), (size, size)):
        c = torch.where(place == 0, first, torch.where(place == 1, second, -size))
        check_route(D, z, min(6, n // groups * top_groups), score=score, correction=c, groups=groups, top_groups=top_groups)


# (rows, k, n, group): by the kernels' own arithmetic on 148 SMs
@pytest.mark.parametrize("rows,k,n,group,scale", [
    (40, 28672, 200, 64, torch.float16),       # clusters of eight, seven steps a team, rings of four
    (64, 28672, 140, 32, torch.float32),       # ... rings of three, two units
    (20, 28672, 100, 128, torch.bfloat16),
    (33, 14336, 4096, 64, torch.bfloat16),     # clusters of four, seven steps
    (24, 8192, 8192, 32, torch.float16),       # clusters of two, eight steps
    (33, 4096, 9700, 128, torch.float32),      # no clusters, eight steps a team
    (56, 6144, 9600, 64, torch.float16),       # twelve steps
    (40, 2048, 20000, 32, torch.float16),      # two units a block, one after the other
    (130, 2048, 9700, 64, torch.bfloat16),     # ... of three chunks of rows, the last of two
    (185, 1056, 9608, 32, torch.float32),      # ... the last of 57
])
def test_product_of_more_rows_whose_rings_go_round(D, rows, k, n, group, scale):
    check_product(D, rows, k, n, group, scale)


@pytest.mark.parametrize("rows,k,n,group,scale", [
    (1, 4096, 12000, 128, torch.float16), (1, 14336, 4800, 32, torch.float32), (2, 14336, 4801, 32, torch.float16), (4, 8192, 9000, 64, torch.bfloat16),      # units that begin within a warp's steps
    (9, 14336, 4800, 32, torch.float16), (16, 14336, 4752, 64, torch.float32), (13, 4096, 12000, 128, torch.bfloat16), (6, 8192, 5000, 32, torch.float32)])
def test_product_of_few_rows_whose_rings_go_round(D, rows, k, n, group, scale):
    check_product(D, rows, k, n, group, scale)


@pytest.mark.parametrize("tokens,top,experts,k,n,group", [(100, 2, 4, 1056, 6000, 32), (300, 1, 5, 2048, 3000, 128), (64, 1, 2, 14336, 500, 64), (16, 2, 8, 4096, 2000, 32), (1, 2, 8, 4096, 6000, 32), (40, 4, 16, 2048, 1500, 64)])
@pytest.mark.parametrize("even", [True, False])
def test_product_of_experts_whose_rings_go_round(D, tokens, top, experts, k, n, group, even):
    """Units of several experts one after the other; with most tokens at one expert, units of other sizes than the average's."""
    g = torch.Generator().manual_seed(tokens)
    e = torch.stack([torch.randperm(experts, generator=g)[:top] for _ in range(tokens)]).int()
    if not even:
        e[torch.rand(tokens, top, generator=g) < 0.8] = experts - 1
        e[torch.rand(tokens, top, generator=g) < 0.1] = -1
    check_product(D, tokens * top, k, n, group, experts=e, n_experts=experts)


def test_products_in_clusters_captured_and_replayed_on_two_streams(D):
    """Clusters of eight and of four, and a product of few rows: graphs replayed at once on two streams with new inputs, each as by itself."""
    jobs = []
    for rows, k, n, group in ((50, 14336, 300, 64), (33, 14336, 4096, 32), (7, 4096, 5000, 128)):
        w, ws = D.quantise_i4(normal(rows, n, k).cuda(), group)
        a, s, out = bytes_of(rows, rows, k), torch.ones(rows).cuda(), torch.empty(rows, n).cuda()
        D.mat_mat_i4(a, s, w, ws, n=n, out=out)
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            for _ in range(4):
                D.mat_mat_i4(a, s, w, ws, n=n, out=out)
        jobs.append((a, s, w, ws, n, out, g))
    streams = [torch.cuda.Stream() for _ in jobs]
    for turn in range(3):
        want = []
        for a, s, w, ws, n, out, _ in jobs:
            a.copy_(bytes_of(100 + turn, *a.shape))
            want.append(D.mat_mat_i4(a, s, w, ws, n=n, dtype=torch.float32))
            out.fill_(0)
        torch.cuda.synchronize()
        for job, st in zip(jobs, streams):
            with torch.cuda.stream(st):
                job[-1].replay()
        torch.cuda.synchronize()
        assert all(torch.equal(job[5], v) for job, v in zip(jobs, want))


@pytest.mark.parametrize("rows", [1, 8, 40])
def test_product_of_the_largest_scales(D, rows):
    """Sums over the groups up to 2^124 (they are kept at sixteen times their value)."""
    a, values, scales = torch.full((rows, 256), 127, dtype=torch.int8).cuda(), torch.full((1, 20, 256), 7, dtype=torch.int8), torch.full((1, 20, 8), 2.0**106)      # 8 * 32 * 127 * 7 * 2^106: 2^123.8
    w, ws = (v.cuda() for v in D.i4_weights(values[0], scales[0]))
    s = torch.full((rows,), 2.0**-100).cuda()
    y = D.mat_mat_i4(a, s, w, ws, n=20, dtype=torch.float32)
    assert torch.equal(y.double(), torch.full((rows, 20), 8 * 32 * 127 * 7 * 2.0**6, dtype=torch.float64).cuda())      # (few bits: exact in any order)
