"""Operators on device tensors against plain forms in 64 bits: norm to 8 bits, 8-bit products, rotation into the paged 4-bit cache, attention over it."""
import math

import pytest
import torch

import device_ops_ref as R

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def D(b200):
    from llama_gguf_b200 import device_ops

    yield device_ops
    torch.cuda.synchronize()
    assert device_ops.watchdog() == 0      # (no bounded wait gave up)


def normal(seed, *shape):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed))


# ------------------------------------------------------------------------------------------------------------------- norm
def check_norm(D, x, w, eps, res, **kw):
    t = x.dtype
    q, s, r = D.add_rms_norm_q8(x, w, eps, residual=res, **kw)
    y = x.cpu().float() if res is None else (x.cpu().float() + res.cpu().float()).to(t).float()
    if res is not None:
        assert torch.equal(r.cpu().float(), y)
    y = y.double()
    eps = float(torch.tensor(eps))
    y = y * (1 / (y.square().mean(1, keepdim=True) + eps).sqrt()) * w.cpu().double()
    top = y.abs().amax(1)
    # rstd, two products: 3 half steps; the division 1
    assert ((s.cpu().double() - top / 127).abs() <= 4.01 * 2.0**-24 * top / 127).all()
    step = torch.where(top > 0, top / 127, 1.0)[:, None]
    # the quotient: 3 (y) + 4 (127 / m) + 1 half steps of at most 127, around the half that rounding takes
    assert ((q.cpu().double() - y / step).abs() <= 0.5 + 127 * 8.1 * 2.0**-24).all()
    assert q.dtype == torch.int8 and s.dtype == torch.float32


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden", [(1, 1), (1, 4096), (3, 31), (5, 896), (2, 2001), (17, 2048), (4, 8192), (300, 136), (2, 16384), (1, 16385), (2, 65536), (1, 40000)])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(D, dtype, rows, hidden, residual):
    x, w = normal(rows, rows, hidden).to(dtype).cuda(), (1 + 0.2 * normal(7, hidden)).cuda()
    res = (5 * normal(3, rows, hidden)).to(dtype).cuda() if residual else None
    check_norm(D, x, w, 1e-5, res)


@pytest.mark.parametrize("dtype", TYPES)
def test_norm_of_rows_apart_and_in_place(D, dtype):
    wide, w = normal(1, 9, 700).to(dtype).cuda(), (1 + 0.2 * normal(7, 513)).cuda()
    res = normal(2, 9, 513).to(dtype).cuda()
    check_norm(D, wide[:, 100:613], w, 1e-6, res)      # rows at odd places
    check_norm(D, wide[:1].expand(9, 700)[:, 8:521], w, 1e-6, res)      # one row again and again
    keep = res.clone()
    q, s, r = D.add_rms_norm_q8(wide[:, :513], w, 1e-6, residual=keep, sum_out=keep)
    q2, s2, r2 = D.add_rms_norm_q8(wide[:, :513], w, 1e-6, residual=res)
    assert r is keep and torch.equal(keep, r2) and torch.equal(q, q2) and torch.equal(s, s2)
    into = torch.full((9, 600), 77, dtype=torch.int8, device="cuda")
    D.add_rms_norm_q8(wide[:, :513], w, 1e-6, residual=res, out=into[:, 3:516])
    assert torch.equal(into[:, 3:516], q) and (into[:, :3] == 77).all() and (into[:, 516:] == 77).all()


def test_norm_of_rows_that_are_zero_tiny_or_not_finite(D):
    x = normal(1, 7, 260)
    x[1] = 0
    x[2] = 2.0**-140
    x[3, 5] = math.inf
    x[4, 259] = math.nan
    x[5] *= 1e18      # (squares up to 1e37: their sum is still an f32 number, and it is taken in 64 bits)
    q, s, _ = D.add_rms_norm_q8(x.cuda(), torch.ones(260).cuda(), 0.0)
    q, s = q.cpu(), s.cpu()
    assert (q[3:5] == 0).all() and torch.isnan(s[3:5]).all()
    assert not torch.isnan(s[[0, 5, 6]]).any() and (q[[0, 5, 6]].abs().amax(1) == 127).all()
    q, s, _ = D.add_rms_norm_q8(x.cuda(), torch.ones(260).cuda(), 1e-6)
    assert (q[1:3].cpu() == 0).all() and (s[1:3].cpu() == 0).all()
    q, s, _ = D.add_rms_norm_q8(x[:1].cuda(), torch.zeros(260).cuda(), 1e-6)
    assert (q == 0).all() and (s == 0).all()
    assert D.add_rms_norm_q8(x[:0].cuda(), torch.ones(260).cuda(), 1e-6)[0].shape == (0, 260)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,n", [(1, 1), (3, 31), (5, 4096), (700, 48), (2, 70000)])
def test_values_of_rows_in_8_bits(D, dtype, rows, n):
    q, s = torch.randint(-128, 128, (rows, n), dtype=torch.int8).cuda(), (0.01 * normal(3, rows)).cuda()
    s[rows // 2] = math.nan
    want = q.double() * s.double()[:, None]
    got = D.read_q8(q, s, dtype)
    assert got.dtype == dtype and torch.equal(torch.isnan(got), torch.isnan(want))
    # the product to f32, that to the type
    tol = (1.001 * 2.0**-24 + (1.001 * R.HALF_STEP[dtype] if dtype != torch.float32 else 0)) * want.abs() + R.LEAST[dtype]
    assert (torch.nan_to_num((got.double() - want).abs()) <= torch.nan_to_num(tol)).all()
    wide = torch.randint(-128, 128, (rows, n + 21), dtype=torch.int8).cuda()[:, 5 : 5 + n]
    assert torch.equal(torch.nan_to_num(D.read_q8(wide, s, dtype)), torch.nan_to_num(D.read_q8(wide.contiguous(), s, dtype)))


# ---------------------------------------------------------------------------------------------------------------- product
def bytes_of(seed, rows, k, extra=0):
    g = torch.Generator().manual_seed(seed)
    buf = torch.randint(-128, 128, (rows, (k + 15) // 16 * 16 + extra), generator=g, dtype=torch.int8).cuda()
    return buf[:, :k]      # (what lies behind a row is not zero)


def check_product(D, a, w, dtype, bias, **kw):
    t, n = a.shape[0], w.shape[0]
    s, ws = (0.01 + torch.rand(t)).cuda(), (0.001 * normal(5, n)).cuda()
    b = normal(6, n).cuda() if bias else None
    y = D.mat_mat_i8(a, s, w, ws, bias=b, dtype=dtype, **kw).double()
    v = (a.double() @ w.double().T) * s.double()[:, None] * ws.double()
    want = v + (b.double() if bias else 0)
    # the sum to f32, two products; the bias's sum; the result's type
    tol = 3.01 * 2.0**-24 * v.abs() + 1.01 * 2.0**-24 * want.abs() + 1.001 * R.HALF_STEP[dtype] * want.abs() + R.LEAST[dtype]
    assert ((y - want).abs() <= tol).all(), float(((y - want).abs() - tol).max())
    return y


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("t,k,n", [(1, 1, 1), (1, 4096, 512), (2, 17, 33), (4, 896, 1537), (8, 64, 8), (9, 1999, 130), (16, 4864, 896), (17, 128, 128), (33, 2047, 260), (61, 1999, 1537),
                                   (64, 512, 2048), (100, 16, 5), (128, 300, 77), (129, 1024, 384), (257, 1000, 1001), (300, 4096, 256), (700, 2048, 640), (1500, 640, 513)])
def test_product(D, dtype, t, k, n):
    check_product(D, bytes_of(1, t, k), bytes_of(2, n, k, 32), dtype, bias=(t + n) % 2 == 0)


@pytest.mark.parametrize("t", [1, 5, 40, 300])
def test_product_longest_sum(D, t):
    """k = 131071 of -128 * -128: 2^31 - 16384, the largest sum that 32 bits hold."""
    k = 131071
    a, w = (torch.full((r, 131072), -128, dtype=torch.int8, device="cuda")[:, :k] for r in (t, 9))
    one = lambda n: torch.ones(n, device="cuda")  # noqa: E731
    assert (D.mat_mat_i8(a, one(t), w, one(9), dtype=torch.float32) == float(k * 16384)).all()


@pytest.mark.parametrize("t", [3, 50, 260])
def test_product_into_rows_apart(D, t):
    a, w = bytes_of(1, t, 333, 64), bytes_of(2, 203, 333)
    buf = torch.full((t, 300), 5.0, device="cuda")
    check_product(D, a, w, torch.float32, True, out=buf[:, 41:244])
    assert (buf[:, :41] == 5).all() and (buf[:, 244:] == 5).all()


@pytest.mark.parametrize("t", [2, 200])
def test_product_passes_on_what_is_not_finite(D, t):
    a, w = bytes_of(1, t, 64), bytes_of(2, 40, 64)
    s = torch.ones(t, device="cuda")
    s[1] = math.nan      # (the norm's mark of a row that is not finite)
    y = D.mat_mat_i8(a, s, w, torch.ones(40, device="cuda"), dtype=torch.float32)
    assert torch.isnan(y[1]).all() and torch.isfinite(y[0]).all() and torch.isfinite(y[2:]).all()
    assert D.mat_mat_i8(a[:0], s[:0], w, torch.ones(40, device="cuda")).shape == (0, 40)


# ----------------------------------------------------------------------------------------------------------------- append
def append_inputs(seed, tokens, nh, nkv, hd, dtype, page, rot, fused=True):
    x = normal(seed, tokens, nh + 2 * nkv, hd).to(dtype).cuda()
    if not fused:      # heads first, and a distance that no word fits
        x = normal(seed, nh + 2 * nkv, tokens, hd + 1).to(dtype).cuda().transpose(0, 1)[..., 1:]
    n_pages = tokens // page + 3
    slots = torch.randperm(n_pages * page, generator=torch.Generator().manual_seed(seed))[:tokens]
    positions = torch.randint(0, 5000, (tokens,), generator=torch.Generator().manual_seed(seed + 1), dtype=torch.int32)
    return x[:, :nh], x[:, nh : nh + nkv], x[:, nh + nkv :], n_pages, slots, positions


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("tokens,nh,nkv,hd,page,rot,neox,fused", [
    (1, 32, 8, 128, 16, 128, False, True), (1, 14, 2, 64, 32, 64, True, True), (7, 4, 1, 128, 48, 64, True, True), (33, 4, 4, 64, 16, 32, False, True),
    (5, 3, 1, 64, 1024, 2, True, True), (70, 2, 2, 128, 64, 128, True, True), (19, 5, 5, 128, 16, 90, True, True), (19, 5, 1, 64, 16, 34, False, False), (9, 6, 2, 128, 32, 128, True, False),
    (300, 8, 2, 64, 128, 64, True, True)])
def test_append(D, dtype, tokens, nh, nkv, hd, page, rot, neox, fused):
    q, k, v, n_pages, slots, positions = append_inputs(tokens, tokens, nh, nkv, hd, dtype, page, rot, fused)
    slots[::5] = -1
    table = D.rotary_table(5000, rot)
    pages = torch.randint(0, 256, (n_pages, nkv, page * (hd + 8)), generator=torch.Generator().manual_seed(9), dtype=torch.uint8)
    dev = pages.cuda()
    out = D.rope_append_q4(q, k, v, table, positions.cuda(), dev, slots.cuda(), use_neox=neox)
    cs = table.cpu()[positions.long()][:, None]
    cos, sin = cs[..., : rot // 2], cs[..., rot // 2 :]
    # the same f32 steps: the same bytes everywhere, those that no token writes among them
    R.put_rows(pages, page, hd, slots, R.rotate(k.cpu().float(), cos, sin, neox), v.cpu().float())
    assert torch.equal(dev.cpu(), pages)
    assert torch.equal(out.cpu(), R.rotate(q.cpu().float(), cos, sin, neox).to(dtype))
    # and the formula in 64 bits: two products and a sum of a pair, none larger than its norm
    want = R.rotate(q.cpu().double(), cos.double(), sin.double(), neox)
    pair = (q.cpu().double().abs().amax(-1, keepdim=True) * math.sqrt(2)) * 3 * 2.0**-24
    assert ((out.cpu().double() - want).abs() <= pair + R.HALF_STEP[dtype] * want.abs() * 1.001 + R.LEAST[dtype]).all()
    kv = [x.cpu().double() for x in D.read_q4(dev, slots.cuda(), hd)]
    live = slots >= 0
    for got, x in zip(kv, (R.rotate(k.cpu().double(), cos.double(), sin.double(), neox), v.cpu().double())):
        assert (got[~live] == 0).all()
        got, x = got[live], x[live]
        d = x.abs().amax(-1, keepdim=True) / 8
        # half a step of 8 to a side, a whole one for the side that stops at 7; 24 half steps of f32 on the way
        assert ((got - x).abs() <= d * (torch.where(x.abs() > 7.5 * d - 1e-4 * d, 1.0, 0.5) + 24 * 8 * 2.0**-24)).all()


def test_append_in_place_and_without_queries(D):
    q, k, v, n_pages, slots, positions = append_inputs(3, 40, 6, 2, 64, torch.bfloat16, 16, 64)
    table = D.rotary_table(5000, 64, base=5e5)
    one, two = D.q4_pages(n_pages, 2, 64, 16), D.q4_pages(n_pages, 2, 64, 16)
    args = (table, positions.cuda())
    out = D.rope_append_q4(q.clone(), k, v, *args, one, slots.cuda(), use_neox=True)
    assert D.rope_append_q4(q, k, v, *args, one, slots.cuda(), use_neox=True, q_out=q) is q and torch.equal(q, out)
    assert D.rope_append_q4(None, k, v, *args, two, slots.cuda(), use_neox=True) is None and torch.equal(one, two)


def test_append_of_rows_that_are_zero_tiny_or_not_finite(D):
    k, v = normal(1, 6, 1, 128), normal(2, 6, 1, 128)
    v[0], v[1], v[2, 0, 9], v[3, 0, 127], v[4] = 0, 2.0**-130, math.inf, math.nan, -v[4].abs()
    v[5] = 0
    v[5, 0, 3], v[5, 0, 90] = -2.0, 2.0      # (the positive one of two)
    pages = D.q4_pages(1, 1, 128, 16)
    D.rope_append_q4(None, k.cuda(), v.cuda(), D.rotary_table(8, 128), torch.zeros(6, dtype=torch.int32).cuda(), pages, torch.arange(6).cuda())
    got = D.read_q4(pages, torch.arange(6).cuda(), 128)[1].cpu()
    assert (got[:2] == 0).all() and torch.isnan(got[2:4]).all() and torch.isfinite(got[4:]).all()
    assert got[5, 0, 90] == 2.0 and got[5, 0, 3] == -1.75


def test_append_skips_bad_entries_and_says_so(D):
    q, k, v, n_pages, slots, positions = append_inputs(3, 8, 4, 2, 64, torch.float32, 16, 64)
    table = D.rotary_table(5000, 64)
    slots[2], slots[5] = n_pages * 16, 1 << 40
    positions[3], positions[6] = 5000, -1
    keep = torch.randint(0, 256, (n_pages, 2, 16 * 72), dtype=torch.uint8)
    pages, status = keep.cuda(), torch.zeros(1, dtype=torch.int32).cuda()
    out = D.rope_append_q4(q, k, v, table, positions.cuda(), pages, slots.cuda(), status=status).cpu()
    good = torch.tensor([0, 1, 2, 4, 5, 7])
    assert torch.isnan(out[[3, 6]]).all() and torch.isfinite(out[good]).all()
    assert status.item() == D.STATUS_BAD_SLOT | D.STATUS_BAD_POSITION
    cs = table.cpu()[positions.clamp(0, 4999).long()][:, None]
    slots[[3, 6]] = -1
    R.put_rows(keep, 16, 64, slots, R.rotate(k.cpu(), cs[..., :32], cs[..., 32:], False), v.cpu())
    assert torch.equal(pages.cpu(), keep)
    status.zero_()
    assert (D.read_q4(pages, torch.tensor([n_pages * 16]).cuda(), 64, status=status)[0] == 0).all() and status.item() == D.STATUS_BAD_SLOT


# -------------------------------------------------------------------------------------------------------------- attention
def cache(seed, lens, nkv, hd, page, spare=2):
    need = [(n + page - 1) // page for n in lens]
    n_pages = sum(need) + spare
    order = torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)).tolist()
    width = max(need + [1]) + 1
    table, at = torch.full((len(lens), width), -7, dtype=torch.int32), 0      # (entries that no position needs are not looked at)
    for s, n in enumerate(need):
        table[s, :n] = torch.tensor(order[at : at + n], dtype=torch.int32)
        at += n
    # NaN wherever no position is, in scales and bytes
    pages = torch.full((n_pages, nkv, page * (hd + 8)), 255, dtype=torch.uint8)
    for s, n in enumerate(lens):
        slots = torch.tensor([int(table[s, j // page]) * page + j % page for j in range(n)], dtype=torch.long)
        scale = 1 + 3 * torch.rand(n, 1, 1, generator=torch.Generator().manual_seed(seed + s))
        R.put_rows(pages, page, hd, slots, normal(seed + 10 + s, n, nkv, hd), scale * normal(seed + 50 + s, n, nkv, hd))
    return pages, table


def check_attention(D, dtype, nh, nkv, hd, page, lens, q_lens, window=0, seed=1, gain=2.0, scale=None, **kw):
    pages, table = cache(seed, lens, nkv, hd, page)
    starts = [0]
    for m in q_lens:
        starts.append(starts[-1] + m)
    q = (gain * normal(seed + 99, starts[-1], nh, hd)).to(dtype)
    status = torch.zeros(1, dtype=torch.int32).cuda()
    args = dict(q_starts=None if all(m == 1 for m in q_lens) and not kw.pop("ragged", False) else torch.tensor(starts, dtype=torch.int32).cuda(), window=window, status=status, scale=scale)
    o = D.attention_paged_q4(q.cuda(), pages.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), **args, **kw)
    want, off = R.attention(q.double(), R.values(pages, page, hd), table.tolist(), lens, starts, page, hd**-0.5 if scale is None else scale, window, pages.shape[0], dtype)
    tol = off + 1.001 * R.HALF_STEP[dtype] * (want.abs() + off) + R.LEAST[dtype]
    got = o.cpu().double()
    assert torch.isfinite(got).all()
    assert ((got - want).abs() <= tol).all(), float(((got - want).abs() - tol).max())
    assert status.item() == 0
    return o


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,page", [(32, 8, 128, 16), (14, 2, 64, 32), (8, 1, 128, 64), (3, 3, 64, 16), (16, 1, 64, 48), (20, 1, 128, 16)])
def test_attention_of_single_tokens(D, dtype, nh, nkv, hd, page):
    check_attention(D, dtype, nh, nkv, hd, page, [1, 0, 16, 17, 333, 15, 1000], [1] * 7)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,lens", [([3, 1, 5], [3, 40, 200]), ([17, 0, 2], [17, 9, 100]), ([40], [90]), ([1, 7], [0, 5]), ([130], [130]), ([64, 65], [64, 300])])
def test_attention_of_several_tokens(D, dtype, q_lens, lens):
    check_attention(D, dtype, 8, 2, 128, 16, lens, q_lens)
    check_attention(D, dtype, 6, 2, 64, 32, lens, q_lens, max_q=max(q_lens))


@pytest.mark.parametrize("window", [1, 5, 16, 100, 5000])
def test_attention_window(D, window):
    check_attention(D, torch.float32, 8, 2, 64, 16, [1, 333, 40], [1, 1, 1], window=window)
    check_attention(D, torch.bfloat16, 8, 2, 128, 32, [50, 333, 40], [50, 3, 20], window=window)
    check_attention(D, torch.float16, 32, 16, 64, 32, [150, 333], [150, 140], window=window, max_q=150)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("q_len", [1, 3])
def test_attention_over_a_long_cache(D, dtype, q_len):
    check_attention(D, dtype, 4, 1, 128, 64, [6000, 31], [q_len, q_len])


def test_attention_of_large_scores_and_other_scales(D):
    """One position takes all of the softmax; the first keys are far below."""
    check_attention(D, torch.float32, 4, 2, 64, 16, [300, 64], [1, 1], gain=60.0)
    check_attention(D, torch.float32, 4, 2, 64, 16, [300, 64], [1, 1], scale=-0.3)
    check_attention(D, torch.float32, 4, 2, 64, 16, [300, 64], [1, 1], scale=0.0)
    check_attention(D, torch.bfloat16, 32, 16, 128, 16, [300, 164], [100, 64], gain=30.0)
    check_attention(D, torch.bfloat16, 32, 16, 128, 16, [300, 164], [100, 64], scale=-0.3)
    check_attention(D, torch.float16, 32, 16, 128, 16, [300, 164], [100, 64], scale=0.0)


@pytest.mark.parametrize("magnitude", [2.0**-100, 1e-6, 1e6, 2.0**100])
@pytest.mark.parametrize("q_lens,nkv", [([1, 1], 2), ([20, 17], 2), ([60, 17], 24)])
def test_attention_of_values_and_queries_of_any_magnitude(D, magnitude, q_lens, nkv):
    """Scales pass through in 32 bits: nothing is rounded to a type of less range."""
    pages, table = cache(5, [70, 20], nkv, 64, 16)
    ks, vs = R.sections(pages, 16, 64)[2:]
    vs.mul_(magnitude)
    starts = [0, q_lens[0], sum(q_lens)]
    q = normal(9, starts[-1], 2 * nkv, 64)
    lens = torch.tensor([70, 20], dtype=torch.int32).cuda()
    for f in (1.0, magnitude):
        ks.mul_(1 / f)
        want, off = R.attention(q.double() * f, R.values(pages, 16, 64), table.tolist(), [70, 20], starts, 16, 0.125, 0, pages.shape[0])
        got = D.attention_paged_q4((q * f).cuda(), pages.cuda(), table.cuda(), lens, q_starts=torch.tensor(starts, dtype=torch.int32).cuda()).cpu().double()
        assert ((got - want).abs() <= off + 2.0**-24 * want.abs()).all()
        ks.mul_(f)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_len,nkv", [(1, 2), (5, 2), (60, 2), (60, 40)])
def test_attention_what_is_masked_is_not_seen(D, dtype, q_len, nkv):
    """NaN and infinite rows behind a sequence's end or ahead of its windows change nothing; inside they make NaN of the rows that see them, and of no others."""
    pages, table = cache(5, [270], nkv, 64, 16)
    lens, q = torch.tensor([270], dtype=torch.int32).cuda(), normal(9, q_len, 2 * nkv, 64).to(dtype).cuda()
    starts, w = torch.tensor([0, q_len], dtype=torch.int32).cuda(), 20
    run = lambda window: D.attention_paged_q4(q, pages.cuda(), table.cuda(), lens, q_starts=starts, window=window)  # noqa: E731
    want = run(w)
    ks, vs = R.sections(pages, 16, 64)[2:]

    def spoil(j, i):
        page = int(table[0, j // 16])
        ks[page, :, j % 16], vs[page, :, j % 16] = math.nan, (math.inf if i % 2 else math.nan)

    for j in list(range(0, 270 - q_len - w + 1)) + list(range(270, 272)):
        spoil(j, j)
    assert torch.equal(run(w), want)
    seen = torch.isnan(run(w + 1)).flatten(1)
    assert seen[0].all() and not seen[1:].any()
    # the last position: only the last token sees it
    spoil(269, 0)
    seen = torch.isnan(run(w)).flatten(1)
    assert seen[-1].all() and not seen[:-1].any()


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_prompts(D, dtype, hd):
    """More rows than a block has, tiles that end anywhere, groups of heads that do not divide a block's rows; enough of them for the kernel of many rows."""
    check_attention(D, dtype, 36, 12, hd, 16, [129, 700], [129, 70])
    check_attention(D, dtype, 56, 8, hd, 48, [400, 33, 5], [45, 33, 5])
    check_attention(D, dtype, 20, 20, hd, 32, [257, 1], [200, 1], window=64)
    check_attention(D, dtype, 28, 28, hd, 64, [40, 70], [90, 70])      # (more tokens than positions: the first ones see nothing)


@pytest.mark.parametrize("dtype", TYPES)
def test_attention_of_prompts_with_scores_far_apart(D, dtype):
    """Scores of thousands, rising from tile to tile: a row's first tile says nothing about the others."""
    check_attention(D, dtype, 24, 12, 64, 16, [300, 700], [100, 64], gain=1000.0)
    check_attention(D, dtype, 96, 24, 128, 32, [600], [40], gain=400.0, window=300)
    check_attention(D, dtype, 96, 24, 64, 32, [600], [40], gain=0.0)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [2.0**-12, 2.0**-8, 1.0])
def test_attention_of_prompts_with_one_large_score(D, dtype, first):
    """The first position's score is 15 to 18 above all others, whose weights, thousands of them, are near the end of fp16; its value is small, so that theirs count."""
    n, q_len, nh, nkv, hd, page = 6000, 40, 96, 24, 64, 16
    k, v = normal(3, n, nkv, hd) / 16, 0.5 + normal(4, n, nkv, hd).abs()
    k[0], v[0] = 1.0, v[0] * first
    table = torch.randperm(n // page, generator=torch.Generator().manual_seed(5)).int()[None]
    pages = torch.zeros(n // page, nkv, page * (hd + 8), dtype=torch.uint8)
    at = torch.arange(n)
    R.put_rows(pages, page, hd, table[0, at // page].long() * page + at % page, k, v)
    q = (torch.linspace(15, 18, nh)[None, :, None] * hd**-0.5 + 0.01 * normal(6, q_len, nh, hd)).to(dtype)
    o = D.attention_paged_q4(q.cuda(), pages.cuda(), table.cuda(), torch.tensor([n], dtype=torch.int32).cuda(), q_starts=torch.tensor([0, q_len], dtype=torch.int32).cuda()).cpu().double()
    want, off = R.attention(q.double(), R.values(pages, page, hd), table.tolist(), [n], [0, q_len], page, hd**-0.5, 0, n // page, dtype)
    tol = off + 1.001 * R.HALF_STEP[dtype] * (want.abs() + off) + R.LEAST[dtype]
    assert ((o - want).abs() <= tol).all(), float(((o - want).abs() - tol).max())


@pytest.mark.parametrize("q_len,nkv", [(9, 2), (50, 2), (50, 20)])
def test_attention_of_several_tokens_with_bad_pages(D, q_len, nkv):
    lens = [300, 200]
    pages, table = cache(5, lens, nkv, 128, 16)
    table[0, 2], table[0, 9], table[1, 12] = -3, pages.shape[0], 2**31 - 1
    q, status = normal(9, 2 * q_len, 2 * nkv, 128).to(torch.bfloat16), torch.zeros(1, dtype=torch.int32).cuda()
    starts = [0, q_len, 2 * q_len]
    got = D.attention_paged_q4(q.cuda(), pages.cuda(), table.cuda(), torch.tensor(lens, dtype=torch.int32).cuda(), q_starts=torch.tensor(starts, dtype=torch.int32).cuda(), status=status)
    want, off = R.attention(q.double(), R.values(pages, 16, 128), table.tolist(), lens, starts, 16, 128**-0.5, 0, pages.shape[0], torch.bfloat16)
    assert ((got.cpu().double() - want).abs() <= off + 2.0**-8 * 1.001 * (want.abs() + off)).all() and status.item() == D.STATUS_BAD_PAGE


def test_attention_bad_pages_lengths_and_starts(D):
    lens = [100, 90, 40]
    pages, table = cache(5, lens, 2, 64, 16)
    q = normal(9, 3, 4, 64)
    bad = table.clone()
    bad[0, 2], bad[1, 0], bad[1, 5] = -3, pages.shape[0], 2**31 - 1
    status = torch.zeros(1, dtype=torch.int32).cuda()
    t32 = lambda *v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    got = D.attention_paged_q4(q.cuda(), pages.cuda(), bad.cuda(), t32(*lens), status=status).cpu().double()
    want, off = R.attention(q.double(), R.values(pages, 16, 64), bad.tolist(), lens, [0, 1, 2, 3], 16, 0.125, 0, pages.shape[0])
    assert ((got - want).abs() <= off + 2.0**-24 * want.abs()).all() and status.item() == D.STATUS_BAD_PAGE
    # no page at all
    status.zero_()
    assert (D.attention_paged_q4(q.cuda(), pages.cuda(), torch.full_like(bad, -1).cuda(), t32(*lens), status=status) == 0).all()
    # lengths: negative as zero, past the table cut
    status.zero_()
    full = table[:, :2].contiguous()
    got = D.attention_paged_q4(q.cuda(), pages.cuda(), full.cuda(), t32(2**31 - 1, -5, 32), status=status)
    assert torch.equal(got, D.attention_paged_q4(q.cuda(), pages.cuda(), full.cuda(), t32(32, 0, 32))) and (got[1] == 0).all() and status.item() == D.STATUS_BAD_LENGTH
    # starts that do not ascend within the tokens
    for starts in ([0, 2, 1, 3], [0, 1, 2, 9], [-1, 1, 2, 3]):
        status.zero_()
        D.attention_paged_q4(q.cuda(), pages.cuda(), table.cuda(), t32(*lens), q_starts=t32(*starts), status=status)
        assert status.item() & D.STATUS_BAD_LENGTH


def test_attention_leaves_other_tokens_and_strided_outputs(D):
    pages, table = cache(5, [40, 33], 2, 64, 16)
    wide = normal(9, 12, 4 + 2, 64 + 8).to(torch.bfloat16).cuda()
    q = wide[:, 1:5, 8:]
    buf = torch.full((12, 4, 80), 3.0, dtype=torch.bfloat16, device="cuda")
    starts, lens = torch.tensor([2, 5, 9], dtype=torch.int32).cuda(), torch.tensor([40, 33], dtype=torch.int32).cuda()
    o = D.attention_paged_q4(q, pages.cuda(), table.cuda(), lens, q_starts=starts, out=buf[:, :, 5:69])
    assert (buf[:2] == 3).all() and (buf[9:] == 3).all() and (buf[:, :, :5] == 3).all() and (buf[:, :, 69:] == 3).all()
    assert torch.equal(o[2:9], D.attention_paged_q4(q[2:9].contiguous(), pages.cuda(), table.cuda(), lens, q_starts=starts - 2))


def test_attention_of_sequences_that_share_a_table(D):
    pages, table = cache(5, [100], 2, 64, 16)
    q, lens = normal(9, 3, 4, 64).cuda(), torch.tensor([100, 60, 7], dtype=torch.int32).cuda()
    one = table.cuda().expand(3, -1)
    assert one.stride(0) == 0
    assert torch.equal(D.attention_paged_q4(q, pages.cuda(), one, lens), D.attention_paged_q4(q, pages.cuda(), one.contiguous(), lens))


# ---------------------------------------------------------------------------------------------------------------- together
def layer(D, s):
    """One attention sublayer as a server runs it: norm, product, rotation and append, attention, norm of the output."""
    nh, nkv, hd = 8, 2, 64
    a, sa, r = D.add_rms_norm_q8(s["x"], s["w1"], 1e-5, residual=s["r"])
    qkv = D.mat_mat_i8(a, sa, s["wqkv"], s["sqkv"], dtype=s["x"].dtype).unflatten(1, (nh + 2 * nkv, hd))
    q = D.rope_append_q4(qkv[:, :nh], qkv[:, nh : nh + nkv], qkv[:, nh + nkv :], s["table"], s["positions"], s["pages"], s["slots"])
    o = D.attention_paged_q4(q, s["pages"], s["page_table"], s["lens"], q_starts=s["starts"]).flatten(1)
    b, sb, _ = D.add_rms_norm_q8(o, s["w2"], 1e-5)
    return r, D.mat_mat_i8(b, sb, s["wo"], s["so"], dtype=s["x"].dtype)


def layer_state(D, dtype, q_lens, cached):
    hidden, nh, nkv, hd, page = 512, 8, 2, 64, 16
    n, lens = sum(q_lens), [m + c for m, c in zip(q_lens, cached)]
    pages, table = cache(3, cached, nkv, hd, page, spare=sum(q_lens) // page + 2 * len(lens) + 4)
    free = [p for p in range(pages.shape[0]) if p not in set(table.flatten().tolist())]
    table = torch.cat([table, torch.full((len(lens), 8), -7, dtype=torch.int32)], 1)
    slots, positions, starts = [], [], [0]
    for s, (m, c) in enumerate(zip(q_lens, cached)):
        for p in range(c, c + m):
            if table[s, p // page] < 0:
                table[s, p // page] = free.pop()
            slots.append(int(table[s, p // page]) * page + p % page)
            positions.append(p)
        starts.append(starts[-1] + m)
    s = dict(x=normal(1, n, hidden).to(dtype), r=(3 * normal(2, n, hidden)).to(dtype), w1=1 + 0.1 * normal(3, hidden), w2=1 + 0.1 * normal(4, nh * hd),
             wqkv=torch.randint(-127, 128, ((nh + 2 * nkv) * hd, hidden), dtype=torch.int8), sqkv=0.0005 + 0.0002 * torch.rand((nh + 2 * nkv) * hd),
             wo=torch.randint(-127, 128, (hidden, nh * hd), dtype=torch.int8), so=0.0005 + 0.0002 * torch.rand(hidden), table=D.rotary_table(2000, hd), pages=pages, page_table=table,
             positions=torch.tensor(positions, dtype=torch.int32), slots=torch.tensor(slots), lens=torch.tensor(lens, dtype=torch.int32), starts=torch.tensor(starts, dtype=torch.int32))
    return {k: v.cuda() for k, v in s.items()}


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("q_lens,cached", [([1, 1, 1], [0, 100, 37]), ([30, 1, 9], [0, 64, 5])])
def test_a_layer(D, dtype, q_lens, cached):
    """The chain against its plain form, each step from the kernels' own inputs so that no rounding decides otherwise than theirs."""
    s = layer_state(D, dtype, q_lens, cached)
    first = {k: v.cpu() for k, v in s.items()}
    r, y = (v.cpu().double() for v in layer(D, s))
    assert torch.equal(r, (first["x"].float() + first["r"].float()).to(dtype).double())
    a, sa, _ = D.add_rms_norm_q8(s["x"], s["w1"], 1e-5, residual=s["r"])
    qkv = D.mat_mat_i8(a, sa, s["wqkv"], s["sqkv"], dtype=dtype).cpu().float().unflatten(1, (12, 64))
    cs = first["table"][first["positions"].long()][:, None]
    R.put_rows(first["pages"], 16, 64, first["slots"], R.rotate(qkv[:, 8:10], cs[..., :32], cs[..., 32:], False), qkv[:, 10:])
    assert torch.equal(first["pages"], s["pages"].cpu())
    q = R.rotate(qkv[:, :8], cs[..., :32], cs[..., 32:], False).to(dtype).double()
    o, off = R.attention(q, R.values(first["pages"], 16, 64), first["page_table"].tolist(), first["lens"].tolist(), first["starts"].tolist(), 16, 0.125, 0, first["pages"].shape[0], dtype)
    o, off = o.flatten(1), (off + R.HALF_STEP[dtype] * 1.001 * (o.abs() + off) + R.LEAST[dtype]).flatten(1)
    rms = (o.square().mean(1, keepdim=True) + 1e-5).sqrt()
    n = o / rms * first["w2"].double()
    step = n.abs().amax(1, keepdim=True) / 127
    w = first["wo"].double() * first["so"].double()[:, None]
    # an element of the normed row is off by its own error (twice: the row's norm carries it too) and by half a step of 8 bits, at worst everywhere with one sign
    slip = 2 * off.amax(1, keepdim=True) / rms * first["w2"].double().abs().max() + 0.51 * step
    assert ((y - n @ w.T).abs() <= slip.expand_as(n) @ w.abs().T + R.HALF_STEP[dtype] * 1.01 * y.abs() + 1e-6).all()


@pytest.mark.parametrize("dtype", TYPES)
def test_a_layer_captured_and_replayed(D, dtype):
    """Two graphs of different batches, captured one after the other, replayed in turn on two streams: each as without a graph."""
    states = [layer_state(D, dtype, [1, 1, 1], [0, 300, 37]), layer_state(D, dtype, [30, 1, 9], [0, 64, 5])]
    want = [[v.clone() for v in layer(D, s)] for s in states]
    graphs, outs = [], []
    for s in states:
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            layer(D, s)
        torch.cuda.current_stream().wait_stream(side)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(D, s))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    for o, w in zip(outs, want):
        assert all(torch.equal(a, b) for a, b in zip(o, w))


def test_two_calls_at_once_on_other_streams(D):
    """Two streams, neither of them the default one, each with its own batch, and a third that reads results after an event."""
    states = [layer_state(D, torch.bfloat16, [1, 1, 1], [0, 700, 37]), layer_state(D, torch.bfloat16, [30, 1, 9], [0, 640, 5])]
    want = [[v.clone() for v in layer(D, s)] for s in states]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in states], [[], []]
    for _ in range(10):
        for i, (s, st) in enumerate(zip(states, streams)):
            with torch.cuda.stream(st):
                got[i].append(layer(D, s))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for r in g:
            assert all(torch.equal(a, b) for a, b in zip(r, w))


def test_calls_from_two_threads(D):
    import threading

    s = layer_state(D, torch.float16, [30, 1, 9], [0, 640, 5])
    want = [v.clone() for v in layer(D, s)]
    torch.cuda.synchronize()
    wrong = []

    def work():
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(20):
                r = layer(D, s)      # (both write the same rows into the cache)
                torch.cuda.current_stream().synchronize()
                if not all(torch.equal(a, b) for a, b in zip(r, want)):
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
    s = {k: v.to("cuda:1") for k, v in layer_state(D, torch.bfloat16, [30, 1, 9], [0, 64, 5]).items()}
    with torch.cuda.device(1):
        want = [v.clone() for v in layer(D, s)]
    assert torch.cuda.current_device() == 0
    assert all(torch.equal(a, b) for a, b in zip(layer(D, s), want)) and torch.cuda.current_device() == 0


def test_what_the_host_says_of_the_longest_changes_no_more_than_rounding(D):
    for max_q in (0, 1, 100, 10**6):
        check_attention(D, torch.float16, 36, 12, 64, 16, [129, 300], [129, 70], max_q=max_q)


def test_the_same_bits_every_time(D):
    s = layer_state(D, torch.bfloat16, [30, 1, 9], [0, 640, 5])
    one = [v.clone() for v in layer(D, s)]
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(one, layer(D, s)))
