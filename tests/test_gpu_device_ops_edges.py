"""Operators on device tensors where magnitudes, masks and sizes are far from ordinary, against plain forms in 64 bits."""
import ctypes as C

import pytest
import torch

import device_ops_exact as X
import device_ops_ref as R
import test_gpu_device_ops as T
from test_gpu_device_ops import TYPES, D, bytes_of, cache, check_norm, check_product, layer, layer_state, normal  # noqa: F401

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------------------------- norm
@pytest.mark.parametrize("dtype,magnitude", [(torch.bfloat16, 1e20), (torch.bfloat16, 1e30), (torch.bfloat16, 1e-25), (torch.bfloat16, 1e-30), (torch.float32, 1e20), (torch.float32, 1e-25),
                                             (torch.float16, 4096.0), (torch.float16, 2.0**-14)])
@pytest.mark.parametrize("rows,hidden", [(2, 256), (300, 4096), (2, 257)])
def test_norm_of_rows_of_any_magnitude(D, dtype, magnitude, rows, hidden):  # noqa: F811
    """Squares leave the range of f32 while the rows and their norms are well inside it: the same in whole words and by elements."""
    w, eps = (1 + 0.2 * normal(7, hidden)).cuda(), 0.0
    x = (magnitude * normal(rows, rows, hidden)).to(dtype).cuda()
    check_norm(D, x, w, eps, None)
    check_norm(D, x, w, eps, (2 * magnitude * normal(3, rows, hidden)).to(dtype).cuda())
    odd = torch.empty(rows, hidden + 1, dtype=dtype, device="cuda")[:, 1:]
    odd.copy_(x)
    assert all(torch.equal(a, b) for a, b in zip(D.add_rms_norm_q8(x, w, eps)[:2], D.add_rms_norm_q8(odd, w, eps)[:2]))


# ---------------------------------------------------------------------------------------------------------------- product
# every plan that a call can have, at sizes that end inside a tile in t, k and n: (tokens per tile, CTAs of a cluster that share K, kernel of many tokens, pairs of CTAs).  The kernels of many tokens: with an odd and an even
# number of tiles of weights (pairs: the last one has one row of tiles), once around and with more than two tiles for each CTA, so that both accumulators come again
PLANS = [((16, 1, 0, 0), 2, 300, 38404), ((16, 2, 0, 0), 3, 643, 4504), ((16, 4, 0, 0), 8, 1063, 2251), ((16, 8, 0, 0), 13, 1905, 130), ((32, 1, 0, 0), 18, 333, 77), ((32, 2, 0, 0), 17, 907, 4713),
         ((32, 4, 0, 0), 19, 700, 130), ((32, 8, 0, 0), 20, 2047, 300), ((64, 1, 0, 0), 65, 200, 333), ((64, 2, 0, 0), 2249, 1461, 1), ((64, 4, 0, 0), 66, 659, 300), ((64, 8, 0, 0), 65, 1919, 131),
         ((128, 1, 0, 0), 4752, 1, 135), ((128, 2, 0, 0), 4749, 4258, 1), ((128, 4, 0, 0), 2335, 2855, 1), ((128, 8, 0, 0), 911, 5655, 1), ((128, 1, 1, 0), 130, 4, 9496), ((128, 1, 1, 0), 130, 131, 9899),
         ((128, 1, 1, 0), 129, 4, 18967), ((128, 1, 1, 0), 130, 2, 19699), ((256, 1, 1, 0), 291, 1476, 6573), ((256, 1, 1, 0), 299, 1463, 6447), ((256, 1, 1, 0), 1312, 388, 8919), ((256, 1, 1, 0), 796, 392, 13688),
         ((256, 1, 1, 1), 5141, 2781, 387), ((256, 1, 1, 1), 6694, 2865, 263), ((256, 1, 1, 1), 269, 1110, 25328), ((256, 1, 1, 1), 313, 897, 25608)]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("plan,t,k,n", PLANS)
def test_product_of_every_plan(D, dtype, plan, t, k, n):  # noqa: F811
    assert D.i8_plan(t, k, n) == plan
    a, w = bytes_of(t, t, k, 16), bytes_of(n, n, k)
    check_product(D, a, w, dtype, bias=t % 2 == 0)
    buf = torch.full((t, n + 9), 5.0, dtype=dtype, device="cuda")
    check_product(D, a, w, dtype, bias=t % 2 == 1, out=buf[:, 4 : n + 4])
    assert (buf[:, :4] == 5).all() and (buf[:, n + 4 :] == 5).all()


# -------------------------------------------------------------------------------------------------------------- attention
def run_attention(D, q, pages, table, lens, starts, **kw):  # noqa: F811
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    return D.attention_paged_q4(q.cuda(), pages.cuda(), table.cuda(), i32(lens), q_starts=None if starts == list(range(len(lens) + 1)) else i32(starts), **kw).double()


def within(got, want, off, dtype):
    low, high = X.rounded(want, off, dtype)
    wrong = ~((got >= low) & (got <= high))
    assert not wrong.any(), (int(wrong.sum()), float(((got - want).abs() / (off + 2.0**-149))[wrong].max()))


def starts_of(q_lens):
    s = [0]
    for m in q_lens:
        s.append(s[-1] + m)
    return s


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("nh,nkv,hd,lens,q_lens", [(8, 2, 128, [1, 0, 333, 1000], [1] * 4), (16, 1, 64, [40, 2500], [1, 1]), (4, 2, 128, [40, 500], [7, 3]), (96, 24, 128, [300, 90], [70, 33]),
                                                   (24, 24, 64, [513], [200])])
@pytest.mark.parametrize("gain", [1.0, 6.0])
def test_attention_is_rounded_once(D, dtype, nh, nkv, hd, lens, q_lens, gain):  # noqa: F811
    """A result is what 64 bits give, rounded to its type: nothing on the way is held in fewer bits than f32 has, but for what the bound counts."""
    pages, table = cache(3, lens, nkv, hd, 16)
    starts = starts_of(q_lens)
    q = (gain * normal(8, starts[-1], nh, hd)).to(dtype)
    want, off = X.attention(q, pages, table, lens, starts, 16, hd**-0.5)
    within(run_attention(D, q, pages, table, lens, starts), want, off, dtype)


def one_large_score(nh, nkv, hd, page, seqs, n, first):
    """Positions of which the first one's key is far ahead of all others; its value is `first` times as large as theirs, and nothing but in channel 0."""
    k, v = normal(3, n, nkv, hd) / 16, 0.5 + normal(4, n, nkv, hd).abs()
    k[0], v[0, :, 0], v[0, :, 1:] = 1.0, v[0, :, 0] * first, 0.0
    table = torch.randperm(n // page, generator=torch.Generator().manual_seed(5)).int()[None].expand(seqs, -1).contiguous()
    pages = torch.zeros(n // page, nkv, page * (hd + 8), dtype=torch.uint8)
    at = torch.arange(n)
    R.put_rows(pages, page, hd, table[0, at // page].long() * page + at % page, k, v)
    return pages, table


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("first", [2.0**-6, 1.0, 8.0])
@pytest.mark.parametrize("high", [14.0, 18.0])
def test_attention_of_single_tokens_with_one_large_score(D, dtype, first, high):  # noqa: F811
    """The first position's weight is e^14 to e^18 times any other's, but its value has one channel: the rest of the result is theirs."""
    n, nh, nkv, hd, page, seqs = 4096, 32, 32, 64, 16, 8
    pages, table = one_large_score(nh, nkv, hd, page, seqs, n, first)
    q = (high * hd**-0.5 + 0.01 * normal(6, seqs, nh, hd)).to(dtype)
    want, off = X.attention(q, pages, table, [n] * seqs, list(range(seqs + 1)), page, hd**-0.5)
    within(run_attention(D, q, pages, table, [n] * seqs, list(range(seqs + 1))), want, off, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("sign", [1.0, -1.0])
@pytest.mark.parametrize("far", [1200, 200, 1279])
def test_attention_of_prompts_whose_references_move(D, dtype, sign, far):  # noqa: F811
    """One key is e^14 and more ahead of what the first tiles have, further than fp16 goes: its weight, nearly all of the result, has f32's bits.  One channel makes the scores, in numbers that
    need no rounding."""
    n, q_len, nh, nkv, hd, page = 1280, 40, 96, 24, 64, 16
    k, v = torch.zeros(n, nkv, hd), normal(4, n, nkv, hd)
    k[:, :, 0] = -(32 + torch.randint(0, 32, (n, nkv), generator=torch.Generator().manual_seed(1)).float()) / 64      # (a row's largest value is exact in 4 bits)
    k[far, :, 0] = 0.375
    table = torch.randperm(n // page, generator=torch.Generator().manual_seed(5)).int()[None]
    pages = torch.zeros(n // page, nkv, page * (hd + 8), dtype=torch.uint8)
    at = torch.arange(n)
    R.put_rows(pages, page, hd, table[0, at // page].long() * page + at % page, k, v)
    q = torch.zeros(q_len, nh, hd)
    q[:, :, 0] = sign * (1024 + torch.randint(0, 128, (q_len, nh), generator=torch.Generator().manual_seed(2)).float()) / 64      # 16 to 18
    q = q.to(dtype)
    want, off = X.attention(q, pages, table, [n], [0, q_len], page, sign, again=True, exact_scores=True)
    within(run_attention(D, q, pages, table, [n], [0, q_len], scale=sign), want, off, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,gone", [(1024, 1), (256, 1), (16, 17)])
def test_attention_of_prompts_without_their_first_pages(D, dtype, page, gone):  # noqa: F811
    """The first tiles have no key that is there: what follows counts as it does for single tokens, with scores far below zero and small values."""
    n, q_len, nh, nkv, hd = 1500, 40, 96, 24, 64
    pages, table = cache(5, [n], nkv, hd, page)
    ks, vs = R.sections(pages, page, hd)[2:]
    vs.mul_(2.0**-10)
    kb = R.sections(pages, page, hd)[0]
    kb[..., 0] = (kb[..., 0] & 0xF0) | 0      # channel 0 of every key is -8 of its scale's, whose sign makes it so
    ks.copy_(torch.where(torch.isnan(ks), ks, ks.abs()))
    table[0, :gone] = torch.tensor([-1, pages.shape[0], 2**31 - 1], dtype=torch.int32).repeat(6)[:gone]
    q = normal(9, q_len, nh, hd)
    q[:, :, 0] = 24.0      # (scores of some -24 * 8 * 0.3 / 8, give or take)
    q = q.to(dtype)
    status = torch.zeros(1, dtype=torch.int32).cuda()
    want, off = X.attention(q, pages, table, [n], [0, q_len], page, hd**-0.5)
    within(run_attention(D, q, pages, table, [n], [0, q_len], status=status), want, off, dtype)
    assert status.item() == D.STATUS_BAD_PAGE
    # ... and none at all
    assert (run_attention(D, q, pages, torch.full_like(table, -1), [n], [0, q_len]) == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("magnitude", [2.0**-115, 2.0**110, 2.0**120])
@pytest.mark.parametrize("q_lens,nkv", [([1, 1], 2), ([60, 17], 24)])
def test_attention_of_values_near_the_ends_of_f32(D, dtype, magnitude, q_lens, nkv):  # noqa: F811
    lens = [700, 120]
    pages, table = cache(5, lens, nkv, 64, 16)
    R.sections(pages, 16, 64)[3].mul_(magnitude)
    starts = starts_of(q_lens)
    q = (3.0 * normal(9, starts[-1], 4 * nkv, 64)).to(dtype)
    want, off = X.attention(q, pages, table, lens, starts, 16, 0.125)
    within(run_attention(D, q, pages, table, lens, starts), want, off, dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("magnitude", [2.0**-115, 2.0**120, 2.0**122])
@pytest.mark.parametrize("q_lens,nkv", [([1, 1], 2), ([60, 17], 24)])
def test_attention_of_queries_near_the_ends_of_f32(D, dtype, magnitude, q_lens, nkv):  # noqa: F811
    """Scores are ordinary: the keys' scales are as small as the queries are large."""
    lens = [700, 120]
    pages, table = cache(5, lens, nkv, 64, 16)
    R.sections(pages, 16, 64)[2].mul_(1 / magnitude)
    starts = starts_of(q_lens)
    q = ((2.0 * normal(9, starts[-1], 4 * nkv, 64)).clamp(-7, 7) * magnitude).to(dtype)
    want, off = X.attention(q, pages, table, lens, starts, 16, 0.125)
    within(run_attention(D, q, pages, table, lens, starts), want, off, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_attention_of_prompts_at_odd_places(D, dtype, hd):  # noqa: F811
    """Queries and results that no word fits, tokens ahead of the first sequence and behind the last, sequences without tokens: the same bits as from rows side by side, and nothing else written."""
    lens, q_lens, nh, nkv = [5, 300, 0, 160, 40], [0, 70, 0, 45, 1], 48, 12
    pages, table = cache(5, lens, nkv, hd, 48)
    starts = [s + 3 for s in starts_of(q_lens)]
    n = starts[-1] + 5
    wide = normal(9, n, nh + 1, hd + 3).to(dtype).cuda()
    q, buf = wide[:, 1:, 1 : hd + 1], torch.full((n, nh, hd + 5), 7.0, dtype=dtype, device="cuda")
    got = run_attention(D, q, pages, table, lens, starts, out=buf[:, :, 3 : hd + 3])
    assert (buf[: starts[0]] == 7).all() and (buf[starts[-1] :] == 7).all() and (buf[:, :, :3] == 7).all() and (buf[:, :, hd + 3 :] == 7).all()
    side = q[starts[0] : starts[-1]].contiguous()
    own = [s - starts[0] for s in starts]
    assert torch.equal(got[starts[0] : starts[-1]], run_attention(D, side, pages, table, lens, own))
    assert takes_prompts(D, q_lens, nh, nkv, hd)
    want, off = X.attention(side, pages, table, lens, own, 48, hd**-0.5)
    within(got[starts[0] : starts[-1]], want, off, dtype)


# ---------------------------------------------------------------------------------------------------------------- results
def test_results_have_memory_of_their_own(D):  # noqa: F811
    """A result that grows in place does not grow into another one, and one that is kept does not keep the others."""
    x = normal(1, 3, 256).bfloat16().cuda()
    pages = D.q4_pages(2, 2, 64, 16)
    for results in (D.add_rms_norm_q8(x, torch.ones(256).cuda(), 1e-5, residual=x), D.read_q4(pages, torch.arange(5).cuda(), 64, torch.bfloat16)):
        keep = [r.clone() for r in results]
        assert len({r.untyped_storage().data_ptr() for r in results}) == len(results)
        assert all(r.untyped_storage().nbytes() == r.numel() * r.element_size() for r in results)
        results[0].resize_(4 * results[0].numel()).fill_(77)
        assert all(torch.equal(a, b) for a, b in zip(results[1:], keep[1:]))


# ---------------------------------------------------------------------------------------------------------------- together
PROMPTS = ([300, 1, 9], [64, 640, 5])      # (a layer whose attention takes both kernels: one sequence has many rows)


def takes_prompts(D, q_lens, nh, nkv, hd):  # noqa: F811
    a = D.Q4Attention(type=0, q_starts=1, kv_lens=1, page_table=1, table_stride=9, tokens=sum(q_lens), table_pages=9, seqs=len(q_lens), n_heads=nh, scale=1.0,
                      cache=D.Q4Pages(data=16, n_pages=4, page_size=16, n_kv_heads=nkv, head_dim=hd))
    blocks = C.c_int64(-1)
    assert D._lib().b200_debug_q4_prompt_blocks(C.byref(a), C.byref(blocks)) == 0
    return blocks.value > 0


@pytest.mark.parametrize("dtype", TYPES)
def test_a_layer_with_a_prompt(D, dtype):  # noqa: F811
    assert takes_prompts(D, PROMPTS[0], 8, 2, 64) and not takes_prompts(D, [30, 1, 9], 8, 2, 64)
    T.test_a_layer(D, dtype, *PROMPTS)


@pytest.mark.parametrize("dtype", TYPES)
def test_a_layer_with_a_prompt_captured_replayed_and_at_once(D, dtype):  # noqa: F811
    """Graphs of a batch with a prompt and of a step, replayed in turn on two streams, then both eagerly at once: the same bits as one after the other."""
    states = [layer_state(D, dtype, *PROMPTS), layer_state(D, dtype, [1, 1, 1], [0, 300, 37])]
    want = [[v.clone() for v in layer(D, s)] for s in states]
    for s, w in zip(states, want):
        assert all(torch.equal(a, b) for a, b in zip(layer(D, s), w))
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for s in states:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(layer(D, s))
        graphs.append(g)
    for _ in range(5):
        for g, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                g.replay()
    torch.cuda.synchronize()
    got = [list(outs)]
    for _ in range(5):
        now = []
        for s, st in zip(states, streams):
            with torch.cuda.stream(st):
                now.append(layer(D, s))
        got.append(now)
    torch.cuda.synchronize()
    for run in got:
        for r, w in zip(run, want):
            assert all(torch.equal(a, b) for a, b in zip(r, w))
