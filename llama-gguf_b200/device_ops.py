"""Operators on tensors that are on the device already (b200_dev_*, include/llama_b200.h "operators on device tensors").

The peers of CudaB200Backend's rms_norm, mat_mat_q, rope, attention_cached and dequantize for a decoder layer that is served with activations in 8 bits
and a paged cache in 4 bits.  Tensors are torch CUDA tensors; the work is queued on the current stream of their device, outputs and workspaces come from torch's
allocator on that stream, so that the calls can be captured into a CUDA graph (a graph has its own workspaces).  Results carry no gradients (arguments
that require one, or have a forward-mode tangent, are refused), and have memory of their own.

    q, s, r = add_rms_norm_q8(x, weight, eps, residual=r)               # rows in 8 bits with a scale each, and the new residual
    qkv = mat_mat_i8(q, s, w, ws)                                       # 8-bit product
    q = rope_append_q4(q, k, v, table, positions, pages, slots)         # rotation; keys and values into the cache
    o = attention_paged_q4(q, pages, page_table, kv_lens, scale)

and its feed-forward with weights in 4 bits, here of routed experts:

    experts, weights = route_experts(logits, 2)                         # each token's experts
    h = mat_mat_i4(q, s, up, up_scales, experts=experts)                # 4-bit weights: [tokens * 2, 2 ff], gate and up
    q, s = glu_q8(h)                                                    # rows in 8 bits again
    y = mat_mat_i4(q, s, down, down_scales, experts=experts)
    q, s, r = add_gated_norm_q8(y, r, weight, eps, mix=weights)         # their weighted sum onto the stream, the next norm's rows

Errors are those of the backend (ShapeMismatch, InvalidArgument, ...).  What lies in device memory (slots, positions, pages, lengths, experts) is checked by the kernels:
a bad entry is never followed, and sets a bit of `status` (an int32 tensor of one element) where one is given: STATUS_*.
"""
import ctypes as C
import importlib.util
import os

import torch

from . import _HERE, _STATUS, DTypeMismatch, NotAvailable, ShapeMismatch, _check, lib

STATUS_BAD_SLOT, STATUS_BAD_POSITION, STATUS_BAD_PAGE, STATUS_BAD_LENGTH, STATUS_BAD_EXPERT = 1, 2, 4, 8, 16


class Q4Pages(C.Structure):
    """b200_q4_pages (include/llama_b200.h)"""
    _fields_ = [("data", C.c_void_p), ("n_pages", C.c_int64), ("page_size", C.c_int32), ("n_kv_heads", C.c_int32), ("head_dim", C.c_int32)]


class Q4Append(C.Structure):
    """b200_q4_append"""
    _fields_ = ([("device", C.c_int32), ("type", C.c_uint32), ("stream", C.c_void_p), ("q", C.c_void_p), ("k", C.c_void_p), ("v", C.c_void_p), ("q_out", C.c_void_p)]
                + [(n, C.c_int64) for n in ("q_token", "q_head", "k_token", "k_head", "v_token", "v_head", "q_out_token", "q_out_head")]
                + [("cos_sin", C.c_void_p), ("table_rows", C.c_int64), ("positions", C.c_void_p), ("slots", C.c_void_p), ("tokens", C.c_int64), ("n_heads", C.c_int32),
                   ("rot_dims", C.c_int32), ("use_neox", C.c_int32), ("cache", Q4Pages), ("status", C.c_void_p)])


class Q4Attention(C.Structure):
    """b200_q4_attention"""
    _fields_ = ([("device", C.c_int32), ("type", C.c_uint32), ("stream", C.c_void_p), ("q", C.c_void_p), ("out", C.c_void_p)]
                + [(n, C.c_int64) for n in ("q_token", "q_head", "out_token", "out_head")]
                + [("q_starts", C.c_void_p), ("kv_lens", C.c_void_p), ("page_table", C.c_void_p), ("table_stride", C.c_int64), ("tokens", C.c_int64),
                   ("table_pages", C.c_int32), ("seqs", C.c_int32), ("max_q", C.c_int32), ("n_heads", C.c_int32), ("window", C.c_int32), ("scale", C.c_float),
                   ("cache", Q4Pages), ("status", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t)])


class Route(C.Structure):
    """b200_route"""
    _fields_ = ([("device", C.c_int32), ("type", C.c_uint32), ("stream", C.c_void_p), ("logits", C.c_void_p), ("ld", C.c_int64), ("tokens", C.c_int64)]
                + [(n, C.c_int32) for n in ("n", "top", "groups", "top_groups", "sigmoid", "renormalise")]
                + [("scale", C.c_float), ("correction", C.c_void_p), ("experts", C.c_void_p), ("weights", C.c_void_p)])


class I4Product(C.Structure):
    """b200_i4_product"""
    _fields_ = ([("device", C.c_int32), ("out_type", C.c_uint32), ("scale_type", C.c_uint32), ("group", C.c_int32), ("stream", C.c_void_p), ("a", C.c_void_p), ("lda", C.c_int64)]
                + [(n, C.c_void_p) for n in ("a_scales", "w", "w_scales", "bias", "out")] + [(n, C.c_int64) for n in ("ldo", "tokens", "k", "n")]
                + [("experts", C.c_void_p), ("top", C.c_int32), ("n_experts", C.c_int32), ("rows_per_pair", C.c_int32), ("status", C.c_void_p)])


class GatedNorm(C.Structure):
    """b200_gated_norm"""
    _fields_ = ([("device", C.c_int32), ("type", C.c_uint32)] + [(n, C.c_void_p) for n in ("stream", "y", "mix", "post_weight", "gate", "residual", "sum", "weight", "q", "scales")]
                + [(n, C.c_int64) for n in ("ldy", "gate_row", "gate_col", "ldr", "lds", "ldq", "rows", "hidden")] + [("top", C.c_int32), ("scale", C.c_float), ("eps", C.c_float)])


_library = None
_calls = None


def _lib():
    global _library
    if _library is None:
        L = lib()
        i64, vp, sp = C.c_int64, C.c_void_p, C.POINTER(C.c_size_t)
        L.b200_dev_watchdog.argtypes = [C.c_int, C.POINTER(C.c_int)]
        L.b200_dev_add_rms_norm_q8.argtypes = [C.c_int, vp, C.c_uint32, vp, i64, vp, i64, vp, i64, vp, C.c_float, vp, i64, vp, i64, i64]
        L.b200_dev_read_q8.argtypes = [C.c_int, vp, C.c_uint32, vp, i64, vp, vp, i64, i64, i64]
        L.b200_dev_mat_mat_i8.argtypes = [C.c_int, vp, C.c_uint32, vp, i64, vp, vp, i64, vp, vp, vp, i64, i64, i64, i64]
        L.b200_dev_route_experts.argtypes = [C.POINTER(Route)]
        L.b200_dev_mat_mat_i4.argtypes = [C.POINTER(I4Product)]
        L.b200_dev_glu_q8.argtypes = [C.c_int, vp, C.c_uint32, C.c_int, vp, i64, vp, i64, vp, i64, i64]
        L.b200_dev_add_gated_norm_q8.argtypes = [C.POINTER(GatedNorm)]
        L.b200_dev_rope_append_q4.argtypes = [C.POINTER(Q4Append)]
        L.b200_dev_read_q4.argtypes = [C.c_int, vp, C.c_uint32, C.POINTER(Q4Pages), vp, i64, vp, vp, vp]
        L.b200_dev_attention_paged_q4_workspace.argtypes = [C.POINTER(Q4Attention), sp]
        L.b200_dev_attention_paged_q4.argtypes = [C.POINTER(Q4Attention)]
        L.b200_debug_i8_plan.argtypes = [i64, i64, i64, C.POINTER(C.c_int)]
        L.b200_debug_q4_prompt_blocks.argtypes = [C.POINTER(Q4Attention), C.POINTER(i64)]
        _library = L
    return _library


def _ops():
    """csrc/device_ops_py.cpp, bound to the loaded library and to this package's exceptions."""
    global _calls
    if _calls is None:
        path = os.path.join(_HERE, "_device_ops.so")
        if not os.path.exists(path):
            raise NotAvailable(f"{path} is missing (it needs torch's headers): build it with `python -c 'import __graft_entry__ as g; g.build()'`")
        L = _lib()
        spec = importlib.util.spec_from_file_location("_device_ops", path)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        names = ("b200_last_error", "b200_dev_add_rms_norm_q8", "b200_dev_read_q8", "b200_dev_mat_mat_i8", "b200_dev_route_experts", "b200_dev_mat_mat_i4", "b200_dev_glu_q8",
                 "b200_dev_add_gated_norm_q8", "b200_dev_rope_append_q4", "b200_dev_read_q4",
                 "b200_dev_attention_paged_q4_workspace", "b200_dev_attention_paged_q4")
        mod.bind(_STATUS, {n: C.cast(getattr(L, n), C.c_void_p).value for n in names})
        _calls = mod
    return _calls


def watchdog(device=0):
    """0, or the code of the bounded wait inside one of these operators that gave up last on this device (its results are then not valid); clears it."""
    v = C.c_int(0)
    _check(_lib().b200_dev_watchdog(int(device), C.byref(v)))
    return v.value


def i8_plan(t, k, n):
    """(tokens per tile, CTAs that share a tile's K, kernel of many tokens, pairs of CTAs) of mat_mat_i8: host logic, no device needed."""
    v = (C.c_int * 4)()
    _check(_lib().b200_debug_i8_plan(int(t), int(k), int(n), v))
    return tuple(v)


def padded_rows(rows, cols, device, dtype=torch.int8):
    """[rows, cols] of 8-bit integers whose rows are a multiple of 16 bytes apart, as mat_mat_i8 takes them."""
    return torch.empty(rows, (cols + 15) // 16 * 16, dtype=dtype, device=device)[:, :cols]


def add_rms_norm_q8(x, weight, eps, residual=None, sum_out=None, out=None, scales=None):
    """(q, scales, r): r = x + residual in the type of x; q [rows, hidden] int8 and scales [rows] f32 with q * scales = the RMS norm of r times weight (f32 [hidden]).

    Without a residual the norm is of x and r is None.  sum_out may be residual (or x) itself.  x, residual: [rows, hidden] f32, f16 or bf16 with contiguous rows."""
    return _ops().add_rms_norm_q8(x, weight, eps, residual, sum_out, out, scales)


def read_q8(q, scales, dtype=torch.float32):
    """[rows, n] of `dtype`: the values that rows in 8 bits stand for, q * scales."""
    return _ops().read_q8(q, scales, dtype)


def mat_mat_i8(a, a_scales, w, w_scales, bias=None, dtype=torch.bfloat16, out=None):
    """a [t, k] int8 (a scale per row) times w [n, k] int8 (a scale per row) -> [t, n] of `dtype` (of `out` where that is given), plus bias [n] f32.

    The sums are exact (k <= 131071).  a and w start on 16 bytes with rows a multiple of 16 bytes apart (padded_rows)."""
    return _ops().mat_mat_i8(a, a_scales, w, w_scales, bias, dtype, out)


def i4_weights(values, scales):
    """(w, w_scales) of mat_mat_i4: values int8 [.., n, k] from -8 to 7 and scales [.., n, k / group] (f32, f16 or bf16; group 32, 64 or 128) as b200_i4_product lays them out.

    What mat_mat_i4 multiplies with is scale * value.  Leading dimensions (experts) stay; rows behind n and channels behind k become zeros."""
    if values.dtype != torch.int8:
        raise DTypeMismatch(f"i4_weights: values: expected torch.int8, got {values.dtype}")
    if values.dim() < 2 or scales.shape[:-1] != values.shape[:-1] or scales.shape[-1] < 1 or values.shape[-1] % scales.shape[-1]:
        raise ShapeMismatch(f"i4_weights: expected [.., n, k] and [.., n, k / group], got {list(values.shape)} and {list(scales.shape)}")
    *lead, n, k = values.shape
    down, right = -n % 16, -k % 64
    v = (torch.nn.functional.pad(values, (0, right, 0, down)) & 15).view(torch.uint8).unflatten(-1, (-1, 2, 4, 2, 4)).unflatten(-6, (-1, 2, 8))
    d = len(lead)
    v = v.permute(*range(d), *(d + i for i in (0, 3, 2, 5, 4, 1, 6, 7)))      # row tile, step, g, t, half, row half, (low, high), byte
    s = torch.nn.functional.pad(scales, (0, 0, 0, down)).unflatten(-2, (-1, 2, 8)).movedim(-1, -3).transpose(-1, -2)
    return (v[..., 0, :] | v[..., 1, :] << 4).flatten(d + 2), s.contiguous()


def read_i4(w, w_scales, n, k):
    """[.., n, k] f32: the values that weights of mat_mat_i4 stand for."""
    d = w.dim() - 3
    b = w.unflatten(-1, (8, 4, 2, 2, 4))
    v = (torch.stack([b << 4, b & 240], -2).view(torch.int8) >> 4).permute(*range(d), *(d + i for i in (0, 5, 2, 1, 4, 3, 6, 7))).flatten(d + 3).flatten(d, d + 2)[..., :n, :k].float()
    s = w_scales.float().transpose(-1, -2).movedim(-3, -1).flatten(d, d + 2)[..., :n, :]
    return (v.unflatten(-1, (s.shape[-1], -1)) * s[..., None]).flatten(-2)


def quantise_i4(x, group=32, dtype=torch.float16):
    """(w, w_scales) of mat_mat_i4 for weights x [.., n, k]: a group's scale is its value of the largest magnitude / -8 in `dtype`, as a Q4_0 block's is, and the values round(x / scale)."""
    if group not in (32, 64, 128) or x.dim() < 2 or x.shape[-1] % group:
        raise ShapeMismatch(f"quantise_i4: expected [.., n, a multiple of the group], groups of 32, 64 or 128, got {list(x.shape)} and {group}")
    g = x.float().unflatten(-1, (-1, group))
    top = g.gather(-1, g.abs().argmax(-1, keepdim=True))
    d = (top / -8).to(dtype)
    v = torch.where(d == 0, 0.0, g / torch.where(d == 0, 1.0, d.float())).round_().clamp_(-8, 7)
    return i4_weights(v.to(torch.int8).flatten(-2), d[..., 0])


def i4_from_q4_0(blocks, k):
    """(w, w_scales) of mat_mat_i4 for rows of GGUF Q4_0 blocks, uint8 [.., n, k / 32 * 18]: the same values, groups of 32 with f16 scales."""
    if blocks.dtype != torch.uint8 or blocks.dim() < 2 or k % 32 or blocks.shape[-1] != k // 32 * 18:
        raise ShapeMismatch(f"i4_from_q4_0: expected uint8 [.., n, {k // 32 * 18}], got {blocks.dtype} {list(blocks.shape)}")
    b = blocks.unflatten(-1, (-1, 18))
    v = torch.cat([b[..., 2:] & 15, b[..., 2:] >> 4], -1).to(torch.int8) - 8
    return i4_weights(v.flatten(-2), b[..., :2].contiguous().view(torch.float16)[..., 0])


def mat_mat_i4(a, a_scales, w, w_scales, n=None, experts=None, bias=None, dtype=torch.bfloat16, out=None, status=None):
    """a [t, k] int8 (a scale per row) times 4-bit weights (a scale per row and group of channels) -> [t, n] of `dtype` (of `out` where that is given), plus bias [n] f32.

    w, w_scales: i4_weights, quantise_i4 or i4_from_q4_0 make them; n None: all rows of their tiles.  experts int32 [tokens, top] (route_experts): w, w_scales and bias have a leading dimension of
    experts, and the result [tokens * top, n] has a row for each of a token's experts; a has a row per token, or [tokens * top] rows, one for each.  Pairs of expert -1 get zeros, other numbers that
    are no expert too (and set STATUS_BAD_EXPERT).  The sums of a group are exact; those over the groups are f32 (below 2^124), in an order that the number of rows may change and, with experts, what other
    tokens choose.  a starts on 16 bytes with rows a multiple of 16 bytes apart (padded_rows).  For few rows: the weights' bytes are what it costs, once for up to 16 rows, else for every 64 (of an expert: for
    every 8, 16 or 64 pairs, by the average expert's number, and anew for every 2048 pairs of the call)."""
    return _ops().mat_mat_i4(a, a_scales, w, w_scales, n, experts, bias, dtype, out, status)


def route_experts(logits, top, score="softmax", correction=None, groups=1, top_groups=1, renormalise=True, scale=1.0, experts=None, weights=None):
    """(experts int32, weights f32) [tokens, top]: each token's experts by its router logits [tokens, n] (f32, f16 or bf16, contiguous rows), best first, the lower number among equals.

    The scores p are the softmax over all experts or (score="sigmoid") 1 / (1 + exp(-logit)); the choice goes by the logits, or by p + correction [n] f32 (a bias for balance, which the weights do not
    have).  groups > 1: of that many groups of neighbours only the best top_groups are left, by the sum of their two best scores.  weights: p, with renormalise over the chosen ones' sum, times scale.
    Logits of -inf (or NaN) are not chosen; places that nothing is left for hold expert -1 with weight 0, so that a row of -inf is a place without a token.  A row with a NaN has weights NaN."""
    return _ops().route_experts(logits, top, score, correction, groups, top_groups, renormalise, scale, experts, weights)


def glu_q8(x, act="silu", out=None, scales=None):
    """(q, scales): q [rows, ff] int8 and scales [rows] f32 with q * scales = act(x[:, :ff]) * x[:, ff:]; act silu, gelu (tanh form) or relu.  x: [rows, 2 ff] f32, f16 or bf16 with contiguous rows."""
    return _ops().glu_q8(x, act, out, scales)


def add_gated_norm_q8(y, residual, weight, eps, mix=None, post_weight=None, gate=None, scale=1.0, sum_out=None, out=None, scales=None):
    """(q, scales, r): r = residual + scale * gate * p in their type; q [rows, hidden] int8 and scales [rows] f32 with q * scales = the RMS norm of r times weight (weight None: both None).

    p is the block's output y [rows, hidden], or with mix f32 [rows, top] the sum of each row's `top` rows of y [rows * top, hidden] by those weights (route_experts' and mat_mat_i4's); with
    post_weight f32 [hidden] its RMS norm times that.  gate: of y's type, [rows, hidden], or 1 in place of either (broadcast).  sum_out may be residual itself."""
    return _ops().add_gated_norm_q8(y, residual, weight, eps, mix, post_weight, gate, scale, sum_out, out, scales)


def q4_pages(n_pages, n_kv_heads, head_dim, page_size, device="cuda"):
    """An empty cache: [pages, kv heads, page_size * (head_dim + 8)] bytes (the layout: b200_q4_pages)."""
    return torch.zeros(n_pages, n_kv_heads, page_size * (head_dim + 8), dtype=torch.uint8, device=device)


def rotary_table(positions, dims, base=10000.0, scale=1.0, device="cuda"):
    """cos_sin of rope_append_q4, [positions, dims] f32: the angle of pair i at position p is (p / scale) * base^(-2i / dims), worked out in 64 bits."""
    angle = (torch.arange(positions, dtype=torch.float64) / scale)[:, None] * base ** (-torch.arange(0, dims, 2, dtype=torch.float64) / dims)
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def rope_append_q4(q, k, v, cos_sin, positions, pages, slots, use_neox=False, q_out=None, status=None):
    """Rotates q and k, puts k and v into the cache in 4 bits, returns the rotated q (q None: None).

    q [tokens, heads, hd], k, v [tokens, kv heads, hd] (any distance between tokens and heads), cos_sin [positions, rot dims] f32 (rotary_table), positions int32 and
    slots int64 [tokens]: token t goes to page slots[t] // page_size, place slots[t] % page_size; slots[t] < 0: it is not cached.  The slots of a call
    are different ones (one that comes twice holds parts of either token).  q_out may be q."""
    return _ops().rope_append_q4(q, k, v, cos_sin, positions, pages, slots, use_neox, q_out, status)


def read_q4(pages, slots, head_dim, dtype=torch.float32, status=None):
    """(k, v) [tokens, kv heads, head_dim]: cached rows as the values they stand for; zeros where slots[t] < 0."""
    return _ops().read_q4(pages, slots, head_dim, dtype, status)


def attention_paged_q4(q, pages, page_table, kv_lens, scale=None, q_starts=None, max_q=0, window=0, out=None, status=None):
    """softmax(scale * q K^T) V over the cached positions, [tokens, heads, head_dim] in the type of q (scale None: head_dim ** -0.5).

    q [tokens, heads, hd]; page_table [sequences, most pages] and kv_lens [sequences] int32: sequence s has kv_lens[s] cached positions, its query tokens (already cached) among
    them.  q_starts int32 [sequences + 1]: its tokens are q_starts[s] .. q_starts[s + 1] - 1 and sit at its last positions, each sees the positions up to its own (the last `window` of
    them, 0: all); None: one token per sequence.  max_q: the most query tokens of a sequence where the host knows it; it only chooses between kernels.  A token that sees nothing
    gets zeros; tokens of `out` ahead of the first sequence and behind the last are left as they were (without `out`: not set)."""
    return _ops().attention_paged_q4(q, pages, page_table, kv_lens, scale, q_starts, max_q, window, out, status)
