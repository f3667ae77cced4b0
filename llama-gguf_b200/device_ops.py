"""Operators on tensors that are on the device already (b200_dev_*, include/llama_b200.h "operators on device tensors").

The peers of CudaB200Backend's rms_norm, mat_mat_q, rope, attention_cached and dequantize for a decoder layer that is served with activations in 8 bits
and a paged cache in 4 bits.  Tensors are torch CUDA tensors; the work is queued on the current stream of their device, outputs and workspaces come from torch's
allocator on that stream, so that the calls can be captured into a CUDA graph (a graph has its own workspaces).  Results carry no gradients.

    q, s, r = add_rms_norm_q8(x, weight, eps, residual=r)               # rows in 8 bits with a scale each, and the new residual
    qkv = mat_mat_i8(q, s, w, ws)                                       # 8-bit product
    q = rope_append_q4(q, k, v, table, positions, pages, slots)         # rotation; keys and values into the cache
    o = attention_paged_q4(q, pages, page_table, kv_lens, scale)

Errors are those of the backend (ShapeMismatch, InvalidArgument, ...).  What lies in device memory (slots, positions, pages, lengths) is checked by the kernels:
a bad entry is never followed, and sets a bit of `status` (an int32 tensor of one element) where one is given: STATUS_*.
"""
import ctypes as C
import math

import torch

from . import BF16, F16, F32, DTypeMismatch, InvalidArgument, ShapeMismatch, Unsupported, UnsupportedDType, _check, lib

STATUS_BAD_SLOT, STATUS_BAD_POSITION, STATUS_BAD_PAGE, STATUS_BAD_LENGTH = 1, 2, 4, 8
_TYPES = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}


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


_library = None


def _lib():
    global _library
    if _library is None:
        L = lib()
        i64, vp, sp = C.c_int64, C.c_void_p, C.POINTER(C.c_size_t)
        L.b200_dev_watchdog.argtypes = [C.c_int, C.POINTER(C.c_int)]
        L.b200_dev_add_rms_norm_q8.argtypes = [C.c_int, vp, C.c_uint32, vp, i64, vp, i64, vp, i64, vp, C.c_float, vp, i64, vp, i64, i64]
        L.b200_dev_mat_mat_i8.argtypes = [C.c_int, vp, C.c_uint32, vp, i64, vp, vp, i64, vp, vp, vp, i64, i64, i64, i64]
        L.b200_dev_rope_append_q4.argtypes = [C.POINTER(Q4Append)]
        L.b200_dev_read_q4.argtypes = [C.c_int, vp, C.c_uint32, C.POINTER(Q4Pages), vp, i64, vp, vp, vp]
        L.b200_dev_attention_paged_q4_workspace.argtypes = [C.POINTER(Q4Attention), sp]
        L.b200_dev_attention_paged_q4.argtypes = [C.POINTER(Q4Attention)]
        _library = L
    return _library


def _type(what, t):
    try:
        return _TYPES[t]
    except KeyError:
        raise UnsupportedDType(f"{what}: {t} (float32, float16 and bfloat16 only)") from None


def _same(what, device, **tensors):
    """All on one CUDA device, and none that a gradient would have to come through."""
    grad = torch.is_grad_enabled()
    for name, t in tensors.items():
        if t is None:
            continue
        if grad and t.requires_grad:
            raise Unsupported(f"{what}: {name} requires a gradient, and results carry none (detach it)")
        if t.device != device:
            raise InvalidArgument(f"{what}: {name} is on {t.device}, expected {device}")
    if device.type != "cuda":
        raise InvalidArgument(f"{what}: tensors on a CUDA device expected, got {device}")


def _vector(what, name, t, n, dtype):
    if t.dtype != dtype:
        raise DTypeMismatch(f"{what}: {name}: expected {dtype}, got {t.dtype}")
    if t.dim() != 1 or t.shape[0] != n or (n > 1 and t.stride(0) != 1):
        raise ShapeMismatch(f"{what}: {name}: expected [{n}] contiguous, got {list(t.shape)}")


def _matrix(what, name, t, rows, cols, dtype):
    if t.dtype != dtype:
        raise DTypeMismatch(f"{what}: {name}: expected {dtype}, got {t.dtype}")
    if t.dim() != 2 or t.shape[0] != rows or t.shape[1] != cols or (cols > 1 and t.stride(1) != 1):
        raise ShapeMismatch(f"{what}: {name}: expected [{rows}, {cols}] with contiguous rows, got {list(t.shape)}")


def _heads(what, name, t, tokens, heads, hd, dtype):
    if t.dtype != dtype:
        raise DTypeMismatch(f"{what}: {name}: expected {dtype}, got {t.dtype}")
    if t.dim() != 3 or t.shape[0] != tokens or (heads is not None and t.shape[1] != heads) or t.shape[2] != hd or t.stride(2) != 1:
        raise ShapeMismatch(f"{what}: {name}: expected [{tokens}, {heads if heads is not None else 'heads'}, {hd}] with contiguous channels, got {list(t.shape)}")


def _pages(what, pages, hd):
    if pages.dtype != torch.uint8:
        raise DTypeMismatch(f"{what}: pages: expected torch.uint8, got {pages.dtype}")
    if pages.dim() != 3 or not pages.is_contiguous() or pages.shape[2] % (hd + 8):
        raise ShapeMismatch(f"{what}: pages: expected [pages, kv heads, page_size * {hd + 8}] contiguous, got {list(pages.shape)}")
    return Q4Pages(pages.data_ptr(), pages.shape[0], pages.shape[2] // (hd + 8), pages.shape[1], hd)


def _status(what, status, device):
    if status is None:
        return None
    if status.dtype != torch.int32 or status.numel() != 1 or status.device != device:
        raise InvalidArgument(f"{what}: status: one int32 on {device} expected")
    return status.data_ptr()


def _ld(t):
    """Distance of rows in elements (torch gives any number where there is one row)."""
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _stream(device):
    return torch.cuda.current_stream(device).cuda_stream


def watchdog(device=0):
    """0, or the code of the bounded wait inside one of these operators that gave up last on this device (its results are then not valid); clears it."""
    v = C.c_int(0)
    _check(_lib().b200_dev_watchdog(int(device), C.byref(v)))
    return v.value


def padded_rows(rows, cols, device, dtype=torch.int8):
    """[rows, cols] of 8-bit integers whose rows are a multiple of 16 bytes apart, as mat_mat_i8 takes them."""
    return torch.empty(rows, (cols + 15) // 16 * 16, dtype=dtype, device=device)[:, :cols]


def add_rms_norm_q8(x, weight, eps, residual=None, sum_out=None, out=None, scales=None):
    """(q, scales, r): r = x + residual in the type of x; q [rows, hidden] int8 and scales [rows] f32 with q * scales = the RMS norm of r times weight (f32 [hidden]).

    Without a residual the norm is of x and r is None.  sum_out may be residual (or x) itself.  x, residual: [rows, hidden] f32, f16 or bf16 with contiguous rows."""
    what = "add_rms_norm_q8"
    if x.dim() != 2:
        raise ShapeMismatch(f"{what}: x: expected [rows, hidden], got {list(x.shape)}")
    rows, hidden = x.shape
    t = _type(what, x.dtype)
    _matrix(what, "x", x, rows, hidden, x.dtype)
    _vector(what, "weight", weight, hidden, torch.float32)
    if residual is not None:
        _matrix(what, "residual", residual, rows, hidden, x.dtype)
        if sum_out is not None:
            _matrix(what, "sum_out", sum_out, rows, hidden, x.dtype)
    elif sum_out is not None:
        raise InvalidArgument(f"{what}: sum_out without a residual")
    if out is not None:
        _matrix(what, "out", out, rows, hidden, torch.int8)
    if scales is not None:
        _vector(what, "scales", scales, rows, torch.float32)
    device = x.device
    _same(what, device, x=x, weight=weight, residual=residual, sum_out=sum_out, out=out, scales=scales)
    q = padded_rows(rows, hidden, device) if out is None else out
    s = torch.empty(rows, dtype=torch.float32, device=device) if scales is None else scales
    r = None
    if residual is not None:
        r = torch.empty(rows, hidden, dtype=x.dtype, device=device) if sum_out is None else sum_out
    _check(_lib().b200_dev_add_rms_norm_q8(device.index, _stream(device), t, x.data_ptr(), _ld(x), residual.data_ptr() if r is not None else None, _ld(residual) if r is not None else 0,
                                           r.data_ptr() if r is not None else None, _ld(r) if r is not None else 0, weight.data_ptr(), eps, q.data_ptr(), _ld(q) if out is not None else (hidden + 15) // 16 * 16,
                                           s.data_ptr(), rows, hidden))
    return q, s, r


def mat_mat_i8(a, a_scales, w, w_scales, bias=None, dtype=torch.bfloat16, out=None):
    """a [t, k] int8 (a scale per row) times w [n, k] int8 (a scale per row) -> [t, n] of `dtype`, plus bias [n] f32.

    The sums are exact (k <= 131071).  a and w start on 16 bytes with rows a multiple of 16 bytes apart (padded_rows)."""
    what = "mat_mat_i8"
    if a.dim() != 2 or w.dim() != 2:
        raise ShapeMismatch(f"{what}: expected [t, k] and [n, k], got {list(a.shape)} and {list(w.shape)}")
    (rows, k), n = a.shape, w.shape[0]
    if out is not None:
        dtype = out.dtype
        _matrix(what, "out", out, rows, n, dtype)
    t = _type(what, dtype)
    _matrix(what, "a", a, rows, k, torch.int8)
    _matrix(what, "w", w, n, k, torch.int8)
    _vector(what, "a_scales", a_scales, rows, torch.float32)
    _vector(what, "w_scales", w_scales, n, torch.float32)
    if bias is not None:
        _vector(what, "bias", bias, n, torch.float32)
    device = a.device
    _same(what, device, a=a, w=w, a_scales=a_scales, w_scales=w_scales, bias=bias, out=out)
    y = torch.empty(rows, n, dtype=dtype, device=device) if out is None else out
    up = lambda m: m.stride(0) if m.shape[0] > 1 else (k + 15) // 16 * 16  # noqa: E731  (one row has no distance)
    _check(_lib().b200_dev_mat_mat_i8(device.index, _stream(device), t, a.data_ptr(), up(a), a_scales.data_ptr(), w.data_ptr(), up(w), w_scales.data_ptr(),
                                      bias.data_ptr() if bias is not None else None, y.data_ptr(), _ld(y), rows, k, n))
    return y


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
    slots int64 [tokens]: token t goes to page slots[t] // page_size, place slots[t] % page_size; slots[t] < 0: it is not cached.  q_out may be q."""
    what = "rope_append_q4"
    if k.dim() != 3:
        raise ShapeMismatch(f"{what}: k: expected [tokens, kv heads, head_dim], got {list(k.shape)}")
    tokens, nkv, hd = k.shape
    t = _type(what, k.dtype)
    c = _pages(what, pages, hd)
    if nkv != c.n_kv_heads:
        raise ShapeMismatch(f"{what}: k has {nkv} heads, the cache {c.n_kv_heads}")
    _heads(what, "k", k, tokens, nkv, hd, k.dtype)
    _heads(what, "v", v, tokens, nkv, hd, k.dtype)
    if q is not None:
        _heads(what, "q", q, tokens, None, hd, k.dtype)
        if q_out is not None:
            _heads(what, "q_out", q_out, tokens, q.shape[1], hd, k.dtype)
    if cos_sin.dim() != 2 or not cos_sin.is_contiguous():
        raise ShapeMismatch(f"{what}: cos_sin: expected [positions, rot dims] contiguous, got {list(cos_sin.shape)}")
    _matrix(what, "cos_sin", cos_sin, cos_sin.shape[0], cos_sin.shape[1], torch.float32)
    _vector(what, "positions", positions, tokens, torch.int32)
    _vector(what, "slots", slots, tokens, torch.int64)
    device = k.device
    _same(what, device, q=q, k=k, v=v, cos_sin=cos_sin, positions=positions, pages=pages, slots=slots, q_out=q_out)
    if q is not None and q_out is None:
        q_out = torch.empty(q.shape, dtype=q.dtype, device=device)
    a = Q4Append(device.index, t, _stream(device), None if q is None else q.data_ptr(), k.data_ptr(), v.data_ptr(), None if q is None else q_out.data_ptr(),
                 *((0, 0) if q is None else q.stride()[:2]), *k.stride()[:2], *v.stride()[:2], *((0, 0) if q is None else q_out.stride()[:2]),
                 cos_sin.data_ptr(), cos_sin.shape[0], positions.data_ptr(), slots.data_ptr(), tokens, 0 if q is None else q.shape[1], cos_sin.shape[1], 1 if use_neox else 0, c,
                 _status(what, status, device))
    _check(_lib().b200_dev_rope_append_q4(C.byref(a)))
    return q_out if q is not None else None


def read_q4(pages, slots, head_dim, dtype=torch.float32, status=None):
    """(k, v) [tokens, kv heads, head_dim]: cached rows as the values they stand for; zeros where slots[t] < 0."""
    what = "read_q4"
    t = _type(what, dtype)
    c = _pages(what, pages, head_dim)
    _vector(what, "slots", slots, slots.numel(), torch.int64)
    device = pages.device
    _same(what, device, pages=pages, slots=slots)
    k, v = torch.empty(2, slots.numel(), c.n_kv_heads, head_dim, dtype=dtype, device=device).unbind(0)
    _check(_lib().b200_dev_read_q4(device.index, _stream(device), t, C.byref(c), slots.data_ptr(), slots.numel(), k.data_ptr(), v.data_ptr(), _status(what, status, device)))
    return k, v


def attention_paged_q4(q, pages, page_table, kv_lens, scale=None, q_starts=None, max_q=0, window=0, out=None, status=None):
    """softmax(scale * q K^T) V over the cached positions, [tokens, heads, head_dim] in the type of q.

    q [tokens, heads, hd]; page_table [sequences, most pages] and kv_lens [sequences] int32: sequence s has kv_lens[s] cached positions, its query tokens (already cached) among
    them.  q_starts int32 [sequences + 1]: its tokens are q_starts[s] .. q_starts[s + 1] - 1 and sit at its last positions, each sees the positions up to its own (the last `window` of
    them, 0: all); None: one token per sequence.  max_q: the most query tokens of a sequence where the host knows it; it only chooses between kernels.  A token that sees nothing
    gets zeros; tokens of `out` behind the last sequence are left as they were."""
    what = "attention_paged_q4"
    if q.dim() != 3:
        raise ShapeMismatch(f"{what}: q: expected [tokens, heads, head_dim], got {list(q.shape)}")
    tokens, nh, hd = q.shape
    t = _type(what, q.dtype)
    c = _pages(what, pages, hd)
    _heads(what, "q", q, tokens, nh, hd, q.dtype)
    if page_table.dim() != 2:
        raise ShapeMismatch(f"{what}: page_table: expected [sequences, pages], got {list(page_table.shape)}")
    seqs, width = page_table.shape
    _matrix(what, "page_table", page_table, seqs, width, torch.int32)
    _vector(what, "kv_lens", kv_lens, seqs, torch.int32)
    if q_starts is not None:
        _vector(what, "q_starts", q_starts, seqs + 1, torch.int32)
    if out is not None:
        _heads(what, "out", out, tokens, nh, hd, q.dtype)
    scale = 1.0 / math.sqrt(hd) if scale is None else float(scale)
    if not math.isfinite(scale):
        raise InvalidArgument(f"{what}: scale {scale}")
    device = q.device
    _same(what, device, q=q, pages=pages, page_table=page_table, kv_lens=kv_lens, q_starts=q_starts, out=out)
    o = torch.empty(tokens, nh, hd, dtype=q.dtype, device=device) if out is None else out
    a = Q4Attention(device.index, t, _stream(device), q.data_ptr(), o.data_ptr(), *q.stride()[:2], *o.stride()[:2], None if q_starts is None else q_starts.data_ptr(), kv_lens.data_ptr(),
                    page_table.data_ptr(), _ld(page_table), tokens, width, seqs, int(max_q), nh, int(window), scale, c, _status(what, status, device), None, 0)
    need = C.c_size_t()
    _check(_lib().b200_dev_attention_paged_q4_workspace(C.byref(a), C.byref(need)))
    if need.value:
        work = torch.empty(need.value, dtype=torch.uint8, device=device)
        a.workspace, a.workspace_bytes = work.data_ptr(), need.value
    _check(_lib().b200_dev_attention_paged_q4(C.byref(a)))
    return o
