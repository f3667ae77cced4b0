"""Operators on tensors that are on the device already (b200_dev_*, include/llama_b200.h "operators on device tensors").

The peers of CudaB200Backend's rms_norm, mat_mat_q, rope, attention_cached and dequantize for a decoder layer that is served with activations in 8 bits
and a paged cache in 4 bits.  Tensors are torch CUDA tensors; the work is queued on the current stream of their device, outputs and workspaces come from torch's
allocator on that stream, so that the calls can be captured into a CUDA graph (a graph has its own workspaces).  Results carry no gradients (arguments
that require one, or have a forward-mode tangent, are refused), and have memory of their own.

    q, s, r = add_rms_norm_q8(x, weight, eps, residual=r)               # rows in 8 bits with a scale each, and the new residual
    qkv = mat_mat_i8(q, s, w, ws)                                       # 8-bit product
    q = rope_append_q4(q, k, v, table, positions, pages, slots)         # rotation; keys and values into the cache
    o = attention_paged_q4(q, pages, page_table, kv_lens, scale)

Errors are those of the backend (ShapeMismatch, InvalidArgument, ...).  What lies in device memory (slots, positions, pages, lengths) is checked by the kernels:
a bad entry is never followed, and sets a bit of `status` (an int32 tensor of one element) where one is given: STATUS_*.
"""
import ctypes as C
import importlib.util
import os

import torch

from . import _HERE, _STATUS, NotAvailable, _check, lib

STATUS_BAD_SLOT, STATUS_BAD_POSITION, STATUS_BAD_PAGE, STATUS_BAD_LENGTH = 1, 2, 4, 8


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
        names = ("b200_last_error", "b200_dev_add_rms_norm_q8", "b200_dev_read_q8", "b200_dev_mat_mat_i8", "b200_dev_rope_append_q4", "b200_dev_read_q4",
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
