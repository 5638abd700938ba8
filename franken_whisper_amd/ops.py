"""The operators of a decode step with drafted tokens over a paged K/V cache,
and linears with 4-bit weights (include/fwhip.h, "decoding with drafted
tokens").

Arrays are native.DeviceArray or torch tensors on the context's device.  Every
call queues its work on the context's stream and returns: a torch program
makes its context on the stream it works on (native.Context(device,
stream=torch.cuda.current_stream().cuda_stream)), or orders the two streams
itself.  bfloat16 is a torch type only; DeviceArrays are float32 or float16.
"""
from __future__ import annotations

import ctypes as C

from . import abi
from .native import Context, check, lib

_TYPES = {"float32": abi.T_F32, "torch.float32": abi.T_F32, "float16": abi.T_F16, "torch.float16": abi.T_F16,
          "torch.bfloat16": abi.T_BF16}
_INTS = {"int32": ("int32", "torch.int32"), "int64": ("int64", "torch.int64"),
         "mask": ("int64", "uint64", "torch.int64", "torch.uint64"), "uint8": ("uint8", "torch.uint8")}


def _ptr(a):
    """Device address, or None."""
    if a is None:
        return None
    if hasattr(a, "data_ptr"):
        if not a.is_cuda:
            raise ValueError("a tensor of these operators must be on the GPU")
        return a.data_ptr()
    return a.ptr


def _strides(a):
    if hasattr(a, "data_ptr"):
        return a.stride()
    out, n = [], 1
    for s in reversed(a.shape):
        out.append(n)
        n *= s
    return tuple(reversed(out))


def _type(a, what):
    t = _TYPES.get(str(a.dtype))
    if t is None:
        raise ValueError(f"{what}: element type {a.dtype} is not float32, float16 or bfloat16")
    return t


def _whole(a, kind, shape, what):
    """Address of a contiguous array of whole numbers, of the shape named."""
    if a is None:
        return None
    if str(a.dtype) not in _INTS[kind]:
        raise ValueError(f"{what}: element type {a.dtype} is not {kind if kind != 'mask' else 'int64 or uint64'}")
    if tuple(a.shape) != shape:
        raise ValueError(f"{what}: shape {tuple(a.shape)} is not {shape}")
    if hasattr(a, "data_ptr") and not a.is_contiguous():
        raise ValueError(f"{what} must be contiguous")
    return _ptr(a)


def _feature_contiguous(a, what):
    st = _strides(a)
    if a.shape[-1] > 1 and st[-1] != 1:
        raise ValueError(f"{what}: the elements of its last dimension must lie next to each other")
    return st


def _cache(k_cache, v_cache):
    """(page, token, head) strides that both caches share."""
    if tuple(k_cache.shape) != tuple(v_cache.shape) or len(k_cache.shape) != 4 or str(k_cache.dtype) != str(v_cache.dtype):
        raise ValueError("k_cache and v_cache must be [pages, page size, heads, head dim] of one type")
    st = _feature_contiguous(k_cache, "k_cache")
    if tuple(_feature_contiguous(v_cache, "v_cache")) != tuple(st):
        raise ValueError("k_cache and v_cache must have the same strides")
    return st


def paged_plan(ctx: Context, lens, n_new, table, held, free_pages, free_count, page_size: int, *, table_out, held_out,
               count_out, row_start, row_req, slot, pos, status, parents=None, mask=None):
    """fwhip_paged_plan: pages, slots, positions and ancestor masks of a step from
    the requests' lengths.  lens, n_new, held, status int32 [n_req]; table
    int32 [n_req, width]; free_pages int32, free_count int32 [1]; row_start
    int32 [n_req + 1]; row_req, pos, parents int32 and slot int64 [n_rows]; mask
    int64 or uint64 [n_rows, words]."""
    n_req, width = table.shape
    n_rows = slot.shape[0]
    per, rows = (n_req,), (n_rows,)
    words = 0 if mask is None else mask.shape[1]
    a = abi.PagedPlanArgs(
        n_req, width, page_size, n_rows, free_pages.shape[0], words, _whole(lens, "int32", per, "lens"),
        _whole(n_new, "int32", per, "n_new"), _whole(parents, "int32", rows, "parents"),
        _whole(table, "int32", (n_req, width), "table"), _whole(held, "int32", per, "held"),
        _whole(free_pages, "int32", tuple(free_pages.shape[:1]), "free_pages"),
        _whole(free_count, "int32", (1,), "free_count"), _whole(table_out, "int32", (n_req, width), "table_out"),
        _whole(held_out, "int32", per, "held_out"), _whole(count_out, "int32", (1,), "count_out"),
        _whole(row_start, "int32", (n_req + 1,), "row_start"), _whole(row_req, "int32", rows, "row_req"),
        _whole(pos, "int32", rows, "pos"), _whole(slot, "int64", rows, "slot"),
        _whole(mask, "mask", (n_rows, words), "mask"), _whole(status, "int32", per, "status"))
    check(lib().fwhip_paged_plan(ctx.h, C.byref(a)))


def paged_append(ctx: Context, k, v, slot, k_cache, v_cache):
    """fwhip_paged_append: rows k, v [rows, heads, head dim] into the caches
    [pages, page size, heads, head dim] at slot int64 [rows] (page * page size +
    offset; outside the cache: skipped)."""
    rows, heads, dim = k.shape
    if tuple(v.shape) != (rows, heads, dim) or str(v.dtype) != str(k.dtype):
        raise ValueError("k and v must be [rows, heads, head dim] of one type")
    cst = _cache(k_cache, v_cache)
    if tuple(k_cache.shape[2:]) != (heads, dim):
        raise ValueError(f"the caches hold heads of {tuple(k_cache.shape[2:])}, the rows {(heads, dim)}")
    ks, vs = _feature_contiguous(k, "k"), _feature_contiguous(v, "v")
    a = abi.PagedAppendArgs(_type(k, "k"), _type(k_cache, "k_cache"), rows, heads, dim, k_cache.shape[0],
                            k_cache.shape[1], ks[0], ks[1], vs[0], vs[1], cst[0], cst[1], cst[2], _ptr(k), _ptr(v),
                            _whole(slot, "int64", (rows,), "slot"), _ptr(k_cache), _ptr(v_cache))
    check(lib().fwhip_paged_append(ctx.h, C.byref(a)))


def tree_attn_workspace(n_req: int, n_heads: int, n_kv_heads: int, head_dim: int, max_new: int, max_len: int) -> int:
    """fwhip_tree_attn_workspace: bytes of workspace that tree_attn of these sizes needs."""
    n = C.c_uint64()
    check(lib().fwhip_tree_attn_workspace(n_req, n_heads, n_kv_heads, head_dim, max_new, max_len, C.byref(n)))
    return n.value


def tree_attn(ctx: Context, q, k_cache, v_cache, table, lens, row_start, out, *, scale: float, max_new: int,
              max_len: int | None = None, mask=None, workspace=None):
    """fwhip_tree_attn: q, out [rows, heads, head dim]; caches [pages, page size,
    K/V heads, head dim]; table int32 [n_req, width]; lens int32 [n_req] (cached
    tokens before this step); row_start int32 [n_req + 1]; mask int64 or uint64
    [rows, words] or None (a causal chain).  max_len (default: the table's
    reach) bounds lens + new tokens, max_new the new tokens of a request.
    workspace: uint8 of tree_attn_workspace bytes, needed when that is not 0."""
    rows, heads, dim = q.shape
    n_req, width = table.shape
    if tuple(out.shape) != (rows, heads, dim) or str(out.dtype) != str(q.dtype):
        raise ValueError("out must have q's shape and type")
    cst = _cache(k_cache, v_cache)
    pages, page_size, kv_heads, cdim = k_cache.shape
    if cdim != dim or str(k_cache.dtype) != str(q.dtype):
        raise ValueError("q and the caches must share their head dimension and type")
    if str(table.dtype) not in _INTS["int32"]:
        raise ValueError("table must be int32")
    ts, qs, os_ = _feature_contiguous(table, "table"), _feature_contiguous(q, "q"), _feature_contiguous(out, "out")
    words = 0 if mask is None else mask.shape[1]
    a = abi.TreeAttnArgs(_type(q, "q"), n_req, rows, heads, kv_heads, dim, pages, page_size, width, max_new,
                         min(width * page_size, 0x7fff0000) if max_len is None else max_len, words, scale, ts[0],
                         qs[0], qs[1], os_[0], os_[1], cst[0], cst[1], cst[2], _ptr(q), _ptr(k_cache), _ptr(v_cache),
                         _ptr(table), _whole(lens, "int32", (n_req,), "lens"),
                         _whole(row_start, "int32", (n_req + 1,), "row_start"),
                         _whole(mask, "mask", (rows, words), "mask"), _ptr(out), _ptr(workspace),
                         0 if workspace is None else
                         workspace.nbytes if hasattr(workspace, "nbytes") else workspace.numel() * workspace.element_size())
    check(lib().fwhip_tree_attn(ctx.h, C.byref(a)))


def q4_linear(ctx: Context, x, q, scale, out, *, group: int = 32, minimum=None, bias=None):
    """fwhip_q4_linear: out [m, n] = x [m, k] W^T (+ bias float32 [n]); q uint8
    [n, k / 2], scale and minimum float16 or float32 [n, k / group]."""
    m, k = x.shape
    n = q.shape[0]
    if tuple(out.shape) != (m, n) or str(out.dtype) != str(x.dtype):
        raise ValueError("out must be [m, n] of x's type")
    if group < 1 or k % group:
        raise ValueError("group must divide k")
    planes = (n, k // group)
    for p, what in ((scale, "scale"), (minimum, "minimum")):
        if p is None:
            continue
        if tuple(p.shape) != planes or str(p.dtype) != str(scale.dtype):
            raise ValueError(f"{what} must be {planes}, both planes of one type")
        if hasattr(p, "data_ptr") and not p.is_contiguous():
            raise ValueError(f"{what} must be contiguous")
    if bias is not None and (tuple(bias.shape) != (n,) or _type(bias, "bias") != abi.T_F32 or
                             (n > 1 and _strides(bias)[0] != 1)):
        raise ValueError("bias must be contiguous float32 [n]")
    xs, ys = _feature_contiguous(x, "x"), _feature_contiguous(out, "out")
    # the row stride of a single row is never used, and a tensor may give it any value
    a = abi.Q4LinearArgs(_type(x, "x"), _type(scale, "scale"), group, m, n, k, xs[0] if m > 1 else k,
                         ys[0] if m > 1 else n, _ptr(x), _whole(q, "uint8", (n, k // 2), "q"), _ptr(scale),
                         _ptr(minimum), _ptr(bias), _ptr(out))
    check(lib().fwhip_q4_linear(ctx.h, C.byref(a)))


def q4_planes(ctx: Context, ggml_dtype: int, raw, raw_bytes: int, rows: int, k: int, q, scale, minimum=None):
    """fwhip_q4_planes: a q4_0, q4_1 or q4_k payload (GgmlFile.raw, on the device)
    of a [rows, k] linear as the planes of q4_linear, group 32.  q uint8 [rows,
    k / 2]; scale (and minimum, except q4_0) [rows, k / 32], float16, for q4_k
    float32."""
    want = abi.T_F32 if ggml_dtype == 12 else abi.T_F16
    for p, what in ((scale, "scale"), (minimum, "minimum")):
        if p is not None and (_type(p, what) != want or tuple(p.shape) != (rows, k // 32) or
                              (hasattr(p, "data_ptr") and not p.is_contiguous())):
            raise ValueError(f"{what} must be contiguous {(rows, k // 32)} of {'float32' if want == abi.T_F32 else 'float16'}")
    check(lib().fwhip_q4_planes(ctx.h, ggml_dtype, _ptr(raw), raw_bytes, rows, k,
                                _whole(q, "uint8", (rows, k // 2), "q"), _ptr(scale), _ptr(minimum)))
