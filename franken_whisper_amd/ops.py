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
import struct
import sys

import numpy as np

from . import abi
from .native import Context, check, lib

# element types by dtype object, numpy's from the start and torch's once a
# tensor comes along (this module does not import torch by itself)
_FLOAT = {np.dtype(np.float32): abi.T_F32, np.dtype(np.float16): abi.T_F16}
_I32, _I64, _U8 = {np.dtype(np.int32)}, {np.dtype(np.int64)}, {np.dtype(np.uint8)}
_MASK = {np.dtype(np.int64), np.dtype(np.uint64)}
_NAMES = ((_I32, "int32"), (_I64, "int64"), (_U8, "uint8"), (_MASK, "int64 or uint64"))
_torch = None


def _know_torch():
    """Whether torch's types were new to the tables above."""
    global _torch
    if _torch is not None or "torch" not in sys.modules:
        return False
    _torch = t = sys.modules["torch"]
    _FLOAT.update({t.float32: abi.T_F32, t.float16: abi.T_F16, t.bfloat16: abi.T_BF16})
    _I32.add(t.int32)
    _I64.add(t.int64)
    _U8.add(t.uint8)
    _MASK.update((t.int64, t.uint64))
    return True


# The argument structs, packed by the struct module (a third of the time that
# filling a ctypes structure takes); the layouts are abi's.
_PLAN, _APPEND = struct.Struct("6i16P"), struct.Struct("7i7q5P")
_ATTN, _Q4 = struct.Struct("12if8q9PQ"), struct.Struct("6i2q6P")
for _s, _c in ((_PLAN, abi.PagedPlanArgs), (_APPEND, abi.PagedAppendArgs), (_ATTN, abi.TreeAttnArgs),
               (_Q4, abi.Q4LinearArgs)):
    assert _s.size == C.sizeof(_c)
_fns = {}


def _call(name, ctx, args):
    fn = _fns.get(name)
    if fn is None:
        fn = lib()[name]  # a function object of its own: this one takes the packed bytes
        fn.restype, fn.argtypes = C.c_int32, [C.c_void_p, C.c_char_p]
        _fns[name] = fn
    code = fn(ctx.h, args)
    if code:
        check(code)


def _ptr(a, what, dev):
    """Device address; a tensor must be on device dev."""
    try:
        if a.get_device() == dev:
            return a.data_ptr()
    except AttributeError:
        p = a.ptr
        return (p if isinstance(p, int) else p.value) or 0
    raise ValueError(f"{what} must be on the context's device")


def _strides(a):
    try:
        return a.stride()
    except AttributeError:
        out, n = [], 1
        for s in reversed(a.shape):
            out.append(n)
            n *= s
        return tuple(reversed(out))


def _type(a, what):
    t = _FLOAT.get(a.dtype)
    if t is None:
        if _know_torch():
            return _type(a, what)
        raise ValueError(f"{what}: element type {a.dtype} is not float32, float16 or bfloat16")
    return t


def _whole(a, kind, shape, what, dev):
    """Address of a contiguous array of whole numbers, of the shape named; 0 for None."""
    if a is None:
        return 0
    if a.dtype not in kind:
        if _know_torch():
            return _whole(a, kind, shape, what, dev)
        raise ValueError(f"{what}: element type {a.dtype} is not {dict((id(k), n) for k, n in _NAMES)[id(kind)]}")
    if a.shape != shape:
        raise ValueError(f"{what}: shape {tuple(a.shape)} is not {shape}")
    try:
        if not a.is_contiguous():
            raise ValueError(f"{what} must be contiguous")
    except AttributeError:
        pass
    return _ptr(a, what, dev)


def _feature_contiguous(a, what):
    st = _strides(a)
    if st[-1] != 1 and a.shape[-1] > 1:
        raise ValueError(f"{what}: the elements of its last dimension must lie next to each other")
    return st


def _cache(k_cache, v_cache):
    """(page, token, head) strides that both caches share."""
    if k_cache.shape != v_cache.shape or len(k_cache.shape) != 4 or k_cache.dtype != v_cache.dtype:
        raise ValueError("k_cache and v_cache must be [pages, page size, heads, head dim] of one type")
    st = _feature_contiguous(k_cache, "k_cache")
    if _feature_contiguous(v_cache, "v_cache") != st:
        raise ValueError("k_cache and v_cache must have the same strides")
    return st


def paged_plan(ctx: Context, lens, n_new, table, held, free_pages, free_count, page_size: int, *, table_out, held_out,
               count_out, row_start, row_req, slot, pos, status, parents=None, mask=None):
    """fwhip_paged_plan: pages, slots, positions and ancestor masks of a step from
    the requests' lengths.  lens, n_new, held, status int32 [n_req]; table
    int32 [n_req, width]; free_pages int32, free_count int32 [1]; row_start
    int32 [n_req + 1]; row_req, pos, parents int32 and slot int64 [n_rows]; mask
    int64 or uint64 [n_rows, words]."""
    dev = ctx.device
    n_req, width = table.shape
    n_rows = slot.shape[0]
    per, rows = (n_req,), (n_rows,)
    words = 0 if mask is None else mask.shape[1]
    table_shape = (n_req, width)
    _call("fwhip_paged_plan", ctx, _PLAN.pack(
        n_req, width, page_size, n_rows, free_pages.shape[0], words, _whole(lens, _I32, per, "lens", dev),
        _whole(n_new, _I32, per, "n_new", dev), _whole(parents, _I32, rows, "parents", dev),
        _whole(table, _I32, table_shape, "table", dev), _whole(held, _I32, per, "held", dev),
        _whole(free_pages, _I32, free_pages.shape[:1], "free_pages", dev), _whole(free_count, _I32, (1,), "free_count", dev),
        _whole(table_out, _I32, table_shape, "table_out", dev), _whole(held_out, _I32, per, "held_out", dev),
        _whole(count_out, _I32, (1,), "count_out", dev), _whole(row_start, _I32, (n_req + 1,), "row_start", dev),
        _whole(row_req, _I32, rows, "row_req", dev), _whole(pos, _I32, rows, "pos", dev), _whole(slot, _I64, rows, "slot", dev),
        _whole(mask, _MASK, (n_rows, words), "mask", dev), _whole(status, _I32, per, "status", dev)))


def paged_append(ctx: Context, k, v, slot, k_cache, v_cache):
    """fwhip_paged_append: rows k, v [rows, heads, head dim] into the caches
    [pages, page size, heads, head dim] at slot int64 [rows] (page * page size +
    offset; outside the cache: skipped)."""
    dev = ctx.device
    rows, heads, dim = k.shape
    if v.shape != k.shape or v.dtype != k.dtype:
        raise ValueError("k and v must be [rows, heads, head dim] of one type")
    cst = _cache(k_cache, v_cache)
    pages, page_size, kv_heads, kv_dim = k_cache.shape
    if kv_heads != heads or kv_dim != dim:
        raise ValueError(f"the caches hold heads of {(kv_heads, kv_dim)}, the rows {(heads, dim)}")
    ks, vs = _feature_contiguous(k, "k"), _feature_contiguous(v, "v")
    _call("fwhip_paged_append", ctx, _APPEND.pack(
        _type(k, "k"), _type(k_cache, "k_cache"), rows, heads, dim, pages, page_size, ks[0], ks[1], vs[0], vs[1],
        cst[0], cst[1], cst[2], _ptr(k, "k", dev), _ptr(v, "v", dev), _whole(slot, _I64, (rows,), "slot", dev),
        _ptr(k_cache, "k_cache", dev), _ptr(v_cache, "v_cache", dev)))


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
    dev = ctx.device
    rows, heads, dim = q.shape
    n_req, width = table.shape
    if out.shape != q.shape or out.dtype != q.dtype:
        raise ValueError("out must have q's shape and type")
    cst = _cache(k_cache, v_cache)
    pages, page_size, kv_heads, cdim = k_cache.shape
    if cdim != dim or k_cache.dtype != q.dtype:
        raise ValueError("q and the caches must share their head dimension and type")
    dtype = _type(q, "q")
    if table.dtype not in _I32:
        raise ValueError("table must be int32")
    ts, qs, os_ = _feature_contiguous(table, "table"), _feature_contiguous(q, "q"), _feature_contiguous(out, "out")
    words = 0 if mask is None else mask.shape[1]
    if max_len is None:
        max_len = min(width * page_size, 0x7fff0000)
    _call("fwhip_tree_attn", ctx, _ATTN.pack(
        dtype, n_req, rows, heads, kv_heads, dim, pages, page_size, width, max_new, max_len, words, scale, ts[0],
        qs[0], qs[1], os_[0], os_[1], cst[0], cst[1], cst[2], _ptr(q, "q", dev), _ptr(k_cache, "k_cache", dev),
        _ptr(v_cache, "v_cache", dev), _ptr(table, "table", dev), _whole(lens, _I32, (n_req,), "lens", dev),
        _whole(row_start, _I32, (n_req + 1,), "row_start", dev), _whole(mask, _MASK, (rows, words), "mask", dev),
        _ptr(out, "out", dev), 0 if workspace is None else _ptr(workspace, "workspace", dev),
        0 if workspace is None else workspace.nbytes))


def _plane(a, shape, dtype, what, dev):
    """Address of a contiguous float array (dtype None: float32)."""
    if a.shape != shape or (a.dtype != dtype if dtype is not None else _type(a, what) != abi.T_F32):
        raise ValueError(f"{what} must be {shape} of {'float32' if dtype is None else dtype}")
    try:
        if not a.is_contiguous():
            raise ValueError(f"{what} must be contiguous")
    except AttributeError:
        pass
    return _ptr(a, what, dev)


def q4_linear(ctx: Context, x, q, scale, out, *, group: int = 32, minimum=None, bias=None):
    """fwhip_q4_linear: out [m, n] = x [m, k] W^T (+ bias float32 [n]); q uint8
    [n, k / 2], scale and minimum float16 or float32 [n, k / group]."""
    dev = ctx.device
    m, k = x.shape
    n = q.shape[0]
    if out.shape != (m, n) or out.dtype != x.dtype:
        raise ValueError("out must be [m, n] of x's type")
    if group < 1 or k % group:
        raise ValueError("group must divide k")
    dtype = _type(x, "x")
    planes = (n, k // group)
    xs, ys = _feature_contiguous(x, "x"), _feature_contiguous(out, "out")
    # the row stride of a single row is never used, and a tensor may give it any value
    _call("fwhip_q4_linear", ctx, _Q4.pack(
        dtype, _type(scale, "scale"), group, m, n, k, xs[0] if m > 1 else k, ys[0] if m > 1 else n, _ptr(x, "x", dev),
        _whole(q, _U8, (n, k // 2), "q", dev), _plane(scale, planes, scale.dtype, "scale", dev),
        0 if minimum is None else _plane(minimum, planes, scale.dtype, "minimum", dev),
        0 if bias is None else _plane(bias, (n,), None, "bias", dev), _ptr(out, "out", dev)))


def q4_planes(ctx: Context, ggml_dtype: int, raw, raw_bytes: int, rows: int, k: int, q, scale, minimum=None):
    """fwhip_q4_planes: a q4_0, q4_1 or q4_k payload (GgmlFile.raw, on the device)
    of a [rows, k] linear as the planes of q4_linear, group 32.  q uint8 [rows,
    k / 2]; scale (and minimum, except q4_0) [rows, k / 32], float16, for q4_k
    float32."""
    dev = ctx.device
    planes = (rows, k // 32)
    for p, what in ((scale, "scale"), (minimum, "minimum")):
        if p is not None and _type(p, what) != (abi.T_F32 if ggml_dtype == 12 else abi.T_F16):
            raise ValueError(f"{what} must be {'float32' if ggml_dtype == 12 else 'float16'} for this payload")
    check(lib().fwhip_q4_planes(ctx.h, ggml_dtype, _ptr(raw, "raw", dev), raw_bytes, rows, k,
                                _whole(q, _U8, (rows, k // 2), "q", dev), _plane(scale, planes, scale.dtype, "scale", dev),
                                None if minimum is None else _plane(minimum, planes, scale.dtype, "minimum", dev)))
