"""What the serving operators refuse, without a GPU: every argument is checked
before the context is, so a NULL context shows which check answers (CPU)."""
import ctypes as C

import numpy as np
import pytest

from franken_whisper_amd import abi, native, ops

A = 1 << 20  # an address as good as any: nothing is read
T = {"f32": abi.T_F32, "f16": abi.T_F16, "bf16": abi.T_BF16}


def _says(fn, args, word, code=abi.ERR_INVALID):
    rc = getattr(native.lib(), fn)(None, C.byref(args) if args is not None else None)
    msg = native.lib().fwhip_last_error().decode()
    assert rc == code and word in msg, (rc, msg)


def _set(make, **kw):
    a = make()
    for k, v in kw.items():
        assert hasattr(a, k)
        setattr(a, k, v)
    return a


def _plan():
    return abi.PagedPlanArgs(2, 8, 16, 10, 20, 1, *[A + 0x10000 * i for i in range(16)])


def _append():
    return abi.PagedAppendArgs(0, 1, 4, 2, 64, 8, 16, 128, 64, 128, 64, 2048, 128, 64, A, 2 * A, 3 * A, 4 * A, 5 * A)


def _attn():
    return abi.TreeAttnArgs(1, 2, 10, 8, 2, 64, 8, 16, 8, 5, 128, 1, 0.125, 8, 512, 64, 512, 64, 2048, 128, 64,
                            A, 2 * A, 3 * A, 4 * A, 5 * A, 6 * A, 7 * A, 8 * A, 9 * A, 1 << 30)


def _q4():
    return abi.Q4LinearArgs(1, 1, 32, 3, 50, 64, 64, 50, A, 2 * A, 3 * A, None, 4 * A, 5 * A)


@pytest.mark.parametrize("fn,make", [("fwhip_paged_plan", _plan), ("fwhip_paged_append", _append),
                                     ("fwhip_tree_attn", _attn), ("fwhip_q4_linear", _q4)])
def test_a_good_call_gets_as_far_as_its_context(fn, make):
    _says(fn, make(), "NULL ctx")
    _says(fn, None, "args is NULL")


@pytest.mark.parametrize("kw,word", [
    (dict(n_req=-1), "negative size"), (dict(width=-1), "negative size"), (dict(n_rows=-1), "negative size"),
    (dict(n_free=-1), "negative size"), (dict(page_size=0), "page_size"), (dict(page_size=1 << 25), "page_size"),
    (dict(len=None), "NULL"), (dict(held=None), "NULL"), (dict(table=None), "NULL"), (dict(slot=None), "NULL"),
    (dict(free_pages=None), "NULL"), (dict(count_out=None), "NULL"), (dict(row_start=None), "NULL"),
    (dict(status=None), "NULL"), (dict(mask=None), "go together"), (dict(parents=None), "go together"),
    (dict(mask_words=0), "mask_words"), (dict(mask_words=5), "mask_words"),
    (dict(held_out=A + 0x40000), "held_out"), (dict(held_out=A), "held_out"), (dict(count_out=A + 0x60000), "count_out"),
    (dict(table_out=A + 0x30000 + 4), "table_out"),
    (dict(status=A + 2), "address"), (dict(parents=A + 1), "address"), (dict(free_count=A + 3), "address"),
    (dict(slot=A + 4), "address"), (dict(mask=A + 4), "address"),
])
def test_plan_refusals(kw, word):
    _says("fwhip_paged_plan", _set(_plan, **kw), word)


def test_plan_takes_its_table_in_place_and_empty_batches():
    _says("fwhip_paged_plan", _set(_plan, table_out=A + 0x30000), "NULL ctx")
    _says("fwhip_paged_plan", _set(_plan, n_req=0, n_rows=0, len=None, n_new=None, held=None, held_out=None, status=None,
                                   table=None, table_out=None, row_req=None, pos=None, slot=None, parents=None, mask=None,
                                   mask_words=0), "NULL ctx")


@pytest.mark.parametrize("kw,word", [
    (dict(src_dtype=3), "element type"), (dict(cache_dtype=-1), "element type"), (dict(n_rows=-1), "bad size"),
    (dict(n_heads=0), "bad size"), (dict(head_dim=0), "bad size"), (dict(n_pages=-1), "bad size"),
    (dict(page_size=0), "page_size"), (dict(k_row=-1), "negative stride"), (dict(token_stride=-1), "negative stride"),
    (dict(k=None), "NULL"), (dict(v=None), "NULL"), (dict(slot=None), "NULL"), (dict(k_cache=None), "NULL"),
    (dict(k=A + 2), "address"), (dict(v_cache=5 * A + 1), "address"), (dict(slot=3 * A + 4), "address"),
    (dict(n_rows=1 << 30, n_heads=1024, head_dim=128), "too many"), (dict(n_heads=1 << 30, head_dim=4), "too many"),
])
def test_append_refusals(kw, word):
    _says("fwhip_paged_append", _set(_append, **kw), word)


@pytest.mark.parametrize("kw,word", [
    (dict(dtype=7), "element type"), (dict(n_req=-1), "negative size"), (dict(n_rows=-1), "negative size"),
    (dict(max_new=-1), "negative size"), (dict(max_len=-1), "negative size"), (dict(n_pages=-1), "negative size"),
    (dict(n_heads=7), "n_kv_heads"), (dict(n_kv_heads=0), "n_kv_heads"), (dict(n_heads=0), "n_kv_heads"),
    (dict(page_size=0), "page_size"), (dict(max_len=129), "max_len"), (dict(n_req=65536), "n_req"),
    (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"), (dict(q_row=-8), "negative stride"), (dict(table_stride=-1), "negative stride"), (dict(q=None), "NULL"),
    (dict(table=None), "NULL"), (dict(row_start=None), "NULL"), (dict(len=None), "NULL"), (dict(out=None), "NULL"),
    (dict(k_cache=None), "NULL"), (dict(q=A + 8), "16-byte"), (dict(v_cache=3 * A + 4), "16-byte"),
    (dict(q_head=4), "multiples of 16"), (dict(page_stride=2047), "multiples of 16"), (dict(out=A), "out must not"), (dict(out=A + 16), "out must not"),
    (dict(mask_words=0), "mask"), (dict(max_new=65), "mask"), (dict(mask=None), "mask"),
    (dict(table=A + 2), "address"), (dict(len=A + 1), "address"), (dict(row_start=A + 2), "address"), (dict(mask=A + 4), "address"),
])
def test_attention_refusals(kw, word):
    _says("fwhip_tree_attn", _set(_attn, **kw), word)


def test_attention_head_dims_that_are_not_built():
    for d in (0, 32, 63, 80, 256):
        _says("fwhip_tree_attn", _set(_attn, head_dim=d), "head_dim", abi.ERR_UNSUPPORTED)


def test_attention_strides_past_the_addressing():
    _says("fwhip_tree_attn", _set(_attn, page_stride=1 << 30), "strides", abi.ERR_UNSUPPORTED)
    _says("fwhip_tree_attn", _set(_attn, token_stride=1 << 30), "strides", abi.ERR_UNSUPPORTED)


def test_attention_workspace_is_checked():
    n = C.c_uint64()
    L = native.lib()
    assert L.fwhip_tree_attn_workspace(1, 8, 8, 64, 8, 1 << 20, None) == abi.ERR_INVALID
    assert L.fwhip_tree_attn_workspace(1, 8, 3, 64, 8, 1 << 20, C.byref(n)) == abi.ERR_INVALID
    assert L.fwhip_tree_attn_workspace(1, 8, 8, 65, 8, 1 << 20, C.byref(n)) == abi.ERR_UNSUPPORTED
    sizes = {}
    for n_req in (0, 1, 2, 7, 64, 300):
        for new in (1, 5, 16, 17, 64, 200):
            for ln in (1, 100, 1000, 10000, 100000, 1000000):
                sizes[n_req, new, ln] = ops.tree_attn_workspace(n_req, 32, 8, 128, new, max(ln, new))
    for (a, b, c), x in sizes.items():  # it grows with each of them
        for (d, e, f), y in sizes.items():
            if a <= d and b <= e and c <= f:
                assert x <= y, ((a, b, c), x, (d, e, f), y)
    need = ops.tree_attn_workspace(1, 8, 2, 64, 5, 1 << 20)
    if need:
        big = dict(n_req=1, width=1 << 16, max_len=1 << 20)
        _says("fwhip_tree_attn", _set(_attn, workspace_bytes=need, **big), "NULL ctx")
        _says("fwhip_tree_attn", _set(_attn, workspace_bytes=need - 1, **big), "workspace")
        _says("fwhip_tree_attn", _set(_attn, workspace=None, **big), "workspace")
        _says("fwhip_tree_attn", _set(_attn, workspace=9 * A + 8, **big), "workspace")


@pytest.mark.parametrize("kw,word,code", [
    (dict(dtype=9), "element type", abi.ERR_INVALID), (dict(scale_dtype=abi.T_BF16), "element type", abi.ERR_INVALID),
    (dict(group=16), "group", abi.ERR_UNSUPPORTED), (dict(group=0), "group", abi.ERR_UNSUPPORTED),
    (dict(m=-1), "m, n", abi.ERR_INVALID), (dict(n=-1), "m, n", abi.ERR_INVALID), (dict(k=0), "m, n", abi.ERR_INVALID),
    (dict(k=80), "m, n", abi.ERR_INVALID), (dict(ldx=63), "ldx", abi.ERR_INVALID), (dict(ldy=49), "ldy", abi.ERR_INVALID),
    (dict(x=None), "NULL", abi.ERR_INVALID), (dict(q=None), "NULL", abi.ERR_INVALID), (dict(y=None), "NULL", abi.ERR_INVALID),
    (dict(scale=None), "NULL", abi.ERR_INVALID), (dict(q=2 * A + 8), "16-byte", abi.ERR_INVALID),
    (dict(x=A + 1), "address", abi.ERR_INVALID), (dict(bias=4 * A + 2), "address", abi.ERR_INVALID),
    (dict(y=A), "overlap", abi.ERR_INVALID), (dict(y=A + 2), "overlap", abi.ERR_INVALID),
    (dict(y=A + 128 - 2, ldx=200, ldy=200), "overlap", abi.ERR_INVALID), (dict(y=A - 98, ldx=200, ldy=200), "overlap", abi.ERR_INVALID),
    (dict(y=A + 200, ldx=200, ldy=210), "overlap", abi.ERR_INVALID), (dict(y=A + 128, ldx=114, ldy=114), "NULL ctx", abi.ERR_INVALID),
    (dict(y=A + 126, ldx=114, ldy=114), "overlap", abi.ERR_INVALID), (dict(y=A - 100, ldx=114, ldy=114), "NULL ctx", abi.ERR_INVALID),
    (dict(k=(1 << 24) + 32, ldx=1 << 25), "2^24", abi.ERR_UNSUPPORTED), (dict(n=(1 << 29) + 1, ldy=1 << 30), "2^29", abi.ERR_UNSUPPORTED),
])
def test_linear_refusals(kw, word, code):
    _says("fwhip_q4_linear", _set(_q4, **kw), word, code)


def test_planes_refusals():
    L = native.lib()

    def says(word, dtype=2, raw=A, nbytes=18 * 6, rows=3, k=64, q=2 * A, s=3 * A, m=None, code=abi.ERR_INVALID):
        rc = L.fwhip_q4_planes(None, dtype, raw, nbytes, rows, k, q, s, m)
        msg = L.fwhip_last_error().decode()
        assert rc == code and word in msg, (rc, msg)

    says("NULL ctx")
    says("NULL ctx", dtype=3, nbytes=20 * 6, m=4 * A)
    says("NULL ctx", dtype=12, nbytes=144 * 3, k=256, m=4 * A)
    says("payloads only", dtype=8, code=abi.ERR_UNSUPPORTED)
    says("multiple", k=48)
    says("multiple", dtype=12, k=64, nbytes=144, m=4 * A)
    says("length", nbytes=18 * 6 - 1)
    says("NULL", q=None)
    says("minimums", m=4 * A)
    says("minimums", dtype=3, nbytes=20 * 6)
    says("aligned", raw=A + 2)
    says("aligned", s=3 * A + 8)


def test_init_on_stream_answers_as_init_does():
    h = C.c_void_p()
    assert native.lib().fwhip_init_on_stream(0, None, None) == abi.ERR_INVALID
    import os
    if not os.path.exists("/dev/kfd"):
        assert native.lib().fwhip_init_on_stream(0, None, C.byref(h)) == abi.ERR_UNSUPPORTED
        assert native.lib().fwhip_last_error().decode().startswith("cpu:")


class _Dev:
    """A device array that is nowhere: shape, type and an address."""

    def __init__(self, shape, dtype):
        self.shape, self.dtype, self.ptr, self.nbytes = shape, np.dtype(dtype), A, 1 << 30


class _Ctx:
    h, device = None, 0


def test_python_refuses_tensors_off_the_contexts_device():
    torch = pytest.importorskip("torch")
    x, q, s, y = torch.zeros(2, 64), torch.zeros(8, 32, dtype=torch.uint8), torch.zeros(8, 2).half(), torch.zeros(2, 8)
    with pytest.raises(ValueError, match="x must be on the context's device"):
        ops.q4_linear(_Ctx, x, q, s, y)
    with pytest.raises(ValueError, match="element type torch.float64"):
        ops.q4_linear(_Ctx, x.double(), q, s, y.double())


def test_python_checks_shapes_and_types():
    x, q, s = _Dev((3, 64), "f4"), _Dev((50, 32), "u1"), _Dev((50, 2), "f2")
    for kw, word in ((dict(out=_Dev((3, 49), "f4")), "out"), (dict(out=_Dev((3, 50), "f2")), "out"),
                     (dict(scale=_Dev((50, 3), "f2")), "scale"), (dict(minimum=_Dev((50, 2), "f4")), "minimum"),
                     (dict(q=_Dev((50, 31), "u1")), "q"), (dict(q=_Dev((50, 32), "i1")), "q"),
                     (dict(bias=_Dev((50,), "f2")), "bias"), (dict(bias=_Dev((49,), "f4")), "bias"),
                     (dict(x=_Dev((3, 64), "f8")), "x")):
        a = dict(x=x, q=q, scale=s, out=_Dev((3, 50), "f4"))
        a.update(kw)
        if "x" in kw:
            a["out"] = _Dev((3, 50), "f8")
        with pytest.raises(ValueError, match=word):
            ops.q4_linear(_Ctx, a["x"], a["q"], a["scale"], a["out"], minimum=a.get("minimum"), bias=a.get("bias"))
    k, cache = _Dev((4, 2, 64), "f4"), _Dev((8, 16, 2, 64), "f2")
    with pytest.raises(ValueError, match="one type"):
        ops.paged_append(_Ctx, k, _Dev((4, 2, 64), "f2"), _Dev((4,), "i8"), cache, cache)
    with pytest.raises(ValueError, match="slot"):
        ops.paged_append(_Ctx, k, k, _Dev((4,), "i4"), cache, cache)
    with pytest.raises(ValueError, match="heads of"):
        ops.paged_append(_Ctx, k, k, _Dev((4,), "i8"), _Dev((8, 16, 3, 64), "f2"), _Dev((8, 16, 3, 64), "f2"))
    qa, c4 = _Dev((5, 4, 64), "f2"), _Dev((8, 16, 2, 64), "f2")
    tab, ln, rs = _Dev((2, 8), "i4"), _Dev((2,), "i4"), _Dev((3,), "i4")
    for kw, word in ((dict(out=_Dev((5, 4, 64), "f4")), "out"), (dict(table=_Dev((2, 8), "i8")), "table"),
                     (dict(lens=_Dev((3,), "i4")), "lens"), (dict(row_start=_Dev((2,), "i4")), "row_start"),
                     (dict(mask=_Dev((4, 1), "i8")), "mask"), (dict(mask=_Dev((5, 1), "i4")), "mask"),
                     (dict(k_cache=_Dev((8, 16, 2, 64), "f4"), v_cache=_Dev((8, 16, 2, 64), "f4")), "share"),
                     (dict(v_cache=_Dev((9, 16, 2, 64), "f2")), "one type")):
        a = dict(q=qa, k_cache=c4, v_cache=c4, table=tab, lens=ln, row_start=rs, out=_Dev((5, 4, 64), "f2"), mask=None)
        a.update(kw)
        with pytest.raises(ValueError, match=word):
            ops.tree_attn(_Ctx, a["q"], a["k_cache"], a["v_cache"], a["table"], a["lens"], a["row_start"], a["out"],
                          scale=1.0, max_new=3, mask=a["mask"])
