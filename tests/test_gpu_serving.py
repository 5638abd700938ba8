"""GPU tests of the serving operators (ops.py: paged_plan, paged_append,
tree_attn, q4_linear, q4_planes) against their plain 64-bit forms
(serving_ref.py), whose bounds are derived there."""
import numpy as np
import pytest
import torch

from franken_whisper_amd import abi, native, ops
from oracle import ggml_ref
from tests import serving_ref as R

pytestmark = pytest.mark.gpu

DT = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}


@pytest.fixture(scope="module")
def tctx():
    c = native.Context(0, stream=torch.cuda.current_stream().cuda_stream)
    yield c
    torch.cuda.synchronize()
    c.close()


def dev(a, dtype=None):
    t = torch.from_numpy(np.ascontiguousarray(a))
    return t.to(dtype).cuda() if dtype is not None else t.cuda()


def host(t):
    return t.detach().to(torch.float64).cpu().numpy() if t.is_floating_point() else t.cpu().numpy()


def close(got, want, tol, what=""):
    got = host(got)
    bad = ~(np.abs(got - want) <= tol)
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4], np.asarray(tol)[bad][:4])


# ---------------------------------------------------------------------------
# plan

def run_plan(ctx, lens, n_new, table, held, free, count, page, n_rows, parents=None, words=0, in_place=False, guard=3):
    """The plan on the device; row arrays have `guard` further rows that must stay."""
    n_req = len(lens)
    i32 = lambda a: dev(np.asarray(a, np.int32))  # noqa: E731
    tab = i32(table)
    out = {"table": tab if in_place else torch.full_like(tab, -77), "held": torch.full((n_req,), -77, dtype=torch.int32).cuda(),
           "count": torch.full((1,), -77, dtype=torch.int32).cuda(),
           "row_start": torch.full((n_req + 1,), -77, dtype=torch.int32).cuda(),
           "row_req": torch.full((n_rows + guard,), -77, dtype=torch.int32).cuda(),
           "pos": torch.full((n_rows + guard,), -77, dtype=torch.int32).cuda(),
           "slot": torch.full((n_rows + guard,), -77, dtype=torch.int64).cuda(),
           "status": torch.full((n_req,), -77, dtype=torch.int32).cuda()}
    if parents is not None:
        out["mask"] = torch.full((n_rows + guard, words), -77, dtype=torch.int64).cuda()
    ops.paged_plan(ctx, i32(lens), i32(n_new), tab, i32(held), i32(free), i32([count]), page, table_out=out["table"],
                   held_out=out["held"], count_out=out["count"], row_start=out["row_start"],
                   row_req=out["row_req"][:n_rows], pos=out["pos"][:n_rows], slot=out["slot"][:n_rows],
                   status=out["status"], parents=None if parents is None else i32(parents),
                   mask=out["mask"][:n_rows] if parents is not None else None)
    torch.cuda.synchronize()
    return {k: v.cpu().numpy() for k, v in out.items()}


def check_plan(got, want, n_rows, words):
    for k in ("table", "held", "row_start", "status"):
        assert np.array_equal(got[k], want[k]), (k, got[k], want[k])
    assert got["count"][0] == want["count"]
    for k in ("row_req", "pos", "slot"):
        full = np.full(got[k].shape[0], -77, np.int64)
        for x, v in want[k].items():
            full[x] = v
        assert np.array_equal(got[k], full), (k, got[k], full)
    if words:
        full = np.full(got["mask"].shape, -77, np.int64)
        for x, v in want["mask"].items():
            for w in range(words):
                full[x, w] = np.uint64(v >> 64 * w & (1 << 64) - 1).astype(np.int64)
        assert np.array_equal(got["mask"], full)


def plan_inputs(rng, n_req, ctx, new, page, extra_width, spare, tree):
    lens = rng.integers(0, ctx + 1, n_req)
    n_new = rng.integers(0, new + 1, n_req)
    width = (ctx + new) // page + 1 + extra_width
    held = -(-lens // page) + (rng.random(n_req) < 0.3) * 1
    held = np.minimum(held, width)
    perm = rng.permutation(int(held.sum()) + spare)
    table = np.full((n_req, width), -1, np.int64)
    at = 0
    for r in range(n_req):
        table[r, : held[r]] = perm[at: at + held[r]]
        at += held[r]
    free = perm[at:]
    parents = None
    if tree:
        parents = np.concatenate([[rng.integers(-1, i) if i else -1 for i in range(n)] for n in n_new] + [[]]).astype(int)
    return lens, n_new, table, held, free, parents


@pytest.mark.parametrize("n_req,ctx,new,page,tree,words", [
    (1, 0, 1, 16, False, 0), (1, 30, 8, 16, True, 1), (3, 50, 5, 1, True, 1), (10, 440, 8, 16, True, 1),
    (64, 3000, 64, 24, True, 1), (33, 700, 130, 64, True, 3), (7, 100, 256, 16, True, 4), (5, 90, 1000, 16, False, 0),
    (300, 900, 17, 32, True, 2), (5000, 64, 3, 16, True, 1), (1, 10, 20000, 16, False, 0), (2, 9000, 64, 1, True, 1), (3, 40, 3000, 16, False, 0)])
def test_plan(tctx, n_req, ctx, new, page, tree, words):
    rng = np.random.default_rng(n_req * 7 + new)
    lens, n_new, table, held, free, parents = plan_inputs(rng, n_req, ctx, new, page, 3, 100000, tree)
    n_rows = int(n_new.sum())
    for in_place in (False, True):
        got = run_plan(tctx, lens, n_new, table, held, free, len(free), page, n_rows, parents, words, in_place)
        check_plan(got, R.plan(lens, n_new, table, held, free, len(free), page, n_rows, parents, words), n_rows, words)


def test_plan_chains_as_a_tree(tctx):
    """A chain given by parents has the chain's positions and lower-triangular masks."""
    n = 256
    got = run_plan(tctx, [5], [n], np.full((1, 40), -1), [0], np.arange(40), 40, 16, n, np.arange(n) - 1, 4)
    assert np.array_equal(got["pos"][:n], 5 + np.arange(n))
    for i in (0, 1, 63, 64, 200, 255):
        v = sum(int(np.uint64(got["mask"][i, w].astype(np.uint64))) << 64 * w for w in range(4))
        assert v == (1 << i + 1) - 1


@pytest.mark.parametrize("spare", [0, 1, 2, 5, 9])
def test_plan_with_too_few_pages(tctx, spare):
    rng = np.random.default_rng(spare)
    lens, n_new, table, held, free, parents = plan_inputs(rng, 12, 100, 40, 16, 3, spare, True)
    n_rows = int(n_new.sum())
    got = run_plan(tctx, lens, n_new, table, held, free, len(free), 16, n_rows, parents, 1)
    want = R.plan(lens, n_new, table, held, free, len(free), 16, n_rows, parents, 1)
    assert want["status"].any()
    check_plan(got, want, n_rows, 1)


def test_plan_with_bad_lengths_parents_and_tables(tctx):
    lens = np.array([10, -3, 40, 2 ** 31 - 2, 7, 0, 3, 9])
    n_new = np.array([4, 5, -2, 6, 70, 0, 3, 2])
    held = np.array([1, 1, 3, 2, 1, 9, -1, 1])
    table = np.arange(8 * 6).reshape(8, 6)
    table[7, 0] = -1  # a held entry that is no page
    free = np.arange(100, 140)
    n_rows = int(np.maximum(n_new, 0).sum())
    parents = np.full(n_rows, -1)
    parents[1:4] = (0, 0, 7)  # row 3 names a later token
    for count in (40, 0, -5, 4000):
        want = R.plan(lens, n_new, table, held, free, count, 16, n_rows, parents, 1)
        got = run_plan(tctx, lens, n_new, table, held, free, count, 16, n_rows, parents, 1)
        check_plan(got, want, n_rows, 1)
    assert want["status"].tolist()[:5] == [4, 2, 2, 2, 4]
    # too few row entries: cut
    for n_rows in (0, 1, 7, 20):
        want = R.plan(lens, n_new, table, held, free, 40, 16, n_rows, parents[:n_rows], 1)
        got = run_plan(tctx, lens, n_new, table, held, free, 40, 16, n_rows, parents[:n_rows], 1)
        check_plan(got, want, n_rows, 1)


def test_plan_of_nothing(tctx):
    got = run_plan(tctx, np.zeros(0), np.zeros(0), np.zeros((0, 5)), np.zeros(0), np.arange(9), 7, 16, 0)
    assert got["row_start"].tolist() == [0] and got["count"][0] == 7
    got = run_plan(tctx, [0, 0], [0, 0], np.full((2, 4), -1), [0, 0], np.zeros(0), 0, 16, 0)
    assert got["row_start"].tolist() == [0, 0, 0] and got["status"].tolist() == [0, 0]


# ---------------------------------------------------------------------------
# append

@pytest.mark.parametrize("src", DT)
@pytest.mark.parametrize("dst", DT)
@pytest.mark.parametrize("rows,heads,dim,page", [(1, 1, 64, 16), (9, 20, 64, 16), (130, 2, 128, 24), (33, 3, 5, 1),
                                                 (7, 6, 72, 100)])
def test_append(tctx, src, dst, rows, heads, dim, page):
    g = torch.Generator().manual_seed(rows + dim)
    k = (torch.randn(rows, heads, dim, generator=g) * 3).to(DT[src])
    v = (torch.randn(rows, heads, dim, generator=g) * 300).to(DT[src])
    k[0, 0, :3] = torch.tensor([float("inf"), float("nan"), -1e5]).to(DT[src])
    pages = rows // page + 3
    cache = torch.randn(2, pages, page, heads, dim, generator=g).to(DT[dst])
    slot = torch.randperm(pages * page, generator=g)[:rows]
    if rows > 2:
        slot[1], slot[2] = -1, pages * page
    want = cache.clone().view(2, -1, heads, dim)
    keep = (slot >= 0) & (slot < pages * page)
    want[0][slot[keep]] = k[keep].to(DT[dst])
    want[1][slot[keep]] = v[keep].to(DT[dst])
    want = want.view_as(cache)
    got = cache.cuda()
    ops.paged_append(tctx, k.cuda(), v.cuda(), slot.cuda(), got[0], got[1])
    assert torch.equal(torch.nan_to_num(got.cpu().float(), nan=123.0), torch.nan_to_num(want.float(), nan=123.0))
    # head-major pages, rows of a fused projection, an odd offset
    fused = torch.zeros(rows, 3 * heads * dim + 1).to(DT[src]).cuda()
    kk, vv = fused[:, 1:1 + heads * dim].view(rows, heads, dim), fused[:, 1 + heads * dim:1 + 2 * heads * dim].view(rows, heads, dim)
    kk.copy_(k)
    vv.copy_(v)
    major = cache.cuda().transpose(2, 3).contiguous()
    views = major.transpose(2, 3)
    ops.paged_append(tctx, kk, vv, slot.cuda(), views[0], views[1])
    assert torch.equal(torch.nan_to_num(views.cpu().float(), nan=123.0), torch.nan_to_num(want.float(), nan=123.0))


def test_append_rounds_to_nearest_even(tctx):
    x = torch.tensor([1 + 2.0 ** -11, 1 + 3 * 2.0 ** -11, 1 + 2.0 ** -8, 1 + 3 * 2.0 ** -8, 65519.0, 65520.0, 2.0 ** -25,
                      1.5 * 2.0 ** -24]).view(1, 1, 8)
    for dt in (torch.float16, torch.bfloat16):
        c = torch.zeros(2, 1, 1, 1, 8, dtype=dt).cuda()
        ops.paged_append(tctx, x.cuda(), -x.cuda(), torch.zeros(1, dtype=torch.int64).cuda(), c[0], c[1])
        assert torch.equal(c[0].cpu().view(-1), x.view(-1).to(dt)) and torch.equal(c[1].cpu().view(-1), -x.view(-1).to(dt))


# ---------------------------------------------------------------------------
# attention

def tree_mask(rng, n_new, words, empty=0.0):
    rows = int(sum(n_new))
    mask = np.zeros((rows, words), np.uint64)
    at = 0
    for n in n_new:
        seen = []
        for i in range(n):
            p = int(rng.integers(max(-1, i - 6), i)) if i else -1
            seen.append((seen[p] if p >= 0 else 0) | 1 << i)
            v = 0 if rng.random() < empty else seen[-1]
            for w in range(words):
                mask[at + i, w] = v >> 64 * w & (1 << 64) - 1
        at += n
    return mask


def attn_inputs(seed, kind, lens, n_new, heads, kv, dim, page, tree, words=None, empty=0.0, spare_rows=2, garbage=True):
    """Inputs of one call: pages of other requests, slots behind a request's end
    and entries behind its pages hold infinities and NaN."""
    rng = np.random.default_rng(seed)
    held = [-(-(a + b) // page) for a, b in zip(lens, n_new)]
    total, width = sum(held) + 4, max(held + [1]) + 1
    perm = rng.permutation(total)
    table = np.full((len(lens), width), -5, np.int32)
    g = torch.Generator().manual_seed(seed)
    kc = torch.randn(total, page, kv, dim, generator=g).to(DT[kind])
    vc = torch.randn(total, page, kv, dim, generator=g).to(DT[kind])
    if garbage:
        junk = torch.tensor([float("nan"), float("inf"), -float("inf"), 1e30]).to(DT[kind])
        used = torch.zeros(total, page, dtype=torch.bool)
    at = 0
    for r, h in enumerate(held):
        table[r, :h] = perm[at: at + h]
        at += h
        if garbage:
            for j in range(lens[r] + n_new[r]):
                used[table[r, j // page], j % page] = True
    if garbage:
        idx = torch.arange(total * page * kv * dim).view(total, page, kv, dim) % 4
        kc = torch.where(used[:, :, None, None], kc, junk[idx])
        vc = torch.where(used[:, :, None, None], vc, junk[idx])
    rows = sum(n_new)
    q = (torch.randn(rows + spare_rows, heads, dim, generator=g) * 1.7).to(DT[kind])
    row_start = np.concatenate([[0], np.cumsum(n_new)]).astype(np.int32)
    mask = None
    if tree:
        words = words or -(-max(n_new + [1]) // 64)
        mask = np.concatenate([tree_mask(rng, n_new, words, empty), np.zeros((spare_rows, words), np.uint64)])
    return dict(kind=kind, q=q, kc=kc, vc=vc, table=table, lens=np.asarray(lens, np.int32), row_start=row_start, mask=mask,
                scale=1.3 / np.sqrt(dim), max_new=max(n_new + [0]), max_len=max([a + b for a, b in zip(lens, n_new)] + [0]))


def reference(s):
    f = lambda t: t.to(torch.float64).numpy()  # noqa: E731
    return R.attn(f(s["q"]), f(s["kc"]), f(s["vc"]), s["table"], s["lens"], s["row_start"], s["mask"], np.float32(s["scale"]).astype(float), s["kind"])


def run_attn(ctx, s, max_new=None, max_len=None, sync=True):
    q = s["q"].cuda()
    out = torch.full_like(q, 7.5)
    n_req = len(s["lens"])
    max_new = s["max_new"] if max_new is None else max_new
    max_len = s["max_len"] if max_len is None else max_len
    need = ops.tree_attn_workspace(n_req, q.shape[1], s["kc"].shape[2], q.shape[2], max_new, max_len)
    ws = torch.full((need,), 255, dtype=torch.uint8).cuda()  # NaN wherever it is read before it is written
    ops.tree_attn(ctx, q, s["kc"].cuda(), s["vc"].cuda(), dev(s["table"]), dev(s["lens"]), dev(s["row_start"]), out,
                  scale=s["scale"], max_new=max_new, max_len=max_len,
                  mask=None if s["mask"] is None else dev(s["mask"].astype(np.int64)), workspace=ws if need else None)
    if sync:
        torch.cuda.synchronize()
    return out


def check_attn(ctx, s, **kw):
    want, tol = reference(s)
    got = run_attn(ctx, s, **kw)
    rows = int(s["row_start"][-1])
    close(got[:rows], want[:rows], tol[:rows], "attention")
    assert (got[rows:] == 7.5).all(), "rows behind the last were written"
    return got


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("lens,n_new,heads,kv,dim,page,tree", [
    ([0], [1], 1, 1, 64, 16, True),                        # one key: the token itself
    ([1], [1], 4, 2, 64, 16, False),
    ([15, 16, 17], [1, 1, 1], 6, 6, 64, 16, False),        # pages' edges
    ([217], [8], 20, 20, 64, 16, True),
    ([0, 5, 0, 33], [3, 0, 7, 16], 8, 2, 64, 16, True),    # empty caches, a request without rows
    ([31, 32, 33, 63, 64, 65, 127, 128, 129], [2] * 9, 2, 2, 128, 24, True),
    ([300, 1], [17, 33], 8, 1, 128, 100, True),            # one K/V head for all
    ([500], [64], 4, 4, 64, 1, True),                      # pages of one token
    ([700, 90], [65, 130], 3, 1, 64, 32, True),            # masks of several words
    ([0, 40], [100, 37], 4, 2, 128, 16, False),            # prompts as chains
    ([2100], [5], 16, 2, 128, 64, True),
    ([505, 511, 600, 637, 0], [8, 1, 40, 3, 2], 8, 2, 128, 16, True), # the edges of where and how the keys are cut
    ([504], [8], 4, 4, 64, 16, True), ([505], [8], 4, 4, 64, 16, True), ([1016, 3], [8, 1], 8, 1, 64, 32, True),
    ([0, 300], [520, 230], 4, 2, 64, 16, False),
    ([1500, 10, 260], [1, 1, 1], 32, 4, 128, 16, False),   # single tokens
])
def test_attention(tctx, kind, lens, n_new, heads, kv, dim, page, tree):
    check_attn(tctx, attn_inputs(len(lens) * 100 + heads, kind, lens, n_new, heads, kv, dim, page, tree))


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("lens,n_new", [([6000], [9]), ([4097, 12, 2000], [3, 16, 40]), ([9000], [1])])
def test_attention_over_a_long_cache(tctx, kind, lens, n_new):
    s = attn_inputs(5, kind, lens, n_new, 8, 2, 64, 16, True)
    a = check_attn(tctx, s)
    assert torch.equal(a, run_attn(tctx, s))  # and the same bits every time
    # looser bounds cost time, not results
    check_attn(tctx, s, max_new=64, max_len=s["table"].shape[1] * 16)


@pytest.mark.parametrize("kind", DT)
def test_attention_rows_whose_mask_is_empty(tctx, kind):
    s = attn_inputs(8, kind, [0, 70, 0], [20, 18, 5], 4, 2, 64, 16, True, empty=0.5)
    got = check_attn(tctx, s)
    empty = (s["mask"][:20] == 0).all(1)
    assert empty.any() and (got[:20][torch.from_numpy(empty).cuda()] == 0).all()


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("dim", [64, 128])
def test_attention_unseen_tokens_never_reach_a_row(tctx, kind, dim):
    """Drafted tokens that hold NaN and infinities: only rows whose mask names them change."""
    s = attn_inputs(9, kind, [37, 250], [24, 70], 4, 2, dim, 16, True)
    rng = np.random.default_rng(1)
    spoiled = []
    for r, t, what in ((0, 3, float("nan")), (0, 10, float("inf")), (1, 0, -float("inf")), (1, 66, float("nan")), (1, 35, float("inf"))):
        j = int(s["lens"][r]) + t
        pg = int(s["table"][r, j // 16])
        e = int(rng.integers(dim))
        s["kc" if t == 10 else "vc"][pg, j % 16, :, e] = what
        spoiled.append((r, t))
    want, tol = reference(s)
    got = host(run_attn(tctx, s))
    clean = 0
    for i in range(int(s["row_start"][-1])):
        r = 0 if i < 24 else 1
        hit = any(rr == r and int(s["mask"][i, t >> 6]) >> (t & 63) & 1 for rr, t in spoiled)
        fin = np.isfinite(want[i])
        if not hit:
            assert fin.all()
            clean += 1
        assert np.array_equal(np.isfinite(got[i]), fin), (i, hit)
        assert np.array_equal(np.isnan(got[i]), np.isnan(want[i]))
        assert (got[i][~fin & ~np.isnan(want[i])] == want[i][~fin & ~np.isnan(want[i])]).all()
        assert (np.abs(got[i][fin] - want[i][fin]) <= tol[i][fin]).all()
    assert 5 < clean < 90


@pytest.mark.parametrize("kind", DT)
def test_attention_infinite_scores(tctx, kind):
    """A key of -inf scores -inf and drops out; if all of a row's keys do, the softmax is 0 / 0."""
    s = attn_inputs(10, kind, [3, 40], [1, 1], 2, 2, 64, 16, False, garbage=False)
    s["q"][:, :, 0] = s["q"][:, :, 0].abs() + 0.5
    for r, js in ((0, range(4)), (1, (0, 7, 39))):
        for j in js:
            s["kc"][int(s["table"][r, j // 16]), j % 16, :, 0] = -float("inf")
    want, tol = reference(s)
    got = host(run_attn(tctx, s))
    assert np.isnan(got[0]).all()
    assert (np.abs(got[1] - want[1]) <= tol[1]).all()
    # equal scores of the type's lowest value are an even mean
    s = attn_inputs(11, kind, [5], [1], 2, 2, 64, 16, False, garbage=False)
    s["kc"][:] = 0
    s["kc"][..., 0] = torch.finfo(DT[kind]).min / (2.0 ** 10 if kind != "f16" else 1)
    s["q"][:] = 0
    s["q"][..., 0] = 1.0
    check_attn(tctx, s)


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("scale", [-0.2, 0.0, 1e-3, 2.0])
def test_attention_scales(tctx, kind, scale):
    """Negative scales, zero (the mean of what a row sees) and sharp ones."""
    for n_new, heads in (([5, 9], 2), ([30, 60], 4)):
        s = attn_inputs(30, kind, [77, 300], n_new, heads, 2, 64, 16, True, empty=0.2)
        s["scale"] = scale
        check_attn(tctx, s)


def test_attention_bad_requests_come_out_as_nan(tctx):
    s = attn_inputs(12, "f16", [40, 50, 60, 70, 20], [3, 4, 5, 2, 1], 4, 2, 64, 16, True)
    want, tol = reference(s)
    for bad in ("page", "negative page", "length", "long", "rows"):
        b = {k: (v.copy() if isinstance(v, np.ndarray) else v) for k, v in s.items()}
        kw = {}
        hit = 2
        if bad == "page":
            b["table"][2, 1] = b["kc"].shape[0]
        elif bad == "negative page":
            b["table"][2, 3] = -1
        elif bad == "length":
            b["lens"][2] = -1
        elif bad == "long":
            b["lens"][2] = 1000
        else:
            kw, hit = {"max_new": 4}, 2
        got = host(run_attn(tctx, b, **kw))
        for r in range(5):
            a, e = s["row_start"][r], s["row_start"][r + 1]
            if r == hit:
                assert np.isnan(got[a:e]).all(), bad
            else:
                assert (np.abs(got[a:e] - want[a:e]) <= tol[a:e]).all(), (bad, r)
    # row starts past the rows: cut, nothing outside is touched
    b = dict(s, row_start=np.array([0, 3, 7, 12, 14, 4000], np.int32))
    got = host(run_attn(tctx, b))
    assert (np.abs(got[:14] - want[:14]) <= tol[:14]).all()


def test_attention_strides(tctx):
    """q and out inside fused rows, head-major pages, K and V in one allocation."""
    s = attn_inputs(13, "bf16", [100, 33], [9, 20], 8, 2, 64, 16, True, spare_rows=0)
    want, tol = reference(s)
    rows = s["q"].shape[0]
    fused = torch.full((rows, 12, 64), 3.0, dtype=torch.bfloat16).cuda()
    fused[:, :8] = s["q"].cuda()
    both = torch.stack([s["kc"], s["vc"]], 1).cuda().transpose(2, 3).contiguous()  # [page, k/v, head, token, dim]
    kc, vc = both[:, 0].transpose(1, 2), both[:, 1].transpose(1, 2)
    buf = torch.full((rows, 3, 8, 64), 7.5, dtype=torch.bfloat16).cuda()
    table = torch.full((2, 50), -9, dtype=torch.int32).cuda()
    table[:, : s["table"].shape[1]] = dev(s["table"])
    ops.tree_attn(tctx, fused[:, :8], kc, vc, table[:, : s["table"].shape[1]], dev(s["lens"]), dev(s["row_start"]), buf[:, 1],
                  scale=s["scale"], max_new=20, max_len=s["max_len"], mask=dev(s["mask"].astype(np.int64)))
    close(buf[:, 1], want, tol)
    assert (buf[:, 0] == 7.5).all() and (buf[:, 2] == 7.5).all()


def test_attention_offsets_past_32_bits(tctx):
    """A pool of over 2^32 bytes and 2^31 elements, the request's pages at both ends."""
    page, kv, dim = 64, 8, 128
    total = (1 << 31) // (page * kv * dim) + 40
    s = attn_inputs(14, "f16", [300], [6], 16, kv, dim, page, True, spare_rows=0)
    kc = torch.zeros(total, page, kv, dim, dtype=torch.float16, device="cuda")
    vc = torch.zeros_like(kc)
    ids = torch.tensor([total - 1, 0, total - 17, 3, total - 2])
    n = 5
    old = torch.from_numpy(s["table"][0, :n].astype(np.int64))
    kc[ids.cuda()] = s["kc"][old].cuda()
    vc[ids.cuda()] = s["vc"][old].cuda()
    want, tol = reference(s)
    table = ids.to(torch.int32).view(1, n).cuda()
    out = torch.empty_like(s["q"]).cuda()
    ops.tree_attn(tctx, s["q"].cuda(), kc, vc, table, dev(s["lens"]), dev(s["row_start"]), out, scale=s["scale"],
                  max_new=6, mask=dev(s["mask"].astype(np.int64)),
                  workspace=torch.empty(ops.tree_attn_workspace(1, 16, kv, dim, 6, n * page) + 16, dtype=torch.uint8).cuda())
    close(out, want, tol)
    # the same slots written by append
    kc[total - 1] = 0
    slot = (torch.arange(page) + (total - 1) * page).cuda()
    ops.paged_append(tctx, s["kc"][int(old[0])].cuda(), s["vc"][int(old[0])].cuda(), slot, kc, vc)
    assert torch.equal(kc[total - 1].cpu(), s["kc"][int(old[0])])


# ---------------------------------------------------------------------------
# 4-bit linear

def q4_inputs(seed, kind, m, n, k, group, minimum, bias, sdt="f16"):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    scale = ((0.5 + torch.rand(n, k // group, generator=g)) / k ** 0.5).to(DT[sdt])
    mn = (scale.float() * -(6 + 3 * torch.rand(n, k // group, generator=g))).to(DT[sdt]) if minimum else None
    x = torch.randn(m, k, generator=g).to(DT[kind])
    return x, q, scale, mn, torch.randn(n, generator=g) if bias else None


def check_q4(ctx, kind, x, q, scale, mn, b, group, pad=0):
    m, k, n = x.shape[0], x.shape[1], q.shape[0]
    h = lambda t: None if t is None else t.to(torch.float64).numpy()  # noqa: E731
    want, tol = R.q4(h(x), q.numpy(), h(scale), h(mn), h(b), group, kind)
    c = lambda t: None if t is None else t.cuda()  # noqa: E731
    xb = torch.full((m, k + pad), float("nan"), dtype=x.dtype).cuda()
    xb[:, pad:] = x.cuda()
    yb = torch.full((m + 1, n + 2 * pad + 1), 7.5, dtype=x.dtype).cuda()
    y = yb[:m, pad:pad + n]
    ops.q4_linear(ctx, xb[:, pad:], c(q), c(scale), y, group=group, minimum=c(mn), bias=c(b))
    close(y, want, tol, (kind, m, n, k, group))
    assert (yb[m:] == 7.5).all() and (yb[:, :pad] == 7.5).all() and (yb[:, pad + n:] == 7.5).all()


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("m,n,k,group,minimum,bias,sdt,pad", [
    (1, 1, 32, 32, False, False, "f16", 0), (1, 17, 64, 32, True, True, "f16", 0), (2, 1280, 1280, 32, False, True, "f16", 0),
    (5, 33, 96, 32, True, False, "f32", 3), (8, 130, 128, 64, False, True, "f16", 8), (15, 64, 320, 64, True, True, "f32", 1),
    (16, 257, 1280, 128, True, False, "f16", 0), (17, 48, 224, 32, False, False, "f16", 8), (31, 100, 640, 128, False, True, "f32", 0),
    (33, 65, 1024, 32, True, True, "f16", 0), (64, 96, 512, 64, False, False, "f16", 5), (65, 31, 384, 128, True, True, "f16", 0),
    (130, 200, 160, 32, True, True, "f16", 16), (300, 129, 256, 32, False, True, "f32", 0), (1, 5120, 5120, 32, False, True, "f16", 0),
    (3, 16, 8192, 128, True, False, "f16", 0),
    # one of each form: few and many outputs, short and long rows, several row tiles
    (10, 33000, 192, 32, True, True, "f16", 3), (16, 32777, 1152, 128, False, False, "f32", 0), (10, 10300, 160, 32, True, True, "f16", 0), (9, 11000, 2112, 64, False, True, "f16", 0), (16, 21000, 2176, 128, True, False, "f16", 0),
    (20, 1000, 1056, 32, True, True, "f16", 8), (32, 4100, 288, 32, False, False, "f32", 0), (27, 8300, 384, 128, True, True, "f16", 0),
    (50, 1281, 160, 32, False, True, "f16", 0), (90, 3850, 224, 32, True, True, "f32", 0), (61, 5130, 320, 64, False, False, "f16", 8),
    (130, 5140, 192, 32, True, False, "f16", 0), (1030, 4097, 256, 64, True, True, "f16", 0), (700, 1600, 544, 32, False, True, "f16", 8), (200, 1300, 640, 128, True, True, "f16", 0)])
def test_q4_linear(tctx, kind, m, n, k, group, minimum, bias, sdt, pad):
    check_q4(tctx, kind, *q4_inputs(m + n, kind, m, n, k, group, minimum, bias, sdt), group, pad)


@pytest.mark.parametrize("kind", DT)
def test_q4_linear_values_far_apart(tctx, kind):
    """Rows of very different sizes, zeros, subnormal and huge values, and a
    non-finite value that must stay in its own row."""
    x, q, s, mn, b = q4_inputs(3, kind, 20, 70, 256, 32, True, True)
    x[0] *= 1e-4
    x[1] *= 200
    x[2] = 0
    if kind != "f16":
        x[3] *= 1e-30
        x[4] *= 1e30
    check_q4(tctx, kind, x, q, s, mn, b, 32)
    clean = torch.empty(20, 70, dtype=DT[kind]).cuda()
    args = [t.cuda() for t in (q, s)]
    ops.q4_linear(tctx, x.cuda(), *args, clean, minimum=mn.cuda(), bias=b.cuda())
    x[5, 100], x[7, 255], x[9, 0] = float("nan"), float("inf"), -float("inf")
    y = torch.empty_like(clean)
    ops.q4_linear(tctx, x.cuda(), *args, y, minimum=mn.cuda(), bias=b.cuda())
    for i in range(20):
        if i in (5, 7, 9):
            assert not torch.isfinite(y[i]).all()
            assert torch.isnan(y[i]).all() if i == 5 else True
        else:
            assert torch.equal(y[i], clean[i])
    # an infinite input gives what the sum of products gives: infinite with the weight's sign, NaN for a zero weight
    w, _ = R.q4_weights(q.numpy(), s.double().numpy(), mn.double().numpy(), 32)
    for i, e, sign in ((7, 255, 1), (9, 0, -1)):
        got = host(y[i])
        exact_inf = np.isinf(got)
        assert (np.sign(got[exact_inf]) == sign * np.sign(w[exact_inf, e])).all()


@pytest.mark.parametrize("kind", DT)
@pytest.mark.parametrize("m,n,k,group,minimum", [(3, 40, 512, 128, True), (20, 40, 1024, 128, False), (70, 100, 256, 32, True)])
def test_q4_linear_near_the_ends_of_the_type(tctx, kind, m, n, k, group, minimum):
    """Sums that overflow on their way to a finite result, and inputs below the
    type's normal numbers (every sum counts what each of them is worth)."""
    x, q, s, mn, b = q4_inputs(m, kind, m, n, k, group, minimum, False, "f32")
    if kind == "f16":
        x = (x.clamp(-4, 4) * 2.0 ** -18).to(torch.float16)  # steps of 2^-24: few bits each, all exact in the oracle too
        s, mn = s * 2.0 ** 12, None if mn is None else mn * 2.0 ** 12
    else:
        x = (x.float() * 2.0 ** 124).clamp(-2.0 ** 126, 2.0 ** 126).to(DT[kind])
        s, mn = s * 2.0 ** -20, None if mn is None else mn * 2.0 ** -20
    check_q4(tctx, kind, x, q, s, mn, b, group)


def test_attention_scale_zero_beside_infinities(tctx):
    """A scale of zero weighs all seen keys alike; rows in one tile with a row
    that is not finite give what they give alone."""
    s = attn_inputs(31, "f32", [40], [4], 4, 1, 64, 16, False)
    s["scale"] = 0.0
    rs = s["row_start"]
    s["q"][int(rs[0])] = 3e38
    want, tol = reference(s)
    s["q"][int(rs[0]) + 2, 1, 5] = float("inf")
    got = run_attn(tctx, s)
    for i in range(4):
        for h in range(4):
            if (i, h) == (2, 1):
                assert torch.isnan(got[int(rs[0]) + i, h]).all()
            else:
                d = np.abs(host(got[int(rs[0]) + i, h]) - want[int(rs[0]) + i, h])
                assert (d <= tol[int(rs[0]) + i, h]).all(), (i, h, d.max())


def test_q4_linear_of_nothing(tctx):
    _, q, s, _, _ = q4_inputs(4, "f32", 1, 8, 64, 32, False, False)
    ops.q4_linear(tctx, torch.empty(0, 64).cuda(), q.cuda(), s.cuda(), torch.empty(0, 8).cuda())
    ops.q4_linear(tctx, torch.empty(3, 64).cuda(), q[:0].cuda(), s[:0].cuda(), torch.empty(3, 0).cuda())


@pytest.mark.parametrize("name,dtype,per,size", [("q4_0", 2, 32, 18), ("q4_1", 3, 32, 20), ("q4_k", 12, 256, 144)])
@pytest.mark.parametrize("rows,k", [(1, 256), (37, 768), (300, 1280)])
def test_q4_planes_of_ggml_payloads(tctx, name, dtype, per, size, rows, k):
    """The planes hold the weights that fwhip_dequant gives, and the linear on
    them the product with the dequantized matrix."""
    rng = np.random.default_rng(rows)
    nb = rows * k // per
    raw = rng.integers(0, 256, (nb, size), dtype=np.uint8)
    halves = 2 if dtype != 2 else 1
    raw[:, : 2 * halves] = (rng.random((nb, halves)) * 0.1 + 0.01).astype(np.float16).view(np.uint8).reshape(nb, -1)
    raw = raw.reshape(-1)
    q = torch.zeros(rows, k // 2, dtype=torch.uint8).cuda()
    sdt = torch.float32 if dtype == 12 else torch.float16
    s = torch.zeros(rows, k // 32, dtype=sdt).cuda()
    mn = torch.zeros_like(s) if dtype != 2 else None
    ops.q4_planes(tctx, dtype, dev(raw), raw.size, rows, k, q, s, mn)
    want = {2: ggml_ref.dequant_q4_0, 3: ggml_ref.dequant_q4_1, 12: ggml_ref.dequant_q4_k}[dtype](raw, rows * k)
    w, mag = R.q4_weights(q.cpu().numpy(), host(s), None if mn is None else host(mn), 32)
    assert (np.abs(w - want.reshape(rows, k)) <= 2 * 2.0 ** -24 * mag).all()  # two roundings of the f32 decode
    x = torch.randn(4, k, generator=torch.Generator().manual_seed(1))
    check_q4(tctx, "f32", x, q.cpu(), s.cpu(), None if mn is None else mn.cpu(), None, 32)


# ---------------------------------------------------------------------------
# together, captured, on other streams

class Step:
    """One layer's drafted step as a program runs it: plan, 4-bit q/k/v, append,
    attention, 4-bit output projection."""

    def __init__(self, ctx, seed=0, kind="f16"):
        g = torch.Generator().manual_seed(seed)
        self.ctx, self.kind = ctx, kind
        self.n_req, self.h, self.kv, self.d, self.page, self.width, self.cap = 3, 4, 2, 64, 16, 8, 24
        self.dim = 256
        o = self.h + 2 * self.kv
        self.wq = torch.randint(0, 256, (o * self.d, self.dim // 2), generator=g, dtype=torch.uint8).cuda()
        self.ws = (torch.rand(o * self.d, self.dim // 32, generator=g) / 64 + 0.005).half().cuda()
        self.oq = torch.randint(0, 256, (self.dim, self.h * self.d // 2), generator=g, dtype=torch.uint8).cuda()
        self.os = (torch.rand(self.dim, self.h * self.d // 32, generator=g) / 64 + 0.005).half().cuda()
        self.kc = torch.zeros(self.n_req * self.width, self.page, self.kv, self.d, dtype=DT[kind]).cuda()
        self.vc = torch.zeros_like(self.kc)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32).cuda()  # noqa: E731
        self.table, self.held, self.held2 = torch.full((self.n_req, self.width), -1, dtype=torch.int32).cuda(), i32(self.n_req), i32(self.n_req)
        self.free = torch.randperm(self.kc.shape[0], generator=g).int().cuda()
        self.count, self.count2 = torch.tensor([self.kc.shape[0]], dtype=torch.int32).cuda(), i32(1)
        self.lens, self.new, self.parents = i32(self.n_req), i32(self.n_req), i32(self.cap)
        self.row_start, self.row_req, self.pos, self.status = i32(self.n_req + 1), i32(self.cap), i32(self.cap), i32(self.n_req)
        self.slot = torch.full((self.cap,), -1, dtype=torch.int64).cuda()
        self.mask = torch.zeros(self.cap, 1, dtype=torch.int64).cuda()
        self.x = torch.zeros(self.cap, self.dim, dtype=DT[kind]).cuda()
        self.qkv = torch.zeros(self.cap, o, self.d, dtype=DT[kind]).cuda()
        self.att = torch.zeros(self.cap, self.h, self.d, dtype=DT[kind]).cuda()
        self.y = torch.zeros(self.cap, self.dim, dtype=DT[kind]).cuda()
        need = ops.tree_attn_workspace(self.n_req, self.h, self.kv, self.d, 16, self.width * self.page)
        self.work = torch.zeros(max(need, 16), dtype=torch.uint8).cuda()

    def set(self, lens, new, seed):
        g = torch.Generator().manual_seed(seed)
        self.lens.copy_(torch.tensor(lens))
        self.new.copy_(torch.tensor(new))
        par = torch.full((self.cap,), -1)
        at = 0
        for n in new:
            for i in range(1, n):
                par[at + i] = int(torch.randint(-1, i, (1,), generator=g))
            at += n
        self.parents.copy_(par)
        self.x.copy_(torch.randn(self.cap, self.dim, generator=g))

    def run(self):
        c, h, kv = self.ctx, self.h, self.kv
        self.slot.fill_(-1)  # rows past this step's have no slot
        ops.paged_plan(c, self.lens, self.new, self.table, self.held, self.free, self.count, self.page, table_out=self.table,
                       held_out=self.held2, count_out=self.count2, row_start=self.row_start, row_req=self.row_req,
                       slot=self.slot, pos=self.pos, status=self.status, parents=self.parents, mask=self.mask)
        self.held.copy_(self.held2)
        self.count.copy_(self.count2)
        ops.q4_linear(c, self.x, self.wq, self.ws, self.qkv.view(self.cap, -1))
        ops.paged_append(c, self.qkv[:, h:h + kv], self.qkv[:, h + kv:], self.slot, self.kc, self.vc)
        ops.tree_attn(c, self.qkv[:, :h], self.kc, self.vc, self.table, self.lens, self.row_start, self.att,
                      scale=self.d ** -0.5, max_new=16, mask=self.mask, workspace=self.work)
        ops.q4_linear(c, self.att.view(self.cap, -1), self.oq, self.os, self.y)


STEPS = [([0, 0, 0], [16, 3, 5], 1), ([12, 3, 2], [4, 4, 1], 2), ([13, 7, 3], [8, 0, 16], 3), ([16, 7, 19], [1, 1, 1], 4),
         ([17, 8, 20], [16, 2, 6], 5), ([30, 9, 21], [8, 8, 8], 6)]


def dense_step(hist, step, lens, new, parents, x):
    """The same step in 64 bits over dense lists of K/V rows."""
    f = lambda t: t.double().cpu().numpy()  # noqa: E731
    h, kv, d = step.h, step.kv, step.d
    w, _ = R.q4_weights(step.wq.cpu().numpy(), f(step.ws), None, 32)
    o, _ = R.q4_weights(step.oq.cpu().numpy(), f(step.os), None, 32)
    qkv = (x @ w.T).reshape(-1, h + 2 * kv, d)
    out, at = [], 0
    for r, n in enumerate(new):
        keys, vals = hist[r]
        keys, vals = keys[: lens[r]], vals[: lens[r]]
        keys = keys + [qkv[at + i, h:h + kv] for i in range(n)]
        vals = vals + [qkv[at + i, h + kv:] for i in range(n)]
        hist[r] = (keys, vals)
        for i in range(n):
            seen = list(range(lens[r]))
            j = i
            while j >= 0:
                seen.append(lens[r] + j)
                j = int(parents[at + j])
            row = np.zeros((h, d))
            for a in range(h):
                k = np.array([keys[s][a // (h // kv)] for s in seen])
                v = np.array([vals[s][a // (h // kv)] for s in seen])
                z = k @ qkv[at + i, a] * d ** -0.5
                p = np.exp(z - z.max())
                row[a] = p @ v / p.sum()
            out.append(row.reshape(-1) @ o.T)
        at += n
    return np.array(out)


@pytest.mark.parametrize("kind", DT)
def test_the_operators_as_one_step(tctx, kind):
    """Six steps with tokens taken back between them, against a dense 64-bit
    form.  Each value passes four roundings of the type (x is exact): q/k/v and
    the attention's output are inputs of the next product, so y is off by at
    most a few half steps of the products' magnitude: 16 half steps of the
    largest row value, plus the f32 form's own error."""
    st = Step(tctx, kind=kind)
    hist = [([], []) for _ in range(st.n_req)]
    for lens, new, seed in STEPS:
        st.set(lens, new, seed)
        st.run()
        torch.cuda.synchronize()
        assert not st.status.any()
        rows = sum(new)
        want = dense_step(hist, st, lens, new, st.parents.cpu().numpy(), host(st.x))
        got = host(st.y)[:rows]
        assert np.abs(got - want).max() <= (16 * R.EPS[kind] + 2.0 ** -19) * np.abs(want).max()
        # positions are the lengths plus the depth
        pos, par, at = st.pos.cpu().numpy(), st.parents.cpu().numpy(), 0
        for r, n in enumerate(new):
            for i in range(n):
                depth, j = 0, int(par[at + i])
                while j >= 0:
                    depth, j = depth + 1, int(par[at + j])
                assert pos[at + i] == lens[r] + depth
            at += n


def test_a_captured_step_replays(tctx):
    """The step captured into a graph on a stream of its own, replayed over
    changing inputs with eager work in between, against the eager step."""
    eager = Step(tctx, seed=2)
    side = torch.cuda.Stream()
    cctx = native.Context(0, stream=side.cuda_stream)
    cap = Step(cctx, seed=2)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cap.run()
    torch.cuda.synchronize()
    cap.table.fill_(-1)  # the capture ran nothing; begin where the eager one does
    for lens, new, seed in STEPS:
        for s in (eager, cap):
            s.set(lens, new, seed)
        eager.run()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        rows = sum(new)
        for name in ("table", "held", "count", "row_start"):
            assert torch.equal(getattr(eager, name), getattr(cap, name)), name
        assert torch.equal(eager.slot[:rows], cap.slot[:rows])
        assert torch.equal(eager.y[:rows], cap.y[:rows])
        assert torch.equal(eager.kc, cap.kc) and torch.equal(eager.vc, cap.vc)
    del graph
    torch.cuda.synchronize()
    cctx.close()


def test_two_streams_at_once(tctx):
    """Two contexts on two streams, each with its own workspace, interleaved."""
    streams = [torch.cuda.Stream() for _ in range(2)]
    ctxs = [native.Context(0, stream=s.cuda_stream) for s in streams]
    ins = [attn_inputs(20 + i, "f16", [5000 + 900 * i, 40], [7, 16], 8, 2, 128, 16, True) for i in range(2)]
    want = [run_attn(tctx, s) for s in ins]
    torch.cuda.synchronize()
    for _ in range(5):
        got = []
        for i in range(2):
            with torch.cuda.stream(streams[i]):
                got.append(run_attn(ctxs[i], ins[i], sync=False))
        torch.cuda.synchronize()
        for i in range(2):
            assert torch.equal(got[i], want[i])
    for c in ctxs:
        c.close()


def test_a_context_of_its_own_and_device_arrays(ctx):
    """The same operators on the context's stream with native.DeviceArray."""
    x, q, s, _, b = q4_inputs(6, "f32", 4, 40, 128, 32, False, True)
    y = ctx.empty((4, 40), np.float32)
    ops.q4_linear(ctx, ctx.array(x.numpy()), ctx.array(q.numpy()), ctx.array(s.numpy()), y, bias=ctx.array(b.numpy()))
    want, tol = R.q4(x.double().numpy(), q.numpy(), s.double().numpy(), None, b.double().numpy(), 32, "f32")
    assert (np.abs(y.download() - want) <= tol).all()
    a = attn_inputs(7, "f32", [20, 0], [4, 3], 4, 2, 64, 16, True, spare_rows=0)
    out = ctx.empty(a["q"].shape, np.float32)
    need = ops.tree_attn_workspace(2, 4, 2, 64, 4, 24)
    ops.tree_attn(ctx, ctx.array(a["q"].numpy()), ctx.array(a["kc"].numpy()), ctx.array(a["vc"].numpy()), ctx.array(a["table"]),
                  ctx.array(a["lens"]), ctx.array(a["row_start"]), out, scale=a["scale"], max_new=4, max_len=24,
                  mask=ctx.array(a["mask"]), workspace=ctx.empty((need,), np.uint8) if need else None)
    want, tol = reference(a)
    assert (np.abs(out.download() - want) <= tol).all()


def test_a_context_on_the_callers_stream_decodes(ctx):
    """fwhip_init_on_stream is a whole context: the decoder gives the same tokens on it."""
    from franken_whisper_amd import synth

    m = synth.Model(synth.MICRO_ML, seed=1)
    states = synth.encoder_states(3, 1, m.cfg.n_audio_ctx, m.cfg.n_text_state)
    toks = []
    side = torch.cuda.Stream()
    for c in (ctx, native.Context(0, stream=0), native.Context(0, stream=side.cuda_stream)):
        d = native.Decoder(c, m, abi.DEC_INT8)
        st = d.state(1, m.cfg.n_audio_ctx)
        st.set_cross(c.array(np.ascontiguousarray(states, np.float32)))
        toks.append(st.greedy(m.tokens.sot_sequence(), 16, m.tokens.filter())[0].tolist())
        st.close()
        d.close()
        if c is not ctx:
            c.close()
    assert toks[0] == toks[1] == toks[2]
