"""The serving operators of a decoder with drafted tokens, as measurable cases.

  plan    block tables, slot maps, positions and ancestor masks of a step from
          the requests' lengths and the drafted tokens' parents (ops.paged_plan)
  append  a step's K/V rows into a paged cache (ops.paged_append)
  attn    attention of drafted trees, or of a causal chain of new tokens, over
          a paged cache (ops.tree_attn)
  q4      a linear with 4-bit weights and group scales (ops.q4_linear)

With `own` false every operator runs in its plain form: elementary torch
operations in 32 bits, rounded once at the end.
"""
import math

import torch

own = False

DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}


def listed():
    return [
        # ten streams of the text decoder (448 positions), eight drafted tokens each: all latency
        {"name": "plan_10", "op": "plan", "n_req": 10, "ctx": 400, "new": 8, "page": 16, "width": 28, "tree": True},
        # a large serving batch with long tables
        {"name": "plan_1024", "op": "plan", "n_req": 1024, "ctx": 32000, "new": 64, "page": 16, "width": 2048,
         "tree": True},
        # one drafted tree of one stream into the f16 cache, from the f32 rows of the decoder
        {"name": "append_8", "op": "append", "rows": 8, "heads": 20, "dim": 64, "page": 16, "src": "f32",
         "dst": "f16"},
        # a batch of prompts
        {"name": "append_16384", "op": "append", "rows": 16384, "heads": 8, "dim": 128, "page": 64, "src": "bf16",
         "dst": "bf16"},
        # one stream of the text decoder with the f32 cache: the smallest call
        {"name": "attn_1_f32", "op": "attn", "n_req": 1, "ctx": 217, "new": 8, "heads": 20, "kv": 20, "dim": 64,
         "page": 16, "dtype": "f32", "tree": True, "holes": False},
        # ten carried prompts of 224 tokens prefilled as chains
        {"name": "attn_10_prompt", "op": "attn", "n_req": 10, "ctx": 224, "new": 224, "heads": 20, "kv": 20,
         "dim": 64, "page": 16, "dtype": "f16", "tree": False, "holes": False},
        # one very long context, a wide tree: few requests, the long axis has to be split
        {"name": "attn_1_long", "op": "attn", "n_req": 1, "ctx": 131061, "new": 64, "heads": 32, "kv": 8, "dim": 128,
         "page": 16, "dtype": "f16", "tree": True, "holes": False},
        # a serving batch with grouped heads and ragged long contexts
        {"name": "attn_16_long", "op": "attn", "n_req": 16, "ctx": 32768, "new": 16, "heads": 32, "kv": 8,
         "dim": 128, "page": 64, "dtype": "bf16", "tree": True, "holes": False},
        # one token through a decoder projection: latency
        {"name": "q4_1_1280", "op": "q4", "m": 1, "n": 1280, "k": 1280, "group": 32, "min": False, "bias": True,
         "dtype": "f32", "scale": "f16"},
        # the logits head for a cohort of ten (an odd number of outputs)
        {"name": "q4_10_logits", "op": "q4", "m": 10, "n": 51866, "k": 1280, "group": 32, "min": False, "bias": False,
         "dtype": "f32", "scale": "f16"},
        # a wide projection for sixteen rows, groups of 128 with minimums
        {"name": "q4_16_wide", "op": "q4", "m": 16, "n": 28672, "k": 8192, "group": 128, "min": True, "bias": False,
         "dtype": "bf16", "scale": "f16"},
        # the first MLP linear over the rows of a whole window
        {"name": "q4_1500_mlp", "op": "q4", "m": 1500, "n": 5120, "k": 1280, "group": 32, "min": True, "bias": True,
         "dtype": "f16", "scale": "f16"},
    ]


def _log_int(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(("plan", "append", "attn", "attn", "attn", "q4", "q4", "q4"))
    if op == "plan":
        page = rng.choice((8, 16, 24, 32, 64, 128))
        new, ctx, n_req = _log_int(rng, 1, 64), _log_int(rng, 1, 32000), _log_int(rng, 1, 1024)
        return {"op": op, "n_req": n_req, "ctx": ctx, "new": new, "page": page,
                "width": (ctx + new) // page + 1 + rng.randint(0, 9), "tree": rng.random() < 0.7}
    heads, dim = rng.choice(((6, 64), (8, 64), (12, 64), (20, 64), (8, 128), (2, 128), (1, 128), (4, 64)))
    page = rng.choice((1, 8, 16, 16, 24, 32, 64, 100, 256))
    if op == "append":
        return {"op": op, "rows": _log_int(rng, 1, 16384), "heads": heads, "dim": dim, "page": page,
                "src": rng.choice(("f32", "f16", "bf16")), "dst": rng.choice(("f32", "f16", "bf16"))}
    if op == "attn":
        tree = rng.random() < 0.7
        new = _log_int(rng, 1, 64) if tree else _log_int(rng, 1, 448)
        group = rng.choice((1, 1, 2, 4, 8))
        dtype = rng.choice(("f32", "f16", "bf16"))
        ctx = 0 if rng.random() < 0.1 else _log_int(rng, 1, 65536)
        # no more cache bytes and no more products than the largest listed case, half of them in f32
        most = 16 * 32768 * 8 * 128 * 2 // (SIZE[dtype] * heads * dim * (ctx + new))
        most = min(most, 16 * 16 * 32768 * 32 * 128 // (new * (ctx + new) * heads * group * dim))
        return {"op": op, "n_req": _log_int(rng, 1, max(1, min(32, most))), "ctx": ctx, "new": new,
                "heads": heads * group, "kv": heads, "dim": dim, "page": page, "dtype": dtype, "tree": tree,
                "holes": tree and rng.random() < 0.3}
    group = rng.choice((32, 32, 64, 128))
    k = group * _log_int(rng, max(1, 128 // group), 8192 // group)
    n = _log_int(rng, 17, 28672)
    m = _log_int(rng, 1, min(2048, max(1, 16 * 28672 * 8192 // (n * k))))
    return {"op": op, "m": m, "n": n, "k": k, "group": group, "min": rng.random() < 0.5, "bias": rng.random() < 0.5,
            "dtype": rng.choice(("f32", "f16", "bf16")), "scale": rng.choice(("f16", "f16", "f32"))}


# ---------------------------------------------------------------------------
# sizes that follow from a case


def _lens(case):
    """Ragged lengths below the case's longest, the first request at the longest."""
    n, ctx, new = case["n_req"], case["ctx"], case["new"]
    lens = [ctx - (r * 7919) % (ctx // 2 + 1) for r in range(n)]
    news = [new - (r * 31) % (new // 2 + 1) for r in range(n)]
    return lens, news


def _pages(case):
    lens, news = _lens(case)
    return [-(-(a + b) // case["page"]) for a, b in zip(lens, news)]


def work(case):
    if case["op"] == "plan":
        n, (lens, news) = case["n_req"], _lens(case)
        rows = sum(news)
        words = -(-case["new"] // 64)
        return {"bytes": 2 * 4 * n * case["width"] + 7 * 4 * n + rows * (4 + 4 + 8 + (4 + 8 * words)), "flops": 0}
    if case["op"] == "append":
        return {"bytes": 2 * case["rows"] * (case["heads"] * case["dim"] * (SIZE[case["src"]] + SIZE[case["dst"]]) + 4),
                "flops": 0}
    if case["op"] == "attn":
        lens, news = _lens(case)
        keys = sum(a + b for a, b in zip(lens, news))
        pairs = sum((a + b) * b for a, b in zip(lens, news))
        e = SIZE[case["dtype"]]
        return {"bytes": 2 * keys * case["kv"] * case["dim"] * e + 2 * sum(news) * case["heads"] * case["dim"] * e,
                "flops": 4 * pairs * case["heads"] * case["dim"]}
    m, n, k, e = case["m"], case["n"], case["k"], SIZE[case["dtype"]]
    planes = (2 if case["min"] else 1) * SIZE[case["scale"]]
    return {"bytes": n * k // 2 + planes * n * (k // case["group"]) + e * (m * k + m * n) + 4 * n * case["bias"],
            "flops": 2 * m * n * k}


# ---------------------------------------------------------------------------
# what a program holds before the call


def _i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def _parents(g, news):
    """A parent for every drafted token: an earlier token of its request, or -1 for a child of the text so far."""
    n = _i32(news).long()
    start = torch.cumsum(n, 0) - n
    at = torch.arange(int(sum(news)), device="cuda") - torch.repeat_interleave(start, n, output_size=int(sum(news)))
    back = 1 + (torch.rand(at.numel(), generator=g, device="cuda") ** 2 * 6).long()
    return torch.clamp(at - back, min=-1).int()


def _prepare_plan(case, g):
    lens, news = _lens(case)
    n, ps, width = case["n_req"], case["page"], case["width"]
    held = _i32([-(-a // ps) for a in lens])
    total = int(sum(-(-a // ps) for a in lens)) + sum(_pages(case)) + 7
    pool = torch.randperm(total, generator=g, device="cuda").int()
    col = torch.arange(width, device="cuda")
    start = torch.cumsum(held, 0) - held
    owned = col[None, :] < held[:, None]
    at = torch.where(owned, start[:, None] + col[None, :], 0)
    table = torch.where(owned, pool[at.long()], -1).int()
    free = pool[int(held.sum()):].contiguous()
    return {"op": "plan", "lens": _i32(lens), "new": _i32(news), "table": table, "held": held, "free": free,
            "count": _i32([free.numel()]), "page": ps, "rows": sum(news), "words": -(-case["new"] // 64),
            "parents": _parents(g, news) if case["tree"] else None}


def _prepare_append(case, g):
    rows, h, d, ps = case["rows"], case["heads"], case["dim"], case["page"]
    src, dst = DTYPES[case["src"]], DTYPES[case["dst"]]
    qkv = torch.randn(rows, 3, h, d, generator=g, device="cuda").to(src)  # a fused projection's rows
    pages = -(-rows * 5 // (4 * ps)) + 1
    cache = torch.randn(2, pages, ps, h, d, generator=g, device="cuda").to(dst)
    slot = torch.randperm(pages * ps, generator=g, device="cuda")[:rows].long()
    return {"op": "append", "k": qkv[:, 1], "v": qkv[:, 2], "slot": slot, "k_cache": cache[0], "v_cache": cache[1]}


def _prepare_attn(case, g):
    lens, news = _lens(case)
    h, kv, d, ps, dt = case["heads"], case["kv"], case["dim"], case["page"], DTYPES[case["dtype"]]
    held = _pages(case)
    total = sum(held) + 3
    n, rows, width = case["n_req"], sum(news), max(held)
    perm = torch.randperm(total, generator=g, device="cuda").int()
    held_t = _i32(held)
    start = torch.cumsum(held_t, 0) - held_t
    col = torch.arange(width, device="cuda")
    owned = col[None, :] < held_t[:, None]
    table = torch.where(owned, perm[torch.where(owned, start[:, None] + col[None, :], 0).long()], -1).int()
    k_cache = torch.randn(total, ps, kv, d, generator=g, device="cuda", dtype=dt)
    v_cache = torch.randn(total, ps, kv, d, generator=g, device="cuda", dtype=dt)
    q = (torch.randn(rows, h + 2 * kv, d, generator=g, device="cuda") * 1.5).to(dt)[:, :h]  # of fused q/k/v rows
    row_start = torch.zeros(n + 1, dtype=torch.int32, device="cuda")
    row_start[1:] = torch.cumsum(_i32(news), 0)
    mask = None
    if case["tree"]:
        parents = _parents(g, news)
        at = torch.arange(rows, device="cuda")
        req = torch.searchsorted(row_start[1:].contiguous(), at.int(), right=True)
        mask = _tree(parents, row_start, req, n, max(news), -(-case["new"] // 64))[0]
        if case["holes"]:  # rows of padding, whose mask is empty
            mask[torch.rand(rows, generator=g, device="cuda") < 0.2] = 0
    return {"op": "attn", "q": q, "k_cache": k_cache, "v_cache": v_cache, "table": table, "lens": _i32(lens),
            "row_start": row_start, "mask": mask, "max_new": max(news), "max_len": max(a + b for a, b in zip(lens, news)),
            "scale": 1.0 / math.sqrt(d)}


def _prepare_q4(case, g):
    m, n, k, gs, dt = case["m"], case["n"], case["k"], case["group"], DTYPES[case["dtype"]]
    q = torch.randint(0, 256, (n, k // 2), generator=g, device="cuda", dtype=torch.uint8)
    step = 0.5 + torch.rand(n, k // gs, generator=g, device="cuda")
    scale = (step * (0.4 / math.sqrt(k))).to(DTYPES[case["scale"]])
    minimum = (scale.float() * -(6.0 + 3.0 * torch.rand(n, k // gs, generator=g, device="cuda"))).to(scale.dtype)
    return {"op": "q4", "x": torch.randn(m, k, generator=g, device="cuda").to(dt), "q": q, "scale": scale,
            "min": minimum if case["min"] else None, "group": gs,
            "bias": torch.randn(n, generator=g, device="cuda") if case["bias"] else None}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    return {"plan": _prepare_plan, "append": _prepare_append, "attn": _prepare_attn, "q4": _prepare_q4}[case["op"]](case, g)


# ---------------------------------------------------------------------------
# plain forms


def _bits(seen, words):
    """Truth values [..., 64 * words] as 64-bit words."""
    b = seen.reshape(*seen.shape[:-1], words, 64).long()
    return (b << torch.arange(64, device=seen.device)).sum(-1)


def _tree(parents, row_start, req, n, longest, words):
    """Each row's ancestors (itself among them) as words, and how many there are above it: (I - P)^-1 of the parents' matrix."""
    rows = parents.numel()
    at = torch.arange(rows, device=parents.device) - row_start[req].long()
    p = torch.zeros(n, longest, longest + 1, device=parents.device)
    p[req, at, torch.where(parents < 0, longest, parents.long())] = 1.0
    eye = torch.eye(longest, device=parents.device)
    seen = torch.linalg.solve_triangular(eye - p[:, :, :longest], eye.expand(n, -1, -1), upper=False)[req, at] > 0.5
    return _bits(torch.nn.functional.pad(seen, (0, 64 * words - longest)), words), seen.sum(-1) - 1


def _plan_plain(s):
    lens, new, table, held, ps = s["lens"].long(), s["new"].long(), s["table"], s["held"].long(), s["page"]
    n, width = table.shape
    row_start = torch.zeros(n + 1, dtype=torch.long, device=table.device)
    row_start[1:] = torch.cumsum(new, 0)
    want = torch.clamp((lens + new + ps - 1) // ps - held, min=0)
    room = want <= width - held
    need = torch.where(room, want, 0)
    total = torch.cumsum(need, 0)
    ok = room & ((need == 0) | (total <= s["count"]))
    taken = torch.where(total <= s["count"], total, 0).max()
    col = torch.arange(width, device=table.device)
    fresh = ok[:, None] & (col >= held[:, None]) & (col < (held + need)[:, None])
    at = s["count"] - 1 - ((total - need)[:, None] + col - held[:, None])
    table_out = torch.where(fresh, s["free"][torch.where(fresh, at, 0)], table)
    rows = torch.arange(s["rows"], device=table.device)
    req = torch.searchsorted(row_start[1:].contiguous(), rows, right=True)
    i = rows - row_start[req]
    token = lens[req] + i
    page = table_out[req, torch.clamp(token // ps, max=width - 1)].long()
    slot = torch.where(ok[req], page * ps + token % ps, -1)
    out = {"table": table_out, "held": (held + torch.where(ok, need, 0)).int(), "count": (s["count"] - taken).int(),
           "row_start": row_start.int(), "row_req": req.int(), "slot": slot,
           "status": (~ok).int()}
    if s["parents"] is None:
        out["pos"] = token.int()
    else:
        out["mask"], depth = _tree(s["parents"], row_start, req, n, 64 * s["words"], s["words"])
        out["pos"] = (lens[req] + depth).int()
    return out


def _append_plain(s):
    h, d = s["k"].shape[1:]
    s["k_cache"].view(-1, h, d)[s["slot"]] = s["k"].to(s["k_cache"].dtype)
    s["v_cache"].view(-1, h, d)[s["slot"]] = s["v"].to(s["v_cache"].dtype)
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _attn_plain(s):
    q, table, lens, row_start = s["q"], s["table"], s["lens"].long(), s["row_start"].long()
    rows, h, d = q.shape
    ps, kv = s["k_cache"].shape[1:3]
    n, longest, most = table.shape[0], s["max_len"], s["max_new"]
    dev = q.device
    req = torch.searchsorted(row_start[1:].contiguous(), torch.arange(rows, device=dev), right=True)
    i = torch.arange(rows, device=dev) - row_start[req]
    j = torch.arange(longest, device=dev)
    new = row_start[1:] - row_start[:-1]
    inside = j[None, :] < (lens + new)[:, None]
    page = torch.where(inside, table[:, j // ps].long(), 0)
    slot = page * ps + j % ps
    k = s["k_cache"].view(-1, kv, d)[slot].float()
    v = torch.where(inside[:, :, None, None], s["v_cache"].view(-1, kv, d)[slot].float(), 0.0)
    # rows of the same request side by side, the query heads of a K/V head after one another
    qp = torch.zeros(n, most, h, d, device=dev)
    qp[req, i] = q.float()
    qp = qp.view(n, most, kv, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, kv, most * (h // kv), d)
    scores = torch.matmul(qp, k.permute(0, 2, 3, 1)) * s["scale"]
    node = j[None, :] - lens[:, None]  # which drafted token a key is, negative for the text so far
    node_r = node[req]
    if s["mask"] is None:
        drafted = node_r <= i[:, None]
    else:
        word = s["mask"].gather(1, torch.clamp(node_r // 64, 0, s["mask"].shape[1] - 1))
        drafted = (word >> (node_r % 64)) & 1 > 0
    seen = torch.zeros(n, most, longest, dtype=torch.bool, device=dev)
    seen[req, i] = inside[req] & ((node_r < 0) | drafted)
    seen = seen[:, None, :, None, :].expand(n, kv, most, h // kv, longest).reshape(n, kv, most * (h // kv), longest)
    scores = torch.where(seen, scores, -math.inf)
    top = scores.max(-1, keepdim=True).values
    p = torch.where(seen, torch.exp(scores - top), 0.0)
    total = p.sum(-1, keepdim=True)
    o = torch.matmul(p, v.permute(0, 2, 1, 3)) / torch.where(total > 0, total, 1.0)
    o = o.view(n, kv, most, h // kv, d).permute(0, 2, 1, 3, 4).reshape(n, most, h, d)
    return o[req, i].to(q.dtype)


def _q4_plain(s):
    n, half = s["q"].shape
    q = s["q"].view(n, half // 16, 16)
    w = torch.cat((q & 15, q >> 4), -1).float().view(n, -1, s["group"])  # element j and j + 16 of each 32 share a byte
    if s["min"] is None:
        w = (w - 8.0) * s["scale"].float()[:, :, None]
    else:
        w = w * s["scale"].float()[:, :, None] + s["min"].float()[:, :, None]
    y = torch.matmul(s["x"].float(), w.view(n, 2 * half).t())
    if s["bias"] is not None:
        y = y + s["bias"]
    return y.to(s["x"].dtype)


# ---------------------------------------------------------------------------
# the framework's operators

_contexts = {}


def _context():
    """The program's context on its current stream."""
    from franken_whisper_amd import native

    stream = torch.cuda.current_stream()
    key = (stream.device_index, stream.cuda_stream)
    if key not in _contexts:
        _contexts[key] = native.Context(key[0], stream=key[1])
    return _contexts[key]


def _plan_own(s):
    from franken_whisper_amd import ops

    n, dev = s["table"].shape[0], s["table"].device
    out = {"table": torch.empty_like(s["table"]), "held": torch.empty_like(s["held"]),
           "count": torch.empty_like(s["count"]), "row_start": torch.empty(n + 1, dtype=torch.int32, device=dev),
           "row_req": torch.empty(s["rows"], dtype=torch.int32, device=dev),
           "slot": torch.empty(s["rows"], dtype=torch.int64, device=dev),
           "status": torch.empty(n, dtype=torch.int32, device=dev),
           "pos": torch.empty(s["rows"], dtype=torch.int32, device=dev)}
    if s["parents"] is not None:
        out["mask"] = torch.empty(s["rows"], s["words"], dtype=torch.int64, device=dev)
    ops.paged_plan(_context(), s["lens"], s["new"], s["table"], s["held"], s["free"], s["count"], s["page"],
                   parents=s["parents"], table_out=out["table"], held_out=out["held"], count_out=out["count"],
                   row_start=out["row_start"], row_req=out["row_req"], slot=out["slot"], pos=out["pos"],
                   status=out["status"], mask=out.get("mask"))
    return out


def _append_own(s):
    from franken_whisper_amd import ops

    ops.paged_append(_context(), s["k"], s["v"], s["slot"], s["k_cache"], s["v_cache"])
    return {"k": s["k_cache"], "v": s["v_cache"]}


def _attn_own(s):
    from franken_whisper_amd import ops

    rows, h, d = s["q"].shape
    out = torch.empty(rows, h, d, dtype=s["q"].dtype, device=s["q"].device)
    if "workspace" not in s:  # a program keeps one for its largest step
        need = ops.tree_attn_workspace(s["table"].shape[0], h, s["k_cache"].shape[2], d, s["max_new"], s["max_len"])
        s["workspace"] = torch.empty(need, dtype=torch.uint8, device=out.device)
    ops.tree_attn(_context(), s["q"], s["k_cache"], s["v_cache"], s["table"], s["lens"], s["row_start"], out,
                  scale=s["scale"], max_new=s["max_new"], max_len=s["max_len"], mask=s["mask"],
                  workspace=s["workspace"])
    return out


def _q4_own(s):
    from franken_whisper_amd import ops

    out = torch.empty(s["x"].shape[0], s["q"].shape[0], dtype=s["x"].dtype, device=s["x"].device)
    ops.q4_linear(_context(), s["x"], s["q"], s["scale"], out, group=s["group"], minimum=s["min"], bias=s["bias"])
    return out


def run(state):
    if own:
        return {"plan": _plan_own, "append": _append_own, "attn": _attn_own, "q4": _q4_own}[state["op"]](state)
    return {"plan": _plan_plain, "append": _append_plain, "attn": _attn_plain, "q4": _q4_plain}[state["op"]](state)


# ---------------------------------------------------------------------------
# the definitions in 64 bits


def _exact_attn(s):
    rows, h, d = s["q"].shape
    ps, kv = s["k_cache"].shape[1:3]
    out = torch.zeros(rows, h, d, dtype=torch.float64, device=s["q"].device)
    starts, lens, table = s["row_start"].tolist(), s["lens"].tolist(), s["table"].cpu()
    for r, ctx in enumerate(lens):
        a, b = starts[r], starts[r + 1]
        count = ctx + b - a
        pages = table[r, : -(-count // ps)].long().to(out.device)
        allowed = torch.ones(b - a, count, dtype=torch.bool, device=out.device)
        for i in range(b - a):
            if s["mask"] is None:
                allowed[i, ctx + i + 1:] = False
            else:
                words = [w % (1 << 64) for w in s["mask"][a + i].tolist()]
                seen = [bool(words[t // 64] >> (t % 64) & 1) for t in range(b - a)]
                allowed[i, ctx:] = torch.tensor(seen, device=out.device)
        some = allowed.any(1)
        for g in range(kv):
            k = s["k_cache"][pages, :, g].reshape(-1, d)[:count].double()
            v = s["v_cache"][pages, :, g].reshape(-1, d)[:count].double()
            for x in range(g * (h // kv), (g + 1) * (h // kv)):
                z = s["q"][a:b, x].double() @ k.t().contiguous() * s["scale"]
                z = z.masked_fill(~allowed, -math.inf)
                p = torch.softmax(z, 1)
                out[a:b, x] = torch.where(some[:, None], torch.where(some[:, None], p, 0.0) @ v, 0.0)
    return out


def _exact_q4(s):
    x, n, k, gs = s["x"].double(), s["q"].shape[0], s["x"].shape[1], s["group"]
    y = torch.zeros(x.shape[0], n, dtype=torch.float64, device=x.device)
    for b in range(k // 32):  # 32 inputs at a time
        byte = s["q"][:, 16 * b: 16 * b + 16].int()
        code = torch.empty(n, 32, dtype=torch.float64, device=x.device)
        code[:, :16], code[:, 16:] = (byte % 16).double(), (byte // 16).double()
        step = s["scale"][:, 32 * b // gs].double()[:, None]
        low = -8.0 * step if s["min"] is None else s["min"][:, 32 * b // gs].double()[:, None]
        y += x[:, 32 * b: 32 * b + 32] @ (code * step + low).t().contiguous()
    return y if s["bias"] is None else y + s["bias"].double()


def exact(case, seed):
    if case["op"] == "plan":
        return None  # whole numbers
    s = prepare(case, seed)
    if case["op"] == "append":
        page = s["k_cache"].shape[1]
        k, v = s["k_cache"].double(), s["v_cache"].double()
        k[s["slot"] // page, s["slot"] % page] = s["k"].double()
        v[s["slot"] // page, s["slot"] % page] = s["v"].double()
        return {"k": k, "v": v}
    if case["op"] == "attn":
        if sum(_lens(case)[1]) * case["heads"] * case["ctx"] > 4e8:
            return None
        return _exact_attn(s)
    return _exact_q4(s)
