"""Plain 64-bit forms of the serving operators, for their tests."""
from __future__ import annotations

import numpy as np

EPS = {"f32": 2.0 ** -24, "f16": 2.0 ** -11, "bf16": 2.0 ** -8}  # half a step, relative
TINY = {"f32": 0.0, "f16": 2.0 ** -25, "bf16": 0.0}              # half a step below the normal range


def plan(lens, n_new, table, held, free, count, page, n_rows, parents=None, words=0):
    """fwhip_paged_plan, one request after another."""
    n_req, width = table.shape
    out = {"table": table.copy(), "held": held.copy(), "row_start": np.zeros(n_req + 1, np.int32),
           "status": np.zeros(n_req, np.int32), "row_req": {}, "pos": {}, "slot": {}, "mask": {}}
    count = min(max(int(count), 0), len(free))
    cum, row, left = 0, 0, count
    for r in range(n_req):
        ln, new, h, st = int(lens[r]), int(n_new[r]), int(held[r]), 0
        if ln < 0 or new < 0 or h < 0 or h > width or ln + max(new, 0) > 2 ** 31 - 1 - page:
            st, need = 2, 0
        else:
            need = max(0, -(-(ln + new) // page) - h)
            if need > width - h:
                st, need = 1, 0
        rows = max(new, 0)
        bad_len = st == 2
        cum += need
        if need and cum > count:
            st |= 1
        elif cum <= count:
            left = count - cum
        ok = not st & 1 and not bad_len
        if ok:
            for t in range(need):
                out["table"][r, h + t] = free[count - 1 - (cum - need) - t]
            out["held"][r] = h + need
        first, last = min(row, n_rows), min(row + rows, n_rows)
        if last - first < rows:
            st |= 2
        fits = parents is None or rows <= 64 * words
        if parents is not None and not fits:
            st |= 4
        seen = []
        for i in range(last - first):
            x = first + i
            out["row_req"][x] = r
            pg = (ln + i) // page
            pid = int(out["table"][r, pg]) if ok else -1
            out["slot"][x] = pid * page + (ln + i) % page if pid >= 0 else -1
            if parents is None or not fits:
                out["pos"][x] = ln + i
                out["mask"][x] = 0
            else:
                p = int(parents[x])
                if p < -1 or p >= i:
                    st |= 4
                    p = -1
                seen.append((seen[p] if p >= 0 else 0) | 1 << i)
                out["mask"][x] = seen[-1]
                out["pos"][x] = ln + bin(seen[-1]).count("1") - 1
        row += rows
        out["row_start"][r + 1] = last
        out["status"][r] = st
    out["count"] = left
    return out


def attn(q, k_cache, v_cache, table, lens, row_start, mask, scale, kind):
    """fwhip_tree_attn and a bound of its error, per output.

    Bound, with u = 2^-24: a score is D products and D - 1 sums in f32, its
    scaling and (in base 2) one more rounding: |dz| <= (D + 4) u scale sum|q k|;
    e^z of it is off by |dz| relative plus 8 u of its own (argument and
    function).  Each weight so carries at most 2 max|dz| + 8 u against the
    normalized one; sums over N keys add N u; a weight that is multiplied as a
    pair of 16-bit numbers is off by 2^-16 of itself (two 8-bit significands;
    an f16 pair less, but its lower half may lie below the normal range: 2^-24
    of the largest weight).  All of that scales sum_j p_j |v_j|; the output is
    rounded once."""
    rows, h, d = q.shape
    pages, page, kv, _ = k_cache.shape
    out, tol = np.zeros((rows, h, d)), np.zeros((rows, h, d))
    u = 2.0 ** -24
    for r in range(len(lens)):
        a, b, ln = int(row_start[r]), int(row_start[r + 1]), int(lens[r])
        n = ln + b - a
        j = np.arange(n)
        pid = table[r, j // page] if n else np.zeros(0, int)
        for i in range(a, b):
            if mask is None:
                sees = j <= ln + i - a
            else:
                bits = [int(mask[i, t >> 6]) >> (t & 63) & 1 for t in range(b - a)]
                sees = np.concatenate([np.ones(ln, bool), np.array(bits, bool)])
            js = j[sees]
            if js.size == 0:
                continue
            for g in range(kv):
                k = k_cache[pid[js], js % page, g].astype(np.float64)
                v = v_cache[pid[js], js % page, g].astype(np.float64)
                for x in range(g * (h // kv), (g + 1) * (h // kv)):
                    qx = q[i, x].astype(np.float64)
                    with np.errstate(invalid="ignore", over="ignore"):
                        z = scale * (k @ qx)
                        dz = (d + 4) * u * abs(scale) * (np.abs(k) @ np.abs(qx)).max()
                        p = np.exp(z - z.max())
                        p = p / p.sum()
                        o, s = p @ v, p @ np.abs(v)
                    out[i, x] = o
                    c = 2 * dz + (js.size + 8) * u + (2.0 ** -16 if kind != "f32" else 0)
                    tol[i, x] = EPS[kind] * (np.abs(o) + c * s) + c * s + TINY[kind]
    return out, tol


def q4_weights(q, scale, minimum, group):
    n, half = q.shape
    b = q.reshape(n, half // 16, 16).astype(np.int64)
    code = np.concatenate([b & 15, b >> 4], -1).reshape(n, 2 * half // group, group).astype(np.float64)
    s = scale.astype(np.float64)[:, :, None]
    if minimum is None:
        code = code - 8
        m = np.zeros_like(s)
    else:
        m = minimum.astype(np.float64)[:, :, None]
    return (code * s + m).reshape(n, -1), (np.abs(code * s) + np.abs(m)).reshape(n, -1)


def q4(x, q, scale, minimum, bias, group, kind):
    """fwhip_q4_linear and a bound of its error: a group's whole-number codes
    times x in f32 sums (the codes as they are or less 8, or the codes and the
    sum of x times 8 apart: at most 8 + 15 per product where |code - 8| <= 8),
    one scaling, a sum over groups: (k + 8) u sum |x| |w|_max with
    |w|_max <= 23 |scale| + |minimum|, far above what happens but in proportion."""
    w, _ = q4_weights(q, scale, minimum, group)
    x64 = x.astype(np.float64)
    y = x64 @ w.T
    big = 23 * np.abs(scale.astype(np.float64)) + (0 if minimum is None else np.abs(minimum.astype(np.float64)))
    s = np.abs(x64).reshape(x.shape[0], -1, group).sum(-1) @ big.T
    if bias is not None:
        y = y + bias.astype(np.float64)
        s = s + np.abs(bias.astype(np.float64))
    # a sum of k terms in some order: sqrt would be usual, this is the worst case over 8 partial sums
    c = (x.shape[1] / 8 + 64) * 2.0 ** -24
    return y, EPS[kind] * (np.abs(y) + c * s) + c * s + TINY[kind]
