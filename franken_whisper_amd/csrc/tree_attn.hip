// tree_attn.hip — attention of drafted trees (or causal chains of new tokens)
// over a paged K/V cache (fwhip_tree_attn).
//
// out_i = sum_j softmax_j(s q_i.k_j) v_j over the keys row i sees: the request's
// cached tokens, and those of its new tokens that the mask row names.  One pass
// over the keys with a running maximum m and sum l:
//   m' = max(m, max_j z_j),  l' = l e^(m-m') + sum_j e^(z_j-m'),  o' likewise.
#include <algorithm>
#include <type_traits>

#include "fw_device.h"
#include "fw_paged.h"
#include "fw_serve.h"

#define TREE_UNITS 1024 // units of a call, at most
#define TREE_CHUNK 128  // keys of a unit, at least
#define TREE_WHOLE 512  // up to as many keys a request is not cut

struct TreeP {
    int n_req, n_rows, heads, kv_heads, n_pages, width, max_new, max_len, words;
    float scale;
    FwDiv page;
    int64_t table_stride, q_row, q_head, out_row, out_head, head_stride;
    uint32_t page_bytes, token_bytes;
    const void *q, *kc, *vc;
    const int32_t *table, *len, *row_start;
    const uint64_t *mask;
    void *out;
    // how the call is cut (tree_cut): row tiles and their rows; units of keys, or 0
    // where a block takes all keys of its request; the units' parts [unit, tile, K/V
    // head, row, D + 4]
    int tiles, tile_rows, units;
    float *parts;
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef short s4v __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// Products of 16 x 16 tiles.  A lane l holds row (A) or column (B) l % 16 of an
// operand and its quarter c = l / 16 of the inner dimension; of the result,
// column l % 16 and rows 4 c + 0..3.  Both inner dimensions may be permuted as
// long as the operands agree, which is what lets scores (keys x rows) become
// weights (keys x rows) of the second product without leaving their lanes.
template <typename T>
struct Mma;
template <>
struct Mma<fw_f16> {
    static constexpr int KT = 2; // key tiles a step: one product of inner dimension 32 takes 32 keys
    static __device__ __forceinline__ f4 dot(u4 a, u4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b), c, 0, 0, 0);
    }
    // p = hi + lo up to 2^-20 of p: two f16 of 11 bits each, cut
    static __device__ __forceinline__ void split(const f4 (&w)[2], u4 &hi, u4 &lo) {
        const float p[8] = {w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]};
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const auto h = __builtin_amdgcn_cvt_pkrtz(p[2 * i], p[2 * i + 1]);
            const auto l = __builtin_amdgcn_cvt_pkrtz(fmaf((float)h[0], -1.0f, p[2 * i]), fmaf((float)h[1], -1.0f, p[2 * i + 1]));
            hi[i] = __builtin_bit_cast(uint32_t, h);
            lo[i] = __builtin_bit_cast(uint32_t, l);
        }
    }
};
template <>
struct Mma<fw_bf16> {
    static constexpr int KT = 2;
    static __device__ __forceinline__ f4 dot(u4 a, u4 b, f4 c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b), c, 0, 0, 0);
    }
    // p = hi + lo up to 2^-16 of p: the upper half of the f32, and the rest rounded to 8 bits
    static __device__ __forceinline__ void split(const f4 (&w)[2], u4 &hi, u4 &lo) {
        const float p[8] = {w[0][0], w[0][1], w[0][2], w[0][3], w[1][0], w[1][1], w[1][2], w[1][3]};
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t x = __float_as_uint(p[2 * i]), y = __float_as_uint(p[2 * i + 1]);
            hi[i] = __builtin_amdgcn_perm(y, x, 0x07060302);
            const b2 l = {(__bf16)(p[2 * i] - __uint_as_float(x & 0xffff0000u)),
                          (__bf16)(p[2 * i + 1] - __uint_as_float(y & 0xffff0000u))};
            lo[i] = __builtin_bit_cast(uint32_t, l);
        }
    }
};
template <>
struct Mma<float> {
    static constexpr int KT = 1;
    static __device__ __forceinline__ f4 dot(u4 a, u4 b, f4 c) {
#pragma unroll
        for (int t = 0; t < 4; t++)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[t]), __uint_as_float(b[t]), c, 0, 0, 0);
        return c;
    }
};

// Over the four lanes that share l % 16.
__device__ __forceinline__ float quarters_max(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float quarters_sum(float v) {
    auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    a = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ void wave_fence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// Weights are 2^7 2^(z - m) with m the largest score so far, up to a slack of 8:
// while a new largest stays within it, m stays, what is there need not be
// scaled, and no weight passes 2^15 (an f16 holds 65504).  The factor cancels in
// o / l; it keeps f16 weights of far smaller keys (down to 2^-21 of 2^m) normal.
#define TREE_BIAS 7.0f
#define TREE_SLACK 8.0f
__device__ __forceinline__ float tree_base(float m) { return m == -INFINITY ? 0.0f : m - TREE_BIAS; }

// What a block finds about its request; bad: out of the call's bounds.
struct TreeReq {
    int row0, n, len;
    bool bad;
};
__device__ __forceinline__ TreeReq tree_req(const TreeP &p, int r) {
    TreeReq q;
    q.row0 = min(max(p.row_start[r], 0), p.n_rows);
    q.n = max(min(p.row_start[r + 1], p.n_rows) - q.row0, 0);
    q.len = p.len[r];
    q.bad = q.len < 0 || q.n > p.max_new || (int64_t)q.len + q.n > p.max_len;
    return q;
}
// The keys of all requests as units of `chunk` keys, the last of each request
// shorter: as few keys a unit as keep the units within p.units (a request adds at
// most one that is not full).  Each wave finds this from the lengths by itself.
// unit < 0: where request r begins; else the request that holds unit (n_req: none).
struct TreeUnits {
    int chunk, r, first, count; // a request, its first unit and how many it has
};
__device__ __forceinline__ TreeUnits tree_units(const TreeP &p, int unit, int r) {
    const int lane = threadIdx.x & 63;
    auto keys = [&](int i) {
        if (i >= p.n_req) return 0;
        const TreeReq q = tree_req(p, i);
        return q.bad || q.n == 0 ? 0 : q.len + q.n;
    };
    int mine = keys(lane); // of the first 64 requests
    double sum = mine;     // exact: whole numbers below 2^53
    for (int i = lane + 64; i < p.n_req; i += 64) sum += keys(i);
    const int64_t total = (int64_t)fw_dpp_wave_sum_f64(sum);
    // fewer than total / chunk + n_req units come of it (the host sees to units > n_req)
    const int64_t whole = p.units - p.n_req + 1, full = (total + whole - 1) / whole;
    TreeUnits u;
    u.chunk = __builtin_amdgcn_readfirstlane((int)max((full + 127) / 128 * 128, (int64_t)TREE_CHUNK));
    u.r = p.n_req;
    u.first = u.count = 0;
    int before = 0;
    for (int i0 = 0; i0 < p.n_req; i0 += 64) {
        if (i0) mine = keys(i0 + lane);
        const int n = (mine + u.chunk - 1) / u.chunk;
        int sum = n; // of this request and those before it
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const int v = __shfl_up(sum, o, 64);
            if (lane >= o) sum += v;
        }
        const uint64_t who = __ballot(unit < 0 ? i0 + lane == r : unit < before + sum);
        if (who) { // the same in every lane, as are all results: they steer the loops
            const int at = __ffsll((unsigned long long)who) - 1;
            u.r = i0 + at;
            u.count = __builtin_amdgcn_readlane(n, at);
            u.first = before + __builtin_amdgcn_readlane(sum, at) - u.count;
            break;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return u;
}
// Whether new token i of the request sees key j < last.
__device__ __forceinline__ bool tree_sees(const TreeP &p, const TreeReq &q, int i, int j, int last) {
    const int t = j - q.len;
    bool yes = j < last;
    if (yes && t >= 0) yes = p.words ? p.mask[(int64_t)(q.row0 + i) * p.words + (t >> 6)] >> (t & 63) & 1 : t <= i;
    return yes;
}
// The same for 32 keys at once, bit b for key j + b.  One window of the mask row
// (or a comparison) a row and step, and a bit test a score.
__device__ __forceinline__ uint32_t tree_window(const TreeP &p, const TreeReq &q, int i, int j, int last) {
    const int t = j - q.len, left = last - j; // t < 0: cached tokens, which every row sees
    uint32_t w = ~0u;
    if (p.words) {
        const uint64_t *row = p.mask + (int64_t)(q.row0 + i) * p.words;
        const int at = max(t, 0) >> 6, sh = max(t, 0) & 63;
        uint64_t v = at < p.words ? row[at] >> sh : 0;
        if (sh > 32 && at + 1 < p.words) v |= row[at + 1] << (64 - sh);
        w = (uint32_t)v;
        if (t < 0) w = t <= -32 ? ~0u : w << -t | ((1u << -t) - 1);
    } else {
        const int v = i - t; // bits 0..v
        w = v < 0 ? 0u : v >= 31 ? ~0u : (2u << v) - 1;
    }
    return left <= 0 ? 0u : left >= 32 ? w : w & ((1u << left) - 1);
}
// Whether new token i of a request with n of them sees any key.
__device__ __forceinline__ bool tree_sees_any(const TreeP &p, const TreeReq &q, int i) {
    if (q.len > 0 || !p.words) return true;
    uint64_t any = 0;
    for (int w = 0; w * 64 < q.n; w++) {
        const uint64_t m = p.mask[(int64_t)(q.row0 + i) * p.words + w];
        any |= q.n - w * 64 >= 64 ? m : m & ((1ull << (q.n - w * 64)) - 1);
    }
    return any != 0;
}

template <typename T>
struct Vec4 {
    typedef uint2 type;
};
template <>
struct Vec4<float> {
    typedef float4 type;
};
template <typename T>
__device__ __forceinline__ typename Vec4<T>::type pack4(f4 v) {
    if constexpr (sizeof(T) == 4) return make_float4(v[0], v[1], v[2], v[3]);
    else
        return make_uint2(fw_cvt<T>(v[0]).b | (uint32_t)fw_cvt<T>(v[1]).b << 16,
                          fw_cvt<T>(v[2]).b | (uint32_t)fw_cvt<T>(v[3]).b << 16);
}

// Bytes from the start of a K/V head's cache to token t of page id.
__device__ __forceinline__ uint64_t tree_at(const TreeP &p, uint32_t t, uint32_t id) {
    return (uint64_t)id * p.page_bytes + (uint64_t)t * p.token_bytes;
}

// Scores are z = zs * (q . k) with zs > 0 in base 2, so that the largest product
// has the largest score: a negative scale turns q's signs, a scale of zero
// makes q zero (NaN where it is not finite).
__device__ __forceinline__ float tree_zs(const TreeP &p) {
    return p.scale == 0.0f ? 1.0f : fabsf(p.scale) * 1.44269504088896340736f;
}
template <typename T>
__device__ __forceinline__ u4 tree_query(u4 v, float scale) {
    if (scale > 0.0f) return v;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        if (scale < 0.0f) v[i] ^= sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
        else if constexpr (sizeof(T) == 4) v[i] = (v[i] & 0x7f800000u) == 0x7f800000u ? 0x7fc00000u : 0;
        else {
            constexpr uint32_t E = std::is_same<T, fw_f16>::value ? 0x7c00u : 0x7f80u;
            v[i] = ((v[i] & E) == E ? 0x7fffu : 0) | ((v[i] >> 16 & E) == E ? 0x7fff0000u : 0);
        }
    }
    return v;
}

// ---------------------------------------------------------------------------
// What both kernels below do with a wave's rows: RT tiles of 16 query rows (new
// token x query head of the K/V head's group), and steps of KEYS keys.
template <typename T, int D, int RT>
struct Rows {
    static constexpr int KT = Mma<T>::KT, KEYS = 16 * KT, NS = D * (int)sizeof(T) / 64, DT = D / 16;
    int node[RT], head[RT]; // of row lr of each tile
    u4 q[RT][NS];
    f4 o[RT][DT];
    float m[RT], l[RT];

    __device__ __forceinline__ void load(const TreeP &p, const TreeReq &rq, int t0, int total, int kvh, int group) {
        const int lane = threadIdx.x & 63, lr = lane & 15, c = lane >> 4;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const int t = min(t0 + x * 16 + lr, total - 1); // the last row again behind the end
            node[x] = t / group;
            head[x] = kvh * group + t % group;
            const T *at = (const T *)p.q + (int64_t)(rq.row0 + node[x]) * p.q_row + head[x] * p.q_head;
#pragma unroll
            for (int s = 0; s < NS; s++) q[x][s] = tree_query<T>(*(const u4 *)((const char *)at + s * 64 + c * 16), p.scale);
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int x = 0; x < RT; x++) {
            m[x] = -INFINITY;
            l[x] = 0.0f;
#pragma unroll
            for (int d = 0; d < DT; d++) o[x][d] = f4{};
        }
    }
    // Products of the step at key j to -inf where a row does not see the key.
    __device__ __forceinline__ void mask(const TreeP &p, const TreeReq &rq, int x, int j, int last, f4 (&z)[KT]) const {
        const uint32_t sees = tree_window(p, rq, node[x], j, last) >> (threadIdx.x >> 2 & 12); // 4 c
#pragma unroll
        for (int k = 0; k < KT; k++)
#pragma unroll
            for (int i = 0; i < 4; i++) z[k][i] = sees >> (k * 16 + i) & 1 ? z[k][i] : -INFINITY;
    }
    // Products q . k to weights (in place); what is there already is scaled where the maximum moves.
    __device__ __forceinline__ void weigh(f4 (&z)[RT][KT], float zs) {
        float mx[RT];
        bool moves = false;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            mx[x] = z[x][0][0];
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) mx[x] = fmaxf(mx[x], z[x][k][i]);
            mx[x] = quarters_max(mx[x]) * zs;
            moves |= mx[x] > m[x] + TREE_SLACK;
        }
        if (__builtin_expect(__any(moves), 0)) {
#pragma unroll
            for (int x = 0; x < RT; x++) {
                const float mn = mx[x] > m[x] + TREE_SLACK ? mx[x] : m[x];
                const float f = __builtin_amdgcn_exp2f(m[x] - TREE_BIAS - tree_base(mn));
                m[x] = mn;
                l[x] *= f;
#pragma unroll
                for (int d = 0; d < DT; d++) o[x][d] *= f;
            }
        }
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const float base = tree_base(m[x]);
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    // rounded before the difference, as the maximum is: its own weight is exact at any size
                    z[x][k][i] = __builtin_amdgcn_exp2f(z[x][k][i] * zs - base);
                    l[x] += z[x][k][i];
                }
        }
    }
    // o += weights times the V tile in LDS (rows of VROW bytes).
    template <int VROW>
    __device__ __forceinline__ void add(const char *vt, const f4 (&w)[RT][KT]) {
        const int lane = threadIdx.x & 63, lr = lane & 15, c = lane >> 4;
        u4 hi[RT], lo[RT];
        if constexpr (sizeof(T) == 2)
#pragma unroll
            for (int x = 0; x < RT; x++) Mma<T>::split(w[x], hi[x], lo[x]);
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if constexpr (sizeof(T) == 2) {
                u4 v;
#pragma unroll
                for (int k = 0; k < 2; k++) {
                    const char *at = vt + (k * 16 + 4 * c + (lr >> 2)) * VROW + d * 32 + (lr & 3) * 8;
                    const uint2 u = __builtin_bit_cast(
                        uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4v *)at));
                    v[2 * k] = u.x;
                    v[2 * k + 1] = u.y;
                }
#pragma unroll
                for (int x = 0; x < RT; x++) o[x][d] = Mma<T>::dot(v, lo[x], Mma<T>::dot(v, hi[x], o[x][d]));
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float v = *(const float *)(vt + (4 * c + i) * VROW + d * 64 + lr * 4);
#pragma unroll
                    for (int x = 0; x < RT; x++)
                        o[x][d] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, w[x][0][i], o[x][d], 0, 0, 0);
                }
            }
        }
    }
    __device__ __forceinline__ bool odd() const {
        bool any = false;
#pragma unroll
        for (int x = 0; x < RT; x++)
#pragma unroll
            for (int d = 0; d < DT; d++)
#pragma unroll
                for (int i = 0; i < 4; i++) any |= !(fabsf(o[x][d][i]) < INFINITY);
        return any;
    }
    // One result of `parts` waves that took different keys of the same rows: the
    // first one gets it.  sm / sl: [parts][rows], ot: [rows][D] in LDS; every
    // thread of the block comes here.
    __device__ __forceinline__ void join(int part, int parts, int row0, int rows, float *sm, float *sl, float *ot) {
        const int lane = threadIdx.x & 63, lr = lane & 15, c = lane >> 4;
        float f[RT];
#pragma unroll
        for (int x = 0; x < RT; x++)
            if (c == 0) {
                sm[part * rows + row0 + x * 16 + lr] = m[x];
                sl[part * rows + row0 + x * 16 + lr] = l[x];
            }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const float *am = sm + row0 + x * 16 + lr, *al = sl + row0 + x * 16 + lr;
            float mx = -INFINITY;
            for (int w = 0; w < parts; w++) mx = fmaxf(mx, am[w * rows]);
            f[x] = __builtin_amdgcn_exp2f(m[x] - TREE_BIAS - tree_base(mx));
            l[x] = 0.0f;
            for (int w = 0; w < parts; w++)
                l[x] = fmaf(__builtin_amdgcn_exp2f(am[w * rows] - TREE_BIAS - tree_base(mx)), al[w * rows], l[x]);
            m[x] = mx;
        }
        for (int w = parts - 1; w >= 0; w--) {
            if (part == w) {
#pragma unroll
                for (int x = 0; x < RT; x++)
#pragma unroll
                    for (int d = 0; d < DT; d++) {
                        f4 *at = (f4 *)(ot + (row0 + x * 16 + lr) * D + ((16 * d + 4 * c) ^ (4 * (lr & 7))));
                        const f4 mine = f[x] == 0.0f ? f4{} : o[x][d] * f[x];
                        o[x][d] = w == parts - 1 ? mine : mine + *at;
                        if (w) *at = o[x][d];
                    }
            }
            __syncthreads();
        }
    }
    // Rows t0 + 0..16 RT - 1: outputs, or this unit's part.
    template <typename B>
    __device__ __forceinline__ void store(const TreeP &p, const B &b, int t0) {
        const TreeReq &rq = b.rq;
        const int lane = threadIdx.x & 63, lr = lane & 15, c = lane >> 4;
#pragma unroll
        for (int x = 0; x < RT; x++) {
            const int t = t0 + x * 16 + lr;
            if (t >= b.total) continue;
            if (b.whole) {
                T *out = (T *)p.out + (int64_t)(rq.row0 + node[x]) * p.out_row + head[x] * p.out_head + 4 * c;
                const bool any = tree_sees_any(p, rq, node[x]);
                const float inv = 1.0f / l[x];
#pragma unroll
                for (int d = 0; d < DT; d++) {
                    f4 v = l[x] == 0.0f ? f4{} + __builtin_nanf("") : o[x][d] * inv; // 0 / 0: every key scored -inf
                    if (!any) v = f4{};
                    *(typename Vec4<T>::type *)(out + 16 * d) = pack4<T>(v);
                }
            } else {
                float *at = b.part(p, D, t - b.t0);
#pragma unroll
                for (int d = 0; d < DT; d++) *(f4 *)(at + 16 * d + 4 * c) = o[x][d];
                if (c == 0) {
                    at[D] = m[x];
                    at[D + 1] = l[x];
                }
            }
        }
    }
};

// Where a block stands: its chunk of keys of one K/V head of one request.
struct TreeBlock {
    TreeReq rq;
    int r, kvh, tile, group, total, t0, first, last;
    int clear; // every row of the block sees every key before this one
    bool whole;
    // false: nothing to do (or done: rows of a bad request)
    template <typename T, int D>
    __device__ __forceinline__ bool find(const TreeP &p) {
        kvh = blockIdx.x % p.kv_heads; // heads of a token lie next to each other, their blocks too
        tile = blockIdx.x / p.kv_heads;
        group = p.heads / p.kv_heads;
        whole = p.units == 0;
        int chunk = 0;
        r = blockIdx.y;
        first = 0;
        if (!whole) {
            const TreeUnits u = tree_units(p, blockIdx.y, 0);
            if (u.r == p.n_req) return false;
            r = __builtin_amdgcn_readfirstlane(u.r);
            chunk = u.chunk;
            first = __builtin_amdgcn_readfirstlane((blockIdx.y - u.first) * chunk);
        }
        rq = tree_req(p, r);
        if (rq.bad) { // may have more rows than there are tiles (with units the join writes them)
            if (tile == 0)
                for (int64_t e = threadIdx.x; e < (int64_t)rq.n * group * D; e += 256) {
                    const int64_t i = e / D / group, h = kvh * group + e / D % group;
                    ((T *)p.out)[(rq.row0 + i) * p.out_row + h * p.out_head + e % D] = fw_cvt<T>(__builtin_nanf(""));
                }
            return false;
        }
        total = rq.n * group;
        t0 = tile * p.tile_rows;
        if (t0 >= total) return false;
        // a chain's rows see no further than the tile's last token
        const int end = p.words ? rq.len + rq.n : rq.len + (min(t0 + p.tile_rows, total) - 1) / group + 1;
        last = whole ? end : min(end, first + chunk);
        clear = min(last, p.words ? rq.len : rq.len + t0 / group + 1);
        return whole || first < end; // the join reads no part behind the end
    }
    // Where this block's part of row t0 + i goes.
    __device__ __forceinline__ float *part(const TreeP &p, int d, int i) const {
        return p.parts + ((((int64_t)blockIdx.y * p.tiles + tile) * p.kv_heads + kvh) * p.tile_rows + i) * (d + 4);
    }
};

// A block's rows once more, one row a wave at a time and key by key, after
// outputs that are not finite: those may come from values that a row does not see
// (0 times infinity) or from the halves of a weight (infinity less infinity),
// which do not meet here.  lds: 4 x (D + 192) floats.
template <typename T, int D>
__device__ __forceinline__ void tree_slow(const TreeP &p, const TreeBlock &b, char *lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float *sq = (float *)lds + wave * (D + 192), *sp = sq + D;
    int64_t *sat = (int64_t *)(sp + 64);
    const int32_t *trow = p.table + (int64_t)b.r * p.table_stride;
    const char *kbase = (const char *)((const T *)p.kc + b.kvh * p.head_stride);
    const char *vbase = (const char *)((const T *)p.vc + b.kvh * p.head_stride);
    for (int t = b.t0 + wave; t < min(b.t0 + p.tile_rows, b.total); t += 4) {
        const int i = t / b.group, h = b.kvh * b.group + t % b.group;
        const T *q = (const T *)p.q + (int64_t)(b.rq.row0 + i) * p.q_row + h * p.q_head;
        wave_fence();
        for (int e = lane; e < D; e += 64) sq[e] = fw_to_f32(q[e]) * (p.scale == 0.0f ? 0.0f : 1.0f); // as tree_query
        wave_fence();
        float m = -INFINITY, l = 0.0f, o[D / 64] = {};
        for (int j0 = b.first; j0 < b.last; j0 += 64) {
            const int j = j0 + lane;
            const bool yes = tree_sees(p, b.rq, i, j, b.last);
            float z = -INFINITY;
            int64_t at = -2; // not seen; -1: no page
            if (yes) {
                const uint32_t pi = fw_div((uint32_t)j, p.page);
                const int32_t id = trow[pi];
                at = (uint32_t)id < (uint32_t)p.n_pages ? (int64_t)tree_at(p, j - pi * p.page.d, id) : -1;
                z = at < 0 ? __builtin_nanf("") : 0.0f;
                if (at >= 0)
                    for (int e = 0; e < D; e++) z = fmaf(sq[e], fw_to_f32(((const T *)(kbase + at))[e]), z);
                z = z * (p.scale * 1.44269504088896340736f);
            }
            if (!__any(yes)) continue;
            const float mn = fmaxf(m, fw_wave_max(z)), base = tree_base(mn);
            const float w = yes ? __builtin_amdgcn_exp2f(z - base) : 0.0f, f = __builtin_amdgcn_exp2f(m - TREE_BIAS - base);
            l = l * f + fw_wave_sum(w);
            m = mn;
            sp[lane] = w;
            sat[lane] = at;
            wave_fence();
            for (int x = 0; x < D / 64; x++) {
                float a = f == 1.0f ? o[x] : o[x] * f;
                for (int k = 0; k < 64; k++)
                    if (sat[k] >= 0) a = fmaf(sp[k], fw_to_f32(((const T *)(vbase + sat[k]))[x * 64 + lane]), a);
                    else if (sat[k] == -1) a += sp[k]; // NaN
                o[x] = a;
            }
            wave_fence();
        }
        if (b.whole) {
            T *out = (T *)p.out + (int64_t)(b.rq.row0 + i) * p.out_row + h * p.out_head;
            const bool any = tree_sees_any(p, b.rq, i);
            for (int x = 0; x < D / 64; x++) out[x * 64 + lane] = fw_cvt<T>(any ? o[x] / l : 0.0f);
        } else {
            float *part = b.part(p, D, t - b.t0);
            for (int x = 0; x < D / 64; x++) part[x * 64 + lane] = o[x];
            if (lane == 0) {
                part[D] = m;
                part[D + 1] = l;
            }
        }
    }
}

// Few rows (at most 16): the four waves take the chunk's steps of KEYS keys in
// turn, all with the same rows, and are joined at the end.  Bound by the cache's
// bytes, so nothing stands between memory and the lanes: a wave's K tile goes
// straight to the registers that multiply it, its V tile through LDS of its
// own, where the transposing read gives each lane the keys of one feature.  The
// next step's tiles are in flight while a step computes; no barriers.
// One token of 64 requests over 4,096 cached each (32 heads on 8, 128 wide, bf16): 172 us,
// 4.66 TB/s.  One request of 225 keys (f32) takes 10 us, four dependent steps a wave.
template <typename T, int D>
__global__ void __launch_bounds__(256, 2) k_tree_few(TreeP p) {
    typedef Rows<T, D, 1> R;
    constexpr int KT = R::KT, KEYS = R::KEYS, NS = R::NS;
    constexpr int VROW = D * (int)sizeof(T) + 32; // bytes of a V row in LDS: rows 8 banks apart
    constexpr int VBYTES = 4 * KEYS * VROW, OBYTES = 16 * D * 4;
    __shared__ __attribute__((aligned(16))) char lds[VBYTES > OBYTES ? VBYTES : OBYTES];
    __shared__ float sm[64], sl[64];
    TreeBlock b;
    if (!b.find<T, D>(p)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, c = lane >> 4;
    R rows;
    rows.load(p, b.rq, b.t0, b.total, b.kvh, b.group);
    const float zs = tree_zs(p);
    char *vt = lds + wave * KEYS * VROW;
    const int32_t *trow = p.table + (int64_t)b.r * p.table_stride;
    const char *kbase = (const char *)((const T *)p.kc + b.kvh * p.head_stride) + c * 16;
    const char *vbase = (const char *)((const T *)p.vc + b.kvh * p.head_stride) + c * 16;
    const int last = b.last;

    {
        int32_t id[KT];
        uint32_t tok[KT]; // within the page
        u4 kf[KT][NS], vf[KT][NS];
        bool gone[KT]; // no such key
        auto pages = [&](int j) {
#pragma unroll
            for (int k = 0; k < KT; k++) {
                const int key = j + k * 16 + lr;
                const uint32_t pi = fw_div((uint32_t)key, p.page);
                id[k] = key < last ? trow[pi] : -1;
                tok[k] = key - pi * p.page.d;
            }
        };
        auto load = [&] {
#pragma unroll
            for (int k = 0; k < KT; k++) {
                gone[k] = (uint32_t)id[k] >= (uint32_t)p.n_pages;
                const uint64_t at = gone[k] ? 0 : tree_at(p, tok[k], id[k]);
                const char *ka = kbase + at, *va = vbase + at;
#pragma unroll
                for (int s = 0; s < NS; s++) kf[k][s] = *(const u4 *)(ka + s * 64);
#pragma unroll
                for (int s = 0; s < NS; s++) vf[k][s] = *(const u4 *)(va + s * 64);
            }
        };
        rows.clear();
        int j0 = b.first + wave * KEYS;
        if (j0 < last) {
            pages(j0);
            load();
            pages(j0 + 4 * KEYS);
        }
        for (; j0 < last; j0 += 4 * KEYS) {
            if (__builtin_expect(__any(gone[0] || gone[KT - 1]), 0)) {
#pragma unroll
                for (int k = 0; k < KT; k++)
                    if (gone[k])
#pragma unroll
                        for (int s = 0; s < NS; s++) {
                            kf[k][s] = ~u4{}; // NaN for whoever sees it
                            vf[k][s] = u4{};
                        }
            }
            f4 z[1][KT];
#pragma unroll
            for (int k = 0; k < KT; k++) {
                f4 a = {};
#pragma unroll
                for (int s = 0; s < NS; s++) a = Mma<T>::dot(kf[k][s], rows.q[0][s], a);
                z[0][k] = a;
            }
            wave_fence();
#pragma unroll
            for (int k = 0; k < KT; k++)
#pragma unroll
                for (int s = 0; s < NS; s++)
                    *(u4 *)(vt + (k * 16 + lr) * VROW + s * 64 + c * 16) = vf[k][s];
            wave_fence();
            if (j0 + 4 * KEYS < last) {
                load();
                pages(j0 + 8 * KEYS);
            }
            if (__builtin_expect(j0 + KEYS > b.clear, 0)) rows.mask(p, b.rq, 0, j0, last, z[0]);
            rows.weigh(z, zs);
            rows.template add<VROW>(vt, z);
        }
    }
    if (__syncthreads_or(rows.odd())) { // and the V tiles become the outputs' place
        tree_slow<T, D>(p, b, lds);
        return;
    }
    rows.l[0] = quarters_sum(rows.l[0]);
    rows.join(wave, 4, 0, 16, sm, sl, (float *)lds);
    if (wave == 0) rows.store(p, b, b.t0);
}

// More rows: WR waves take RT tiles of rows each, 4 / WR waves the same rows
// with different keys.  All share the K and V tiles of a step, which come
// through registers into one of two places in LDS: while a step computes, the
// next step's tiles are on their way from memory and one barrier a step
// separates the two places.
// 16 requests x 16 drafted tokens over 32,768 cached each (32 heads on 8, bf16, 64 rows a
// block): 318 us, 4.87 TB/s, the cache's bytes once.  64 drafted tokens over 131,061
// (f16, 128 rows a block): 280 us, 490 TFLOP/s of the formula's products, where the vector
// instructions (weights, their two halves) are active 56% of the time and the matrix
// units 35%; 32 rows a wave fill the registers.
template <typename T, int D, int RT, int WR>
__global__ void __launch_bounds__(256, RT > 1 ? 2 : D == 64 && sizeof(T) == 2 ? 4 : 3) k_tree_wide(TreeP p) {
    typedef Rows<T, D, RT> R;
    constexpr int KT = R::KT, KEYS = R::KEYS, NS = R::NS, WK = 4 / WR, TK = WK * KEYS; // keys of a step
    constexpr int NC = D * (int)sizeof(T) / 16, NL = TK * NC / 256; // 16-byte pieces of a key; of a thread, for K and for V
    constexpr int KROW = D * (int)sizeof(T) + 16;                              // rows 4 banks apart: 16-byte reads
    constexpr int VROW = D * (int)sizeof(T) + (sizeof(T) == 2 ? 32 : 16);      // 8 apart: the transposing reads
    constexpr int TILE = TK * (KROW + VROW), OBYTES = WK > 1 ? WR * RT * 16 * D * 4 : 0;
    __shared__ __attribute__((aligned(16))) char lds[2 * TILE > OBYTES ? 2 * TILE : OBYTES];
    __shared__ float sm[WK * WR * RT * 16], sl[WK * WR * RT * 16];
    TreeBlock b;
    if (!b.find<T, D>(p)) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, c = lane >> 4;
    const int wr = wave / WK, wk = wave % WK, t0 = b.t0 + wr * RT * 16;
    R rows;
    rows.load(p, b.rq, t0, b.total, b.kvh, b.group);
    const float zs = tree_zs(p);
    const int32_t *trow = p.table + (int64_t)b.r * p.table_stride;
    const int piece = threadIdx.x % NC, own = threadIdx.x / NC; // keys own + i * (256 / NC) of a step
    const char *kbase = (const char *)((const T *)p.kc + b.kvh * p.head_stride) + piece * 16;
    const char *vbase = (const char *)((const T *)p.vc + b.kvh * p.head_stride) + piece * 16;
    const int last = b.last;

    {
        int32_t id[NL];
        uint32_t tok[NL]; // within the page
        u4 kf[NL], vf[NL];
        bool gone[NL]; // no such key
        auto pages = [&](int j) {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int key = j + own + i * (256 / NC);
                const uint32_t pi = fw_div((uint32_t)key, p.page);
                id[i] = key < last ? trow[pi] : -1;
                tok[i] = key - pi * p.page.d;
            }
        };
        auto load = [&] {
#pragma unroll
            for (int i = 0; i < NL; i++) {
                gone[i] = (uint32_t)id[i] >= (uint32_t)p.n_pages;
                const uint64_t at = gone[i] ? 0 : tree_at(p, tok[i], id[i]);
                kf[i] = *(const u4 *)(kbase + at);
                vf[i] = *(const u4 *)(vbase + at);
            }
        };
        auto put = [&](char *at) {
            bool any = false;
#pragma unroll
            for (int i = 0; i < NL; i++) any |= gone[i];
            if (__builtin_expect(__any(any), 0)) {
#pragma unroll
                for (int i = 0; i < NL; i++)
                    if (gone[i]) {
                        kf[i] = ~u4{}; // NaN for whoever sees it
                        vf[i] = u4{};
                    }
            }
#pragma unroll
            for (int i = 0; i < NL; i++) {
                const int key = own + i * (256 / NC);
                *(u4 *)(at + key * KROW + piece * 16) = kf[i];
                *(u4 *)(at + TK * KROW + key * VROW + piece * 16) = vf[i];
            }
        };
        rows.clear();
        int j0 = b.first;
        pages(j0);
        load();
        pages(j0 + TK);
        put(lds);
        load();
        pages(j0 + 2 * TK);
        __syncthreads();
        for (int at = 0; j0 < last; j0 += TK, at ^= 1) {
            const char *kt = lds + at * TILE + wk * KEYS * KROW, *vt = lds + at * TILE + TK * KROW + wk * KEYS * VROW;
            put(lds + (at ^ 1) * TILE);
            load();
            pages(j0 + 3 * TK);
            f4 z[RT][KT];
#pragma unroll
            for (int k = 0; k < KT; k++) {
                u4 f[NS];
#pragma unroll
                for (int s = 0; s < NS; s++) f[s] = *(const u4 *)(kt + (k * 16 + lr) * KROW + s * 64 + c * 16);
#pragma unroll
                for (int x = 0; x < RT; x++) {
                    f4 a = {};
#pragma unroll
                    for (int s = 0; s < NS; s++) a = Mma<T>::dot(f[s], rows.q[x][s], a);
                    z[x][k] = a;
                }
            }
            const int j = j0 + wk * KEYS;
            if (__builtin_expect(j + KEYS > b.clear, 0))
#pragma unroll
                for (int x = 0; x < RT; x++) rows.mask(p, b.rq, x, j, last, z[x]);
            rows.weigh(z, zs);
            rows.template add<VROW>(vt, z);
            __syncthreads();
        }
    }
    if (__syncthreads_or(rows.odd())) {
        tree_slow<T, D>(p, b, lds);
        return;
    }
#pragma unroll
    for (int x = 0; x < RT; x++) rows.l[x] = quarters_sum(rows.l[x]);
    if constexpr (WK > 1) rows.join(wk, WK, wr * RT * 16, WR * RT * 16, sm, sl, (float *)lds);
    if (wk == 0) rows.store(p, b, t0);
}

// The parts of a request's units into its outputs: NW waves a row and head.  64
// parts at a time a lane each finds their weights, then D / 4 lanes a part and
// 256 NW / D parts at once add them up.  One wave where there are many rows, four
// where few rows have many parts.
template <typename T, int D, int NW>
__global__ void __launch_bounds__(256) k_tree_join(TreeP p) {
    constexpr int W = D / 4, N = 64 * NW, G = N / W; // G parts at once
    __shared__ f4 sum[256 / W][W];
    const int r = blockIdx.z, h = blockIdx.y, tid = threadIdx.x % N, own = threadIdx.x / N, lane = threadIdx.x & 63;
    const TreeReq rq = tree_req(p, r);
    const int group = p.heads / p.kv_heads, kvh = h / group;
    const TreeUnits un = tree_units(p, -1, r);
    const int64_t step = (int64_t)p.tiles * p.kv_heads * p.tile_rows * (D + 4);
    for (int64_t i = (int64_t)blockIdx.x * (256 / N) + own; i < rq.n; i += (int64_t)gridDim.x * (256 / N)) {
        T *out = (T *)p.out + (rq.row0 + i) * p.out_row + (int64_t)h * p.out_head;
        if (rq.bad) {
            if (tid < W) *(typename Vec4<T>::type *)(out + 4 * tid) = pack4<T>(f4{} + __builtin_nanf(""));
            continue;
        }
        const bool any = tree_sees_any(p, rq, (int)i);
        const int t = (int)i * group + h % group, tile = t / p.tile_rows;
        const int keys = rq.len + (p.words ? rq.n : (min((tile + 1) * p.tile_rows, rq.n * group) - 1) / group + 1);
        const int parts = (keys + un.chunk - 1) / un.chunk; // at most un.count
        const float *at = p.parts + un.first * step + (((int64_t)tile * p.kv_heads + kvh) * p.tile_rows + t % p.tile_rows) * (D + 4);
        float mx = -INFINITY;
        for (int s = lane; s < parts; s += 64) mx = fmaxf(mx, at[s * step + D]);
        mx = fw_dpp_wave_max(mx);
        const float base = tree_base(mx);
        float l = 0.0f;
        f4 o = {};
        for (int s0 = 0; s0 < parts; s0 += 64) {
            float mine = 0.0f;
            if (s0 + lane < parts) {
                const float2 ml = *(const float2 *)(at + (s0 + lane) * step + D);
                mine = __builtin_amdgcn_exp2f(ml.x - TREE_BIAS - base);
                l = fmaf(mine, ml.y, l);
            }
            const int n = min(parts - s0, 64);
#pragma unroll 4
            for (int k = 0; k < n; k += G) { // the same turns for every lane: the exchange needs them all
                const int s = k + tid / W;
                const float f = __shfl(mine, s & 63);
                if (s < n) {
                    const f4 v = *(const f4 *)(at + (s0 + s) * step + 4 * (tid % W));
#pragma unroll
                    for (int e = 0; e < 4; e++) o[e] = fmaf(f, v[e], o[e]);
                }
            }
        }
        l = fw_wave_sum(l);
        f4 *all = &sum[own * G][0];
        all[tid] = o;
        if constexpr (NW == 1) wave_fence();
        else __syncthreads();
        if (tid < W) {
#pragma unroll
            for (int g = 1; g < G; g++) o += all[g * W + tid];
            const float inv = 1.0f / l;
            const f4 v = l == 0.0f ? f4{} + __builtin_nanf("") : o * inv; // 0 / 0: every key scored -inf
            *(typename Vec4<T>::type *)(out + 4 * tid) = pack4<T>(any ? v : f4{});
        }
        if constexpr (NW == 1) wave_fence();
        else __syncthreads();
    }
}

// How a call of these sizes is cut.  Up to 16 rows per K/V head share one tile
// (k_tree_few); 32, 64 or 128 rows a block above that (k_tree_wide), 128 only over
// long caches, where what a block reads matters more than how many blocks there
// are.  Where that gives fewer than 256 (one a CU) the keys are cut into units
// (tree_units), as many as run at once: 2 to 4 blocks a CU, by the registers and
// LDS of the kernel.
// Measured on both sides, us, this rule / the other:
//   24 requests x 8 over 4,096 (192 blocks) cut 90 / 109 whole, 20 x 32 over 3,000 (160)
//     98 / 119; 32 x 1 over 4,096 (256) whole 92 / 107 cut, 40 x 16 over 2,048 (320) 83 / 91;
//   units of 128 keys or more, 1 x 1 over 2,048 13.8 / 15.9 (256) / 19.8 (512), 16 x 1 over
//     1,024 22.6 / 22.7 / 26.0; up to 512 keys whole: 10 x 16 over 440 (20 heads) 12.5 / 16.8
//     cut, 1 x 8 over 217 10.2 / 13.2: the join is a launch and its latency;
//   64 rows a block over short caches, 10 chains of 224 over 224 (20 heads of 64) 21.3 / 24.0,
//     64 of them 79 / 93, one of 500 (32 heads on 8, of 128) 21.0 / 26.5, but 10 x 200 over 100
//     28.3 / 27.0; 128 over long ones, 1 x 64 over 131,061 277 / 310, 8 x 512 over 4,096 401 / 415,
//     2 x 64 over 32,768 (heads of 64) 86 / 92.
struct TreeCut {
    int rows, units;
    int64_t tiles;
    uint64_t bytes;
};
static TreeCut tree_cut(int32_t n_req, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim, int32_t max_new,
                        int32_t max_len) {
    TreeCut t;
    const int64_t rows = (int64_t)max_new * (n_heads / n_kv_heads);
    t.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : rows <= 64 || max_len <= TREE_WHOLE ? 64 : 128;
    t.tiles = (rows + t.rows - 1) / t.rows;
    const int64_t at_once = head_dim == 64 ? (t.rows == 128 ? 768 : TREE_UNITS) : t.rows == 32 || t.rows == 128 ? 512 : 768;
    const int64_t per = std::max<int64_t>(1, (int64_t)n_kv_heads * t.tiles), base = per * n_req;
    const int64_t most = max_len <= TREE_WHOLE ? 0 : ((int64_t)max_len + TREE_CHUNK - 1) / TREE_CHUNK * n_req; // units of TREE_CHUNK
    const int64_t units = std::min(at_once / per, most);
    t.units = base >= 256 || units <= n_req ? 0 : (int)units;
    // enough for every smaller call too
    t.bytes = (uint64_t)std::min(at_once, per * most) * t.rows * (head_dim + 4) * 4;
    return t;
}

template <typename T, int D>
static void tree_go(hipStream_t st, const TreeP &p, int n_req) {
    // without units a block per request
    const dim3 grid(p.kv_heads * p.tiles, p.units ? p.units : n_req), block(256);
    if (p.tile_rows == 16) hipLaunchKernelGGL((k_tree_few<T, D>), grid, block, 0, st, p);
    else if (p.tile_rows == 32) hipLaunchKernelGGL((k_tree_wide<T, D, 1, 2>), grid, block, 0, st, p);
    else if (p.tile_rows == 64) hipLaunchKernelGGL((k_tree_wide<T, D, 1, 4>), grid, block, 0, st, p);
    else hipLaunchKernelGGL((k_tree_wide<T, D, 2, 4>), grid, block, 0, st, p);
    if (!p.units) return;
    // about four blocks a CU, each going through several rows where there are more
    const bool one = (int64_t)p.max_new * p.heads * n_req >= 1024;
    const int64_t rows = one ? ((int64_t)p.max_new + 3) / 4 : p.max_new, most = std::max(1, 1024 / std::max(1, p.heads * n_req));
    const dim3 jgrid((unsigned)std::max<int64_t>(1, std::min(rows, most)), p.heads, n_req);
    if (one) hipLaunchKernelGGL((k_tree_join<T, D, 1>), jgrid, block, 0, st, p);
    else hipLaunchKernelGGL((k_tree_join<T, D, 4>), jgrid, block, 0, st, p);
}
template <typename T>
static void tree_dim(hipStream_t st, int d, const TreeP &p, int n_req) {
    if (d == 64) tree_go<T, 64>(st, p, n_req);
    else tree_go<T, 128>(st, p, n_req);
}

extern "C" fwhip_status fwhip_tree_attn_workspace(int32_t n_req, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                                  int32_t max_new, int32_t max_len, uint64_t *bytes) {
    if (!bytes) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn_workspace: bytes is NULL");
    if (n_req < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || max_new < 0 || max_len < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn_workspace: bad size");
    if (head_dim != 64 && head_dim != 128)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_tree_attn_workspace: head_dim must be 64 or 128");
    *bytes = tree_cut(n_req, n_heads, n_kv_heads, head_dim, max_new, max_len).bytes;
    return FWHIP_OK;
}

extern "C" fwhip_status fwhip_tree_attn(fwhip_ctx *c, const fwhip_tree_attn_args *a) {
    if (!a) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: args is NULL");
    if (!fw_is_dtype(a->dtype)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: unknown element type");
    if (a->n_req < 0 || a->n_rows < 0 || a->n_pages < 0 || a->width < 0 || a->max_new < 0 || a->max_len < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: negative size");
    if (a->n_heads < 1 || a->n_kv_heads < 1 || a->n_heads % a->n_kv_heads || a->n_heads > 65535)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: n_kv_heads must divide n_heads, n_heads in 1..65535");
    if (a->head_dim != 64 && a->head_dim != 128)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_tree_attn: head_dim must be 64 or 128");
    if (a->page_size < 1 || a->page_size > (1 << 24))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: page_size must be in 1..2^24");
    if ((int64_t)a->max_len > (int64_t)a->width * a->page_size || a->max_len > 0x7fff0000)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: max_len exceeds the table (width * page_size)");
    if (a->n_req > 65535) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: n_req must be below 65536");
    const int64_t strides[] = {a->table_stride, a->q_row, a->q_head, a->out_row, a->out_head, a->page_stride,
                               a->token_stride, a->head_stride};
    for (int64_t s : strides)
        if (s < 0) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: negative stride");
    if (a->n_req && a->n_rows) {
        if (!a->q || !a->out || !a->len || !a->row_start || !a->table || (a->n_pages && (!a->k_cache || !a->v_cache)))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: NULL argument");
        if (a->n_pages < 1) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: a cache of no pages");
        const int eb = fw_dtype_bytes(a->dtype);
        if (!fw_aligned(a->q, 16) || !fw_aligned(a->k_cache, 16) || !fw_aligned(a->v_cache, 16) || !fw_aligned(a->out, 16))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: q, the caches and out must be 16-byte aligned");
        for (int k = 1; k < 8; k++)
            if (strides[k] * eb % 16)
                return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: strides must be multiples of 16 bytes");
        if (!fw_aligned(a->table, 4) || !fw_aligned(a->len, 4) || !fw_aligned(a->row_start, 4) || !fw_aligned(a->mask, 8))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: an address is not a multiple of its element's size");
        const int64_t qn = (a->n_heads - 1) * a->q_head + a->head_dim, on = (a->n_heads - 1) * a->out_head + a->head_dim;
        if (fw_rows_overlap(a->out, a->out_row, on, a->q, a->q_row, qn, a->n_rows, eb))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: out must not overlap q");
    }
    if (a->page_stride > 0x3fffffff || a->token_stride > 0x3fffffff)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_tree_attn: page and token strides must be below 2^30 elements");
    if (!(fabsf(a->scale) < INFINITY)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: scale must be finite");
    if (a->mask ? a->mask_words < 1 || (int64_t)a->mask_words * 64 < a->max_new : a->mask_words != 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: mask needs 64 * mask_words >= max_new (mask_words 0 without)");
    uint64_t need = 0;
    fwhip_status rc = fwhip_tree_attn_workspace(a->n_req, a->n_heads, a->n_kv_heads, a->head_dim, a->max_new, a->max_len,
                                                &need);
    if (rc != FWHIP_OK) return rc;
    if (need && (!a->workspace || a->workspace_bytes < need || !fw_aligned(a->workspace, 16)))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: workspace too small (fwhip_tree_attn_workspace) or not 16-byte aligned");
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: NULL ctx");
    if (a->n_req == 0 || a->n_rows == 0 || a->max_new == 0) return FWHIP_OK;
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_tree_attn: hipSetDevice failed");
    TreeP p;
    p.n_req = a->n_req;
    p.n_rows = a->n_rows;
    p.heads = a->n_heads;
    p.kv_heads = a->n_kv_heads;
    p.n_pages = a->n_pages;
    p.width = a->width;
    p.max_new = a->max_new;
    p.max_len = a->max_len;
    p.words = a->mask ? a->mask_words : 0;
    p.scale = a->scale;
    p.page = fw_div_make((uint32_t)a->page_size);
    p.table_stride = a->table_stride;
    p.q_row = a->q_row;
    p.q_head = a->q_head;
    p.out_row = a->out_row;
    p.out_head = a->out_head;
    p.page_bytes = (uint32_t)(a->page_stride * fw_dtype_bytes(a->dtype));
    p.token_bytes = (uint32_t)(a->token_stride * fw_dtype_bytes(a->dtype));
    p.head_stride = a->head_stride;
    p.q = a->q;
    p.kc = a->k_cache;
    p.vc = a->v_cache;
    p.table = a->table;
    p.len = a->len;
    p.row_start = a->row_start;
    p.mask = a->mask;
    p.out = a->out;
    const TreeCut cut = tree_cut(a->n_req, a->n_heads, a->n_kv_heads, a->head_dim, std::min(a->max_new, a->n_rows), a->max_len);
    if (cut.tiles * a->n_kv_heads > 1 << 23) // threads of a grid's first dimension stay below 2^32
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_tree_attn: more than 2^23 row tiles x K/V heads");
    p.tiles = (int)cut.tiles;
    p.units = cut.units;
    p.tile_rows = cut.rows;
    p.parts = (float *)a->workspace;
    if (a->dtype == FWHIP_T_F32) tree_dim<float>(c->stream, a->head_dim, p, a->n_req);
    else if (a->dtype == FWHIP_T_F16) tree_dim<fw_f16>(c->stream, a->head_dim, p, a->n_req);
    else tree_dim<fw_bf16>(c->stream, a->head_dim, p, a->n_req);
    return fw_launched("fwhip_tree_attn");
}
