// q4.hip — linears with 4-bit weights and group scales (fwhip_q4_linear), and
// the planes they read from a ggml payload (fwhip_q4_planes).
//
// y[m][n] = sum_g d[n][g] (sum_{k in g} x[m][k] c[n][k]) + lo[n][g] (sum_{k in g} x[m][k]) + b[n]
// with codes c in 0..15 (lo = the minimum) or c - 8 (no minimum): the group's
// inner sums need whole-number codes only, and the scales enter once a group.
#include <algorithm>
#include <type_traits>

#include "fw_device.h"
#include "fw_serve.h"

struct Q4P {
    int m, n, k, group;
    int64_t ldx, ldy;
    const void *x;
    const uint8_t *q;
    const void *scale, *minimum;
    const float *bias;
    void *y;
    int scale32, vec, pair; // planes of f32; x rows 16-byte (f32) or 8-byte aligned; four f16 scales so aligned
    int chunk, stage, lds;   // inputs staged at a time; bytes of a stage, and of LDS in all
};

typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));

// A step is 128 inputs (four 32-weight blocks) of 16 outputs: lane l of a wave
// loads block l / 16 of row l % 16, 16 bytes, so a load covers 64 whole bytes of
// a row.  The product of one block wants bytes 4 c .. 4 c + 3 of that block in
// lane quarter c, which is the 4 x 4 exchange of words between quarters below:
// two swaps of half waves, two of quarters.
__device__ __forceinline__ void q4_exchange(u4 &w) {
    auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
    auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
    auto x = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
    auto y = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
    w = u4{x[0], x[1], y[0], y[1]};
}
// The four quarters' values of one register, to every lane.
__device__ __forceinline__ f4 q4_quarters(float v) {
    const uint32_t u = __float_as_uint(v);
    auto a = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    auto e = __builtin_amdgcn_permlane32_swap(a[0], a[0], false, false);
    auto o = __builtin_amdgcn_permlane32_swap(a[1], a[1], false, false);
    return f4{__uint_as_float(e[0]), __uint_as_float(o[0]), __uint_as_float(e[1]), __uint_as_float(o[1])};
}

// Eight codes as operands of a product, in the order of a unit's inputs (below).
// f16: a code in the low bits of 1024 (or, four bits up, of 64) is that number
// plus the code; what is too much is taken off again, exactly, and with it the
// 8 of weights without minimums.
struct Q4Magic { // in registers: an instruction that masks and sets bits takes one constant from the scalars, none from the code
    uint32_t lo, hi;
};
__device__ __forceinline__ uint32_t q4_bits(uint32_t w, uint32_t mask, uint32_t set) { return (w & mask) | set; }
template <bool MIN>
__device__ __forceinline__ u4 q4_codes_f16(uint32_t w, Q4Magic k) {
    const uint32_t v = w >> 8;
    const h2 lo = MIN ? h2{(_Float16)1024, (_Float16)1024} : h2{(_Float16)1032, (_Float16)1032};
    const h2 hi = MIN ? h2{(_Float16)64, (_Float16)64} : h2{(_Float16)72, (_Float16)72};
    u4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, q4_bits(w, 0x000f000fu, k.lo)) - lo);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, q4_bits(w, 0x00f000f0u, k.hi)) - hi);
    r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, q4_bits(v, 0x000f000fu, k.lo)) - lo);
    r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, q4_bits(v, 0x00f000f0u, k.hi)) - hi);
    return r;
}
// bf16: 128 + code; there is no packed bf16 subtraction, so the 128 (and the 8)
// leave with the sums of the inputs (CORR below).  That costs five bits of the
// f32 sum, 2^-19 of the result against the 2^-9 of its rounding.
__device__ __forceinline__ u4 q4_codes_bf16(uint32_t w, Q4Magic k) {
    u4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = q4_bits(w >> (4 * i), 0x000f000fu, k.lo);
    return r;
}

// x in LDS, as the products read it: per row `chunk` inputs of 16 bits in units
// of 8, the unit (block, c) holding inputs 4 c + 0, 2, 16, 18, 1, 3, 17, 19 of its
// block.  f16 and bf16 as they are; f32 as two f16 parts of x / s, where s is
// the power of two that takes the largest |x| of the row's turn of inputs to
// 2^14..2^15: hi + lo is within 2^-22 of x, or 2^-39 of that largest (where the
// second part falls below f16's normal numbers).
template <typename T>
struct Q4X {
    static constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
};

// Four inputs as they lie in memory, and their values.
template <typename T>
struct Q4Four {
    typename std::conditional<sizeof(T) == 4, u4, uint2>::type v;
    __device__ __forceinline__ void load(const T *at, bool vec) {
        if (vec) v = *(const decltype(v) *)at;
        else if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = ((const uint32_t *)at)[i];
        } else {
            const uint16_t *a = (const uint16_t *)at;
            v = make_uint2(a[0] | (uint32_t)a[1] << 16, a[2] | (uint32_t)a[3] << 16);
        }
    }
    __device__ __forceinline__ void clear() { v = decltype(v){}; }
    __device__ __forceinline__ float sum(float t) const { // t + the four
        if constexpr (sizeof(T) == 4) return t + ((__uint_as_float(v[0]) + __uint_as_float(v[1])) + (__uint_as_float(v[2]) + __uint_as_float(v[3])));
        else if constexpr (std::is_same<T, fw_bf16>::value) {
            typedef __bf16 b2 __attribute__((ext_vector_type(2)));
            const b2 one = {(__bf16)1.0f, (__bf16)1.0f};
            t = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, v.x), one, t, false);
            return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, v.y), one, t, false);
        } else {
            const h2 one = {(_Float16)1.0f, (_Float16)1.0f};
            t = __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.x), one, t, false);
            return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, v.y), one, t, false);
        }
    }
};
__device__ __forceinline__ uint32_t q4_pair(float a, float b) { return fw_cvt<fw_f16>(a).b | (uint32_t)fw_cvt<fw_f16>(b).b << 16; }

// One output, product by product: w = (code - 8) scale or code scale + minimum.
template <typename T, bool MIN>
__device__ __forceinline__ float q4_one(const Q4P &p, int m, int n) {
    float acc = 0.0f;
    for (int k = 0; k < p.k; k++) {
        const uint8_t byte = p.q[(int64_t)n * (p.k / 2) + (k >> 5) * 16 + (k & 15)];
        const float code = (float)(k & 16 ? byte >> 4 : byte & 15);
        const int64_t g = (int64_t)n * (p.k / p.group) + k / p.group;
        const float d = p.scale32 ? ((const float *)p.scale)[g] : fw_to_f32(((const fw_f16 *)p.scale)[g]);
        float w = (code - 8.0f) * d;
        if (MIN) w = fmaf(code, d, p.scale32 ? ((const float *)p.minimum)[g] : fw_to_f32(((const fw_f16 *)p.minimum)[g]));
        acc = fmaf(fw_to_f32(((const T *)p.x)[m * p.ldx + k]), w, acc);
    }
    return acc;
}

// The kernel: MT * 16 rows of x by WN waves of NT * 16 outputs each, WK waves
// taking turns of MS steps of the same outputs.  Each weight is read once, and
// straight into the registers that multiply it, a turn ahead; x is what many
// lanes need, so it goes through LDS: all of it where it fits, else in two stages
// of `chunk` inputs, one on its way while the other is read.  Beside x lie its
// sums, where weights have a minimum: what the minimums (and the offsets of the
// codes) add is one more small product, of sums and scales.  GB: the 32-weight
// blocks of a group.  Of a turn's 4 MS blocks a lane quarter loads the scales of
// its MS, which the quarters then exchange.
//
// Bound by the weights' bytes up to about 16 rows: one row through 28,672 x 8,192
// (bf16, groups of 128 with minimums) takes 29 us, 4.3 TB/s where the same access
// alone takes 24 (4.9), sixteen rows 37 us: staging x for 224 blocks is the rest.
// With more rows by the instructions around the products (unpacking, scales): 1,500
// rows through 5,120 x 1,280 (f16, groups of 32 with minimums) take 58 us, 336
// TFLOP/s; 2,048 through 8,192 x 4,096 (bf16, groups of 128) 255 us, 538 TFLOP/s.
template <typename T, bool MIN, int GB, int MT, int NT, int WN, int WK, int MS>
__global__ void __launch_bounds__(64 * WN * WK) k_q4(Q4P p) {
    constexpr bool BF = std::is_same<T, fw_bf16>::value, F32 = std::is_same<T, float>::value, CORR = MIN || BF;
    constexpr int PARTS = Q4X<T>::PARTS, NW = WN * WK, R = MT * 16;
    constexpr int SP = MS > GB ? MS / GB : 1;     // scales a lane loads a turn
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, lr = lane & 15, c = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); // the same in all lanes: loops and branches stay scalar
    const int wn = wave / WK, wk = wave % WK;
    const int m0 = blockIdx.y * R, rows = min(R, p.m - m0);
    const int n0 = (blockIdx.x * WN + wn) * NT * 16;
    const int cturns = p.chunk / (128 * MS), turns = (p.k + 128 * MS - 1) / (128 * MS);
    const int xrow = p.chunk * 2 + 16; // bytes of a row: rows 4 banks apart
    const int plane = rows * xrow;
    char *stage0 = lds; // one or two stages: x [part][row][xrow], CORR: sums [turn][MS][4][R], f32: scales [turn][R]
    Q4Magic magic = BF ? Q4Magic{0x43004300u, 0} : Q4Magic{0x64006400u, 0x54005400u};
    asm volatile("" : "+v"(magic.lo), "+v"(magic.hi));

    f4 acc[MT][NT];
#pragma unroll
    for (int x = 0; x < MT; x++)
#pragma unroll
        for (int y = 0; y < NT; y++) acc[x][y] = f4{};

    const int groups = p.k / (32 * GB), blocks = p.k / 32;
    const uint8_t *qrow[NT];
    int64_t srow[NT];
#pragma unroll
    for (int y = 0; y < NT; y++) {
        const int n = min(n0 + y * 16 + lr, p.n - 1); // the last again behind the end
        qrow[y] = p.q + (int64_t)n * (p.k / 2);
        srow[y] = (int64_t)n * groups;
    }
    // a turn's weights and scales, as stored (converting here would wait for them)
    u4 wq[MS][NT];
    uint32_t sc[SP][NT], mn[SP][NT];
    auto load = [&](int t) {
        const bool whole = (t + 1) * 4 * MS <= blocks;
#pragma unroll
        for (int y = 0; y < NT; y++) {
#pragma unroll
            for (int u = 0; u < MS; u++) {
                int blk = (t * MS + u) * 4 + c;
                if (!whole) blk = min(blk, blocks - 1);
                wq[u][y] = *(const u4 *)(qrow[y] + (uint32_t)blk * 16);
            }
            const int g = (t * 4 + c) * MS / GB; // the first of this quarter's groups
            if (!p.scale32 && p.pair && SP == 4 && whole) { // four f16 in one load
                const uint2 a = *(const uint2 *)((const uint16_t *)p.scale + srow[y] + g);
                sc[0][y] = a.x, sc[1][y] = a.x >> 16, sc[2][y] = a.y, sc[3][y] = a.y >> 16;
                if (MIN) {
                    const uint2 b = *(const uint2 *)((const uint16_t *)p.minimum + srow[y] + g);
                    mn[0][y] = b.x, mn[1][y] = b.x >> 16, mn[2][y] = b.y, mn[3][y] = b.y >> 16;
                }
            } else {
#pragma unroll
                for (int j = 0; j < SP; j++) {
                    const int64_t at = srow[y] + min(g + j, groups - 1);
                    if (p.scale32) {
                        sc[j][y] = ((const uint32_t *)p.scale)[at];
                        if (MIN) mn[j][y] = ((const uint32_t *)p.minimum)[at];
                    } else {
                        sc[j][y] = ((const uint16_t *)p.scale)[at];
                        if (MIN) mn[j][y] = ((const uint16_t *)p.minimum)[at];
                    }
                }
            }
        }
    };
    auto value = [&](uint32_t v) { return p.scale32 ? __uint_as_float(v) : fw_to_f32(fw_f16{(uint16_t)v}); };

    // staging x: a unit of 8 inputs per lane, 16 MS of them a row's turn; AT rows'
    // turns a lane are on their way from memory at once
    constexpr int UN = 16 * MS, PER = NW * 64 / UN;
    // fewer where their registers would be missed: f32 fetches are twice as wide, and
    // 8 tiles with a scale a block fill the file
    constexpr int AT = F32 ? 2 : MT * NT >= 8 && GB == 1 ? 1 : 4;
    const int u = lane % UN, item0 = threadIdx.x / UN;
    const float per_row = 1.0f / (float)rows; // (i + 1/2) / rows, cut, is i / rows: items stay below 2^16
    // A lane's items of a batch: row and turn within the stage, where their inputs
    // begin in memory and their units in LDS.  The first batch is the same in every
    // stage but for the turns before it, so this is found once.
    struct Items {
        int r[AT], t[AT];
        const T *from[AT];
    };
    Q4Four<T> xe[AT], xh[AT];
    auto items = [&](int i0, int n) {
        Items w;
#pragma unroll
        for (int j = 0; j < AT; j++) {
            const int it = i0 + j * PER;
            w.t[j] = it < n ? (int)(((float)it + 0.5f) * per_row) : 1 << 20; // none: behind the last turn
            w.r[j] = it < n ? it - w.t[j] * rows : 0;
            w.from[j] = (const T *)p.x + (int64_t)(m0 + w.r[j]) * p.ldx + (it < n ? (int64_t)w.t[j] * (128 * MS) : 0) + ((u >> 2) * 32 + (u & 3) * 4);
        }
        return w;
    };
    auto inside = [&](const Items &w, int t0, int j) { return (t0 + w.t[j]) * 4 * MS + (u >> 2) < blocks; };
    auto fetch = [&](const Items &w, int t0) {
#pragma unroll
        for (int j = 0; j < AT; j++) {
            const T *at = inside(w, t0, j) ? w.from[j] + (int64_t)t0 * (128 * MS) : (const T *)p.x;
            xe[j].load(at, p.vec);
            xh[j].load(at + 16, p.vec);
        }
    };
    auto put = [&](const Items &w, int t0, int to, char *xt) {
        float *sums = (float *)(xt + PARTS * plane), *scal = sums + (CORR ? cturns * MS * 4 * R : 0);
#pragma unroll
        for (int j = 0; j < AT; j++) {
            const int t = w.t[j], r = w.r[j];
            if (t >= to - t0) continue;
            if (!inside(w, t0, j)) {
                xe[j].clear();
                xh[j].clear();
            }
            if constexpr (CORR) {
                // sums of the inputs of each group (or part of one, where it is longer than a quarter)
                float v = xh[j].sum(xe[j].sum(0.0f));
                v = v + fw_dpp_f32<FW_DPP_XOR1>(v);
                v = v + fw_dpp_f32<FW_DPP_XOR2>(v);
                if constexpr (GB >= 2 && MS >= 2) v = v + fw_dpp_f32<FW_DPP_HALF_MIRROR>(v);
                if constexpr (GB >= 4 && MS >= 4) v = v + fw_dpp_f32<FW_DPP_MIRROR>(v);
                // block b of the turn: quarter b / MS, its scale (b % MS) / GB
                const int b = u >> 2;
                if ((u & 3) == 0 && b % MS % GB == 0) sums[((t * MS + b % MS / GB) * 4 + b / MS) * R + r] = v;
            }
            char *to_lds = xt + r * xrow + t * (256 * MS) + u * 16;
            if constexpr (F32) {
                float e[4], h[4], el[4], hl[4], mx = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = __uint_as_float(xe[j].v[i]);
                    h[i] = __uint_as_float(xh[j].v[i]);
                    mx = fmaxf(mx, fabsf(e[i]) < INFINITY ? fabsf(e[i]) : 0.0f);
                    mx = fmaxf(mx, fabsf(h[i]) < INFINITY ? fabsf(h[i]) : 0.0f);
                }
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_XOR1>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_XOR2>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_HALF_MIRROR>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_MIRROR>(mx));
#pragma unroll
                for (int o = 16; o < UN; o *= 2) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
                // mx = 1.f x 2^(ex - 127); x is scaled by 2^(14 - (ex - 127)), in two factors that are normal numbers
                const int ex = max((int)(__float_as_uint(mx) >> 23), 1), up = 141 - ex;
                const float f1 = __uint_as_float((uint32_t)(127 + up / 2) << 23), f2 = __uint_as_float((uint32_t)(127 + up - up / 2) << 23);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = e[i] * f1 * f2;
                    h[i] = h[i] * f1 * f2;
                    // second parts; of values that are not finite: nothing more
                    el[i] = fabsf(e[i]) < INFINITY ? e[i] - (float)(_Float16)e[i] : 0.0f;
                    hl[i] = fabsf(h[i]) < INFINITY ? h[i] - (float)(_Float16)h[i] : 0.0f;
                }
                // up is -113..140: the inverse 2^-up as a number, subnormal ones included
                if (u == 0) scal[t * R + r] = __builtin_ldexpf(1.0f, -up);
                *(u4 *)to_lds = u4{q4_pair(e[0], e[2]), q4_pair(h[0], h[2]), q4_pair(e[1], e[3]), q4_pair(h[1], h[3])};
                *(u4 *)(to_lds + plane) = u4{q4_pair(el[0], el[2]), q4_pair(hl[0], hl[2]), q4_pair(el[1], el[3]), q4_pair(hl[1], hl[3])};
            } else {
                const uint2 e = xe[j].v, h = xh[j].v;
                *(u4 *)to_lds = u4{__builtin_amdgcn_perm(e.y, e.x, 0x05040100), __builtin_amdgcn_perm(h.y, h.x, 0x05040100),
                                   __builtin_amdgcn_perm(e.y, e.x, 0x07060302), __builtin_amdgcn_perm(h.y, h.x, 0x07060302)};
            }
        }
    };

    const int stage_bytes = p.stage, full = rows * min(turns, cturns);
    const Items first = items(item0, full);
    // the items of a stage: the first batch is fetched already, the others (if any) here
    auto fill = [&](int t0, int to, char *xt) {
        put(first, t0, to, xt);
        for (int i0 = item0 + AT * PER; i0 < full; i0 += AT * PER) {
            const Items w = items(i0, full);
            fetch(w, t0);
            put(w, t0, to, xt);
        }
    };
    if (wk < turns) load(wk);
    fetch(first, 0);
    fill(0, min(turns, cturns), stage0);
    if (cturns < turns) fetch(first, cturns);
    __syncthreads();
    int mine = wk; // this wave's next turn
    for (int t0 = 0, at = 0; t0 < turns; t0 += cturns, at ^= 1) {
        const int to = min(turns, t0 + cturns);
        const char *xt = stage0 + at * stage_bytes;
        const float *sums = (const float *)(xt + PARTS * plane), *scal = sums + (CORR ? cturns * MS * 4 * R : 0);

        const char *xl[MT]; // this lane's units of each row tile (the last row again behind the end)
#pragma unroll
        for (int x = 0; x < MT; x++) xl[x] = xt + min(x * 16 + lr, rows - 1) * xrow + c * 16;
        for (; mine < to; mine += WK) {
            const int t = mine, tl = t - t0;
            u4 w[MS][NT];
            float d[SP][NT];
#pragma unroll
            for (int y = 0; y < NT; y++) {
#pragma unroll
                for (int u = 0; u < MS; u++) w[u][y] = wq[u][y];
#pragma unroll
                for (int j = 0; j < SP; j++) {
                    // blocks behind the last weigh nothing
                    const bool in = (t * 4 + c) * MS + j * GB < blocks;
                    d[j][y] = in ? value(sc[j][y]) : 0.0f;
                    if constexpr (CORR) {
                        // what every code is off by, times the inputs' sums: a product over the quarters' groups
                        float e = MIN ? (in ? value(mn[j][y]) : 0.0f) + (BF ? -128.0f * d[j][y] : 0.0f) : -136.0f * d[j][y];
                        // (a group longer than a quarter: each quarter has the sum of its own part)
#pragma unroll
                        for (int x = 0; x < MT; x++)
                            acc[x][y] = __builtin_amdgcn_mfma_f32_16x16x4f32(sums[((tl * MS + j) * 4 + c) * R + x * 16 + lr], e, acc[x][y], 0, 0, 0);
                    }
                }
            }
            if (t + WK < turns) load(t + WK);
            f4 dq[SP][NT];
#pragma unroll
            for (int y = 0; y < NT; y++)
#pragma unroll
                for (int j = 0; j < SP; j++) dq[j][y] = q4_quarters(d[j][y]);
            f4 mid[MT][NT];
            if constexpr (F32)
#pragma unroll
                for (int x = 0; x < MT; x++)
#pragma unroll
                    for (int y = 0; y < NT; y++) mid[x][y] = f4{};
            f4 dot[MT][NT];
#pragma unroll
            for (int u = 0; u < MS; u++) {
#pragma unroll
                for (int y = 0; y < NT; y++) q4_exchange(w[u][y]);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int b = u * 4 + i; // the turn's block
                    u4 code[NT];
#pragma unroll
                    for (int y = 0; y < NT; y++)
                        code[y] = BF ? q4_codes_bf16(w[u][y][i], magic) : q4_codes_f16<MIN>(w[u][y][i], magic);
#pragma unroll
                    for (int x = 0; x < MT; x++) {
                        const char *at = xl[x] + tl * (256 * MS) + b * 64;
                        const u4 a = *(const u4 *)at;
                        u4 al;
                        if constexpr (F32) al = *(const u4 *)(at + plane);
#pragma unroll
                        for (int y = 0; y < NT; y++) {
                            f4 z = b % GB ? dot[x][y] : f4{};
                            if constexpr (BF)
                                z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, code[y]), z, 0, 0, 0);
                            else {
                                if constexpr (F32)
                                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, al), __builtin_bit_cast(h8, code[y]), z, 0, 0, 0);
                                z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, code[y]), z, 0, 0, 0);
                            }
                            dot[x][y] = z;
                            if (b % GB == GB - 1 || b == 4 * MS - 1) {
                                const float f = dq[b % MS / GB][y][b / MS];
                                f4 &sum = F32 ? mid[x][y] : acc[x][y];
#pragma unroll
                                for (int j = 0; j < 4; j++) sum[j] = fmaf(f, z[j], sum[j]);
                            }
                        }
                    }
                }
            }
            if constexpr (F32) {
#pragma unroll
                for (int x = 0; x < MT; x++) {
                    const f4 f = *(const f4 *)(scal + tl * R + x * 16 + 4 * c);
#pragma unroll
                    for (int y = 0; y < NT; y++)
#pragma unroll
                        for (int j = 0; j < 4; j++) acc[x][y][j] = fmaf(f[j], mid[x][y][j], acc[x][y][j]);
                }
            }
        }
        if (to < turns) {
            const int t1 = min(turns, to + cturns);
            fill(to, t1, stage0 + (at ^ 1) * stage_bytes);
            if (t1 < turns) fetch(first, t1);
            __syncthreads();
        }
    }

    // the waves that shared outputs add up, in order
    if constexpr (WK > 1) {
        __syncthreads();
        f4 *part = (f4 *)stage0; // [wave][x][y][lane]
        if (wk)
#pragma unroll
            for (int x = 0; x < MT; x++)
#pragma unroll
                for (int y = 0; y < NT; y++) part[((wave * MT + x) * NT + y) * 64 + lane] = acc[x][y];
        __syncthreads();
        if (wk) return;
#pragma unroll
        for (int v = 1; v < WK; v++)
#pragma unroll
            for (int x = 0; x < MT; x++)
#pragma unroll
                for (int y = 0; y < NT; y++) acc[x][y] += part[(((wave + v) * MT + x) * NT + y) * 64 + lane];
    }
#pragma unroll
    for (int y = 0; y < NT; y++) {
        const int n = n0 + y * 16 + lr;
        if (n >= p.n) continue;
        const float bias = p.bias ? p.bias[n] : 0.0f;
#pragma unroll
        for (int x = 0; x < MT; x++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const int r = x * 16 + 4 * c + j;
                if (r >= rows) continue;
                float v = acc[x][y][j];
                // what an infinity or NaN, or a sum that overflowed on its way, left: once more, product by product
                if (__builtin_expect(!(fabsf(v) < INFINITY), 0)) v = q4_one<T, MIN>(p, m0 + r, n);
                ((T *)p.y)[(int64_t)(m0 + r) * p.ldy + n] = fw_cvt<T>(v + bias);
            }
    }
}

template <typename T, bool MIN, int GB, int MT, int NT, int WN, int WK, int MS>
static void q4_go(hipStream_t st, Q4P p) {
    constexpr bool CORR = MIN || std::is_same<T, fw_bf16>::value, F32 = std::is_same<T, float>::value;
    const int rows = std::min(p.m, MT * 16);
    // All of x in one stage where it fits 64 KiB of LDS; else two stages, of whole
    // rounds of the waves' turns in 80 KiB together (two blocks a CU) where one
    // fits, of as many turns as 144 KiB hold where not.
    const int turn = MS * (Q4X<T>::PARTS * rows * 256 + (CORR ? 256 * MT : 0)) + (F32 ? 64 * MT : 0);
    const int fixed = Q4X<T>::PARTS * rows * 16, join = WK > 1 ? WN * WK * MT * NT * 1024 : 0;
    const int all_turns = (p.k + 128 * MS - 1) / (128 * MS);
    int turns = all_turns, stages = 1;
    if (turns * (int64_t)turn + fixed > 65536) {
        stages = 2;
        turns = (40960 - fixed) / turn / WK * WK;
        if (turns < 1) turns = std::max(1, std::min(WK, (73728 - fixed) / turn));
    }
    p.chunk = turns * MS * 128;
    p.stage = turns * turn + fixed;
    p.lds = std::max(stages * p.stage, join);
    const Q4P all = p;
    for (int64_t at = 0; at < all.m; at += 65535 * 16 * MT) { // the grid's reach in rows
        p.m = (int)std::min<int64_t>(all.m - at, 65535 * 16 * MT);
        p.x = (const T *)all.x + at * all.ldx;
        p.y = (T *)all.y + at * all.ldy;
        const dim3 grid((unsigned)((p.n + 16 * NT * WN - 1) / (16 * NT * WN)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT)));
        hipLaunchKernelGGL((k_q4<T, MIN, GB, MT, NT, WN, WK, MS>), grid, dim3(64 * WN * WK), p.lds, st, p);
    }
}

// Which form runs.  x is staged once a block, so many outputs and rows a block
// save staging and unpacking; few spread a small product over the chip, the waves
// of a block then sharing outputs and taking turns of the inputs.  Longer turns
// carry fewer scale loads and waits but leave more idle at the end of short rows.
// Measured on both sides, us, the form that runs / the next best of the others:
//   1..16 rows, up to 640 tiles of 16 outputs: 1 x 5120 x 1280 5.2 / 7.9
//     k < 2048, from 2048 tiles on 16 waves a block: 10 x 51866 x 1280 (f32) 16.8 / 18.9,
//     1 x 51866 x 1280 13.0 / 13.4; less, 8 waves: 1 x 12288 x 1280 8.3 / 11.3
//     up to 1280 tiles: 8 x 14336 x 4096 14.2 / 20.0; above: 16 x 28672 x 8192 37 / 43
//   more, by how many blocks of 64 rows x 256 outputs, 32 x 128 or 32 x 64 there are,
//     else of 16 x 64, 16 x 32 or 16 x 16:
//     1500 x 5120 x 1280 58 / 71 and 700 x 5120 x 1280 28 / 31;
//     128 x 8192 x 8192 (groups of 128) 49 / 54, 440 x 1280 x 5120 (f32) 62 / 75, 128 x 5120 x 1280 13 / 15;
//     64 x 5120 x 5120 25.8 / 27.3 (but 200 x 1280 x 5120 in f32, whose staging is twice the work, 47 / 40);
//     24 x 5120 x 5120 17 / 19, 32 x 5120 x 1280 (f32) 10 / 13; 90 x 1280 x 1280 (f32) 9.2 / 9.9;
//     24 x 1280 x 5120 (f32) 21 / 23, 20 x 1280 x 1280 5.9 / 6.4
//   groups of 32: turns of 128 inputs, 256 x 5120 x 5120 57 / 60 with 256; longer groups
//     (fewer scales in registers): 256, 64 x 14336 x 4096 28 / 34 with 128.
template <typename T, bool MIN, int GB>
static void q4_rows(hipStream_t st, const Q4P &p) {
    constexpr int MS = GB == 1 ? 1 : 2;
    const int64_t tiles = (p.n + 15) / 16, mt = (p.m + 15) / 16;
    if (mt == 1 && tiles > 640) {
        if (p.k < 2048 && tiles >= 2048) q4_go<T, MIN, GB, 1, 1, 16, 1, 1>(st, p);
        else if (p.k < 2048) q4_go<T, MIN, GB, 1, 1, 8, 1, 2>(st, p);
        else if (tiles <= 1280) q4_go<T, MIN, GB, 1, 1, 4, 2, 4>(st, p);
        else q4_go<T, MIN, GB, 1, 1, 8, 1, 4>(st, p);
    } else if (mt > 1 && (tiles + 15) / 16 * ((mt + 3) / 4) >= 216) q4_go<T, MIN, GB, 4, 2, 8, 1, 1>(st, p);
    else if (mt > 1 && (tiles + 7) / 8 * ((mt + 1) / 2) >= 140) q4_go<T, MIN, GB, 2, 1, 8, 1, MS>(st, p);
    else if (mt > 1 && (tiles + 3) / 4 * ((mt + 1) / 2) >= 140 * Q4X<T>::PARTS) q4_go<T, MIN, GB, 2, 1, 4, 2, MS>(st, p);
    else if (mt > 1 && (tiles + 3) / 4 * mt >= 150) q4_go<T, MIN, GB, 1, 1, 4, 2, 1>(st, p);
    else if (mt > 1 && (tiles + 1) / 2 * mt >= 160) q4_go<T, MIN, GB, 1, 1, 2, 4, 1>(st, p);
    else q4_go<T, MIN, GB, 1, 1, 1, 8, 1>(st, p);
}
template <typename T>
static void q4_type(hipStream_t st, const Q4P &p) {
    if (p.group == 128) {
        if (p.minimum) q4_rows<T, true, 4>(st, p);
        else q4_rows<T, false, 4>(st, p);
    } else if (p.group == 64) {
        if (p.minimum) q4_rows<T, true, 2>(st, p);
        else q4_rows<T, false, 2>(st, p);
    } else {
        if (p.minimum) q4_rows<T, true, 1>(st, p);
        else q4_rows<T, false, 1>(st, p);
    }
}

extern "C" fwhip_status fwhip_q4_linear(fwhip_ctx *c, const fwhip_q4_linear_args *a) {
    if (!a) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: args is NULL");
    if (!fw_is_dtype(a->dtype) || (a->scale_dtype != FWHIP_T_F32 && a->scale_dtype != FWHIP_T_F16))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: unknown element type");
    if (a->group != 32 && a->group != 64 && a->group != 128)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_q4_linear: group must be 32, 64 or 128");
    if (a->m < 0 || a->n < 0 || a->k < a->group || a->k % a->group)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: m, n >= 0 and k a positive multiple of group");
    if (a->k > 1 << 24 || a->n > 1 << 29)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_q4_linear: k above 2^24 or n above 2^29");
    if (a->ldx < a->k || a->ldy < a->n) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: ldx < k or ldy < n");
    if (a->m && a->n) {
        if (!a->x || !a->q || !a->scale || !a->y) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: NULL argument");
        const int eb = fw_dtype_bytes(a->dtype), sb = fw_dtype_bytes(a->scale_dtype);
        if (!fw_aligned(a->q, 16)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: q must be 16-byte aligned");
        if (!fw_aligned(a->x, eb) || !fw_aligned(a->y, eb) || !fw_aligned(a->scale, sb) || !fw_aligned(a->minimum, sb) ||
            !fw_aligned(a->bias, 4))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: an address is not a multiple of its element's size");
        if (fw_rows_overlap(a->y, a->ldy, a->n, a->x, a->ldx, a->k, a->m, eb))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: y must not overlap x");
    }
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: NULL ctx");
    if (a->m == 0 || a->n == 0) return FWHIP_OK;
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_q4_linear: hipSetDevice failed");
    const int eb = fw_dtype_bytes(a->dtype), vb = 4 * eb;
    const int vec = fw_aligned(a->x, vb) && (a->m == 1 || a->ldx * eb % vb == 0);
    const int pair = fw_aligned(a->scale, 8) && fw_aligned(a->minimum, 8) && a->k / a->group % 4 == 0;
    const Q4P p = {a->m, a->n, a->k, a->group, a->ldx, a->ldy, a->x, a->q, a->scale, a->minimum, a->bias, a->y,
                   a->scale_dtype == FWHIP_T_F32, vec, pair, 0, 0, 0};
    if (a->dtype == FWHIP_T_F32) q4_type<float>(c->stream, p);
    else if (a->dtype == FWHIP_T_F16) q4_type<fw_f16>(c->stream, p);
    else q4_type<fw_bf16>(c->stream, p);
    return fw_launched("fwhip_q4_linear");
}

// ---------------------------------------------------------------------------
// A ggml payload as planes: one thread per 32 weights.
//   q4_0  f16 d, 16 bytes: byte j holds weights j and j + 16 (already the planes' order)
//   q4_1  f16 d, f16 m, 16 bytes
//   q4_k  f16 d, f16 dmin, 8 six-bit scales and minimums in 12 bytes, 128 bytes of
//         codes: of each 64 weights, byte t holds weights t and t + 32
__device__ __forceinline__ uint16_t ld16(const uint8_t *b) { return *(const uint16_t *)b; }

template <int T>
__global__ void __launch_bounds__(256) k_q4_planes(const uint8_t *raw, int64_t nb, uint8_t *q, void *scale, void *minimum) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= nb) return;
    uint8_t o[16];
    if constexpr (T != FWHIP_GGML_Q4_K) {
        constexpr int HEAD = T == FWHIP_GGML_Q4_1 ? 4 : 2;
        const uint8_t *b = raw + i * (16 + HEAD);
        ((uint16_t *)scale)[i] = ld16(b);
        if constexpr (T == FWHIP_GGML_Q4_1) ((uint16_t *)minimum)[i] = ld16(b + 2);
        for (int j = 0; j < 16; j++) o[j] = b[HEAD + j];
    } else {
        const uint8_t *b = raw + (i >> 3) * 144, *sc = b + 4;
        const int k = (int)(i & 7);
        int s, mn; // get_scale_min_k4 (ggml.rs:100-115)
        if (k < 4) {
            s = sc[k] & 63;
            mn = sc[k + 4] & 63;
        } else {
            s = (sc[k + 4] & 15) | ((sc[k - 4] >> 6) << 4);
            mn = (sc[k + 4] >> 4) | ((sc[k] >> 6) << 4);
        }
        ((float *)scale)[i] = fw_to_f32(fw_f16{ld16(b)}) * (float)s;
        ((float *)minimum)[i] = -(fw_to_f32(fw_f16{ld16(b + 2)}) * (float)mn);
        const uint8_t *c = b + 16 + 32 * (k >> 1);
        const int sh = 4 * (k & 1);
        for (int j = 0; j < 16; j++) o[j] = (uint8_t)(((c[j] >> sh) & 15) | (((c[j + 16] >> sh) & 15) << 4));
    }
    for (int j = 0; j < 16; j++) q[i * 16 + j] = o[j];
}

extern "C" fwhip_status fwhip_q4_planes(fwhip_ctx *c, int32_t ggml_dtype, const void *raw, uint64_t raw_bytes,
                                        int32_t rows, int32_t k, uint8_t *q, void *scale, void *minimum) {
    if (ggml_dtype != FWHIP_GGML_Q4_0 && ggml_dtype != FWHIP_GGML_Q4_1 && ggml_dtype != FWHIP_GGML_Q4_K)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_q4_planes: q4_0, q4_1 and q4_k payloads only");
    const int per = ggml_dtype == FWHIP_GGML_Q4_K ? 256 : 32;
    const int bytes = ggml_dtype == FWHIP_GGML_Q4_K ? 144 : ggml_dtype == FWHIP_GGML_Q4_1 ? 20 : 18;
    if (rows < 0 || k < per || k % per) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: rows >= 0 and k a positive multiple of the type's block");
    const int64_t nb = (int64_t)rows * (k / 32);
    if (raw_bytes != (uint64_t)rows * (uint64_t)(k / per) * (uint64_t)bytes)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: raw_bytes is not the payload's length");
    if (nb > (1ll << 39) / 256) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: too many weights");
    if (rows && (!raw || !q || !scale)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: NULL argument");
    if ((ggml_dtype == FWHIP_GGML_Q4_0) != (minimum == nullptr) && rows)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: q4_0 has no minimums, q4_1 and q4_k have");
    if (!fw_aligned(raw, 4) || !fw_aligned(q, 16) || !fw_aligned(scale, 16) || !fw_aligned(minimum, 16))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: raw must be 4-byte and the planes 16-byte aligned");
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_planes: NULL ctx");
    if (!rows) return FWHIP_OK;
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_q4_planes: hipSetDevice failed");
    const dim3 grid((unsigned)((nb + 255) / 256));
    const uint8_t *b = (const uint8_t *)raw;
    if (ggml_dtype == FWHIP_GGML_Q4_0) hipLaunchKernelGGL((k_q4_planes<FWHIP_GGML_Q4_0>), grid, dim3(256), 0, c->stream, b, nb, q, scale, minimum);
    else if (ggml_dtype == FWHIP_GGML_Q4_1) hipLaunchKernelGGL((k_q4_planes<FWHIP_GGML_Q4_1>), grid, dim3(256), 0, c->stream, b, nb, q, scale, minimum);
    else hipLaunchKernelGGL((k_q4_planes<FWHIP_GGML_Q4_K>), grid, dim3(256), 0, c->stream, b, nb, q, scale, minimum);
    return fw_launched("fwhip_q4_planes");
}
