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
    int scale32, vec, shift; // planes of f32; x rows 16-byte (f32) or 8-byte aligned; log2 of the group's blocks
    int chunk, lds;          // inputs staged at a time; bytes of LDS
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

// Eight codes as operands of a product, in the order q4_unit gives the inputs.
// f16: a code in the low bits of 1024 (or, four bits up, of 64) is that number
// plus the code; what is too much is taken off again, exactly, and with it the
// 8 of weights without minimums.
template <bool MIN>
__device__ __forceinline__ u4 q4_codes_f16(uint32_t w) {
    const uint32_t v = w >> 8;
    const h2 lo = MIN ? h2{(_Float16)1024, (_Float16)1024} : h2{(_Float16)1032, (_Float16)1032};
    const h2 hi = MIN ? h2{(_Float16)64, (_Float16)64} : h2{(_Float16)72, (_Float16)72};
    u4 r;
    r[0] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (w & 0x000f000fu) | 0x64006400u) - lo);
    r[1] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (w & 0x00f000f0u) | 0x54005400u) - hi);
    r[2] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (v & 0x000f000fu) | 0x64006400u) - lo);
    r[3] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(h2, (v & 0x00f000f0u) | 0x54005400u) - hi);
    return r;
}
// bf16: 128 + code; there is no packed bf16 subtraction, so the 128 (and the 8)
// leave with the sums of the inputs (CORR below).  That costs five bits of the
// f32 sum, 2^-19 of the result against the 2^-9 of its rounding.
__device__ __forceinline__ u4 q4_codes_bf16(uint32_t w) {
    u4 r;
#pragma unroll
    for (int i = 0; i < 4; i++) r[i] = (w >> (4 * i) & 0x000f000fu) | 0x43004300u;
    return r;
}

// x in LDS, as the products read it: per row KC inputs of 16 bits in units of 8,
// the unit (block, c) holding inputs 4 c + 0, 2, 16, 18, 1, 3, 17, 19 of its
// block.  f16 and bf16 as they are; f32 as two f16 parts of x / s, where s is
// the power of two that takes the largest |x| of the row's 128 to 2^14..2^15:
// hi + lo is within 2^-22 of x down to 2^-28 of that largest.
template <typename T>
struct Q4X {
    static constexpr int PARTS = std::is_same<T, float>::value ? 2 : 1;
};

template <typename T>
__device__ __forceinline__ void q4_load4(const T *at, bool vec, int left, float (&v)[4]) {
    if (vec && left >= 4) {
        if constexpr (sizeof(T) == 4) {
            const f4 a = *(const f4 *)at;
#pragma unroll
            for (int i = 0; i < 4; i++) v[i] = a[i];
        } else {
            const uint2 a = *(const uint2 *)at;
            v[0] = fw_to_f32(T{(uint16_t)a.x});
            v[1] = fw_to_f32(T{(uint16_t)(a.x >> 16)});
            v[2] = fw_to_f32(T{(uint16_t)a.y});
            v[3] = fw_to_f32(T{(uint16_t)(a.y >> 16)});
        }
    } else {
#pragma unroll
        for (int i = 0; i < 4; i++) v[i] = i < left ? fw_to_f32(at[i]) : 0.0f;
    }
}
template <typename T>
__device__ __forceinline__ uint32_t q4_pair(float a, float b) {
    typedef typename std::conditional<std::is_same<T, float>::value, fw_f16, T>::type H;
    return fw_cvt<H>(a).b | (uint32_t)fw_cvt<H>(b).b << 16;
}

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
// taking the steps of the same outputs in turn.  x is staged in LDS for up to
// `chunk` inputs at a time, its block sums beside it where weights have a
// minimum; each wave streams its weights straight to registers, U steps ahead.
// GB = 4: one scale a step (groups of 128), else one a block.
template <typename T, bool MIN, int GB, int MT, int NT, int WN, int WK, int U>
__global__ void __launch_bounds__(64 * WN * WK) k_q4(Q4P p) {
    constexpr bool BF = std::is_same<T, fw_bf16>::value, F32 = std::is_same<T, float>::value, CORR = MIN || BF;
    constexpr int PARTS = Q4X<T>::PARTS, NTH = 64 * WN * WK;
    extern __shared__ __attribute__((aligned(16))) char lds[];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, lr = lane & 15, c = lane >> 4;
    const int wn = wave / WK, wk = wave % WK;
    const int m0 = blockIdx.y * MT * 16, rows = min(MT * 16, p.m - m0);
    const int n0 = (blockIdx.x * WN + wn) * NT * 16;
    const int steps = (p.k + 127) / 128, csteps = p.chunk / 128;
    const int xrow = p.chunk * 2 + 16; // bytes of a row: rows 4 banks apart
    const int plane = rows * xrow;
    int *odd = (int *)lds;                                    // [MT * 16]: rows with a value that is not finite
    char *xt = lds + MT * 64;                                 // x: [part][row][xrow]
    float *sums = (float *)(xt + PARTS * plane);              // CORR: [step][block][MT * 16]
    float *scal = sums + (CORR ? csteps * 4 * MT * 16 : 0);   // f32: [step][MT * 16]

    f4 acc[MT][NT], mid[MT][NT];
#pragma unroll
    for (int x = 0; x < MT; x++)
#pragma unroll
        for (int y = 0; y < NT; y++) acc[x][y] = f4{};
    if (CORR)
        for (int i = threadIdx.x; i < MT * 16; i += NTH) odd[i] = 0;

    int nrow[NT];
#pragma unroll
    for (int y = 0; y < NT; y++) nrow[y] = min(n0 + y * 16 + lr, p.n - 1); // the last again behind the end
    u4 wq[U][NT];
    float sc[U][NT], mn[U][NT];
    const int groups = p.k / p.group;
    auto load = [&](int s0, int to) { // steps s0, s0 + WK, ... below `to`
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int s = s0 + u * WK, blk = s * 4 + c;
            const bool in = s < to && blk * 32 < p.k;
            const int g = blk >> p.shift;
#pragma unroll
            for (int y = 0; y < NT; y++) {
                wq[u][y] = u4{};
                sc[u][y] = mn[u][y] = 0.0f;
                if (!in) continue;
                wq[u][y] = *(const u4 *)(p.q + (int64_t)nrow[y] * (p.k / 2) + blk * 16);
                const int64_t at = (int64_t)nrow[y] * groups + g;
                if (p.scale32) {
                    sc[u][y] = ((const float *)p.scale)[at];
                    if (MIN) mn[u][y] = ((const float *)p.minimum)[at];
                } else {
                    sc[u][y] = fw_to_f32(((const fw_f16 *)p.scale)[at]);
                    if (MIN) mn[u][y] = fw_to_f32(((const fw_f16 *)p.minimum)[at]);
                }
            }
        }
    };

    for (int s0 = 0; s0 < steps; s0 += csteps) {
        const int to = min(steps, s0 + csteps);
        load(s0 + wk, to);
        if (s0) __syncthreads();
        // stage x: a unit of 8 inputs per lane, 16 lanes a row's step
        for (int it = threadIdx.x >> 4; it < rows * (to - s0); it += NTH / 16) {
            const int r = it % rows, st = it / rows, u = lane & 15; // unit u: block u / 4, part u % 4
            const int k = (s0 + st) * 128 + (u >> 2) * 32 + (u & 3) * 4;
            const T *at = (const T *)p.x + (int64_t)(m0 + r) * p.ldx + k;
            float e[4], h[4];
            const bool in = (k & ~31) < p.k;
            q4_load4<T>(at, p.vec, in ? 4 : 0, e);
            q4_load4<T>(at + 16, p.vec, in ? 4 : 0, h);
            if constexpr (F32) {
                float mx = 0.0f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    mx = fmaxf(mx, fabsf(e[i]) < INFINITY ? fabsf(e[i]) : 0.0f);
                    mx = fmaxf(mx, fabsf(h[i]) < INFINITY ? fabsf(h[i]) : 0.0f);
                }
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_XOR1>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_XOR2>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_HALF_MIRROR>(mx));
                mx = fmaxf(mx, fw_dpp_f32<FW_DPP_MIRROR>(mx));
                // mx = 1.f x 2^(ex - 127); x is scaled by 2^(14 - (ex - 127)), in two factors that are normal numbers
                const int ex = max((int)(__float_as_uint(mx) >> 23), 1), up = 141 - ex;
                const float f1 = __uint_as_float((uint32_t)(127 + up / 2) << 23), f2 = __uint_as_float((uint32_t)(127 + up - up / 2) << 23);
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[i] = e[i] * f1 * f2;
                    h[i] = h[i] * f1 * f2;
                }
                // up is -113..140: the inverse 2^-up as a number, subnormal ones included
                if (u == 0) scal[st * MT * 16 + r] = __builtin_ldexpf(1.0f, -up);
            }
            u4 v = {q4_pair<T>(e[0], e[2]), q4_pair<T>(h[0], h[2]), q4_pair<T>(e[1], e[3]), q4_pair<T>(h[1], h[3])};
            char *to_lds = xt + r * xrow + st * 256 + u * 16;
            *(u4 *)to_lds = v;
            if constexpr (F32) {
                float el[4], hl[4];
#pragma unroll
                for (int i = 0; i < 4; i++) { // parts of values that are not finite: nothing more
                    el[i] = fabsf(e[i]) < INFINITY ? e[i] - (float)(_Float16)e[i] : 0.0f;
                    hl[i] = fabsf(h[i]) < INFINITY ? h[i] - (float)(_Float16)h[i] : 0.0f;
                }
                v = u4{q4_pair<T>(el[0], el[2]), q4_pair<T>(hl[0], hl[2]), q4_pair<T>(el[1], el[3]), q4_pair<T>(hl[1], hl[3])};
                *(u4 *)(to_lds + plane) = v;
            }
            if constexpr (CORR) {
                float t = ((e[0] + e[1]) + (e[2] + e[3])) + ((h[0] + h[1]) + (h[2] + h[3]));
                t = t + fw_dpp_f32<FW_DPP_XOR1>(t);
                t = t + fw_dpp_f32<FW_DPP_XOR2>(t);
                if ((u & 3) == 0) sums[(st * 4 + (u >> 2)) * MT * 16 + r] = t;
                if (!(fabsf(t) < INFINITY)) odd[r] = 1;
            }
        }
        __syncthreads();

        for (int s = s0 + wk; s < to; s += U * WK) {
            u4 w[U][NT];
            float d[U][NT], e[U][NT];
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int y = 0; y < NT; y++) {
                    w[u][y] = wq[u][y];
                    d[u][y] = sc[u][y];
                    e[u][y] = MIN ? (BF ? fmaf(-128.0f, sc[u][y], mn[u][y]) : mn[u][y]) : -136.0f * sc[u][y];
                }
            if (s + U * WK < to) load(s + U * WK, to);
#pragma unroll
            for (int u = 0; u < U; u++) {
                const int st = s + u * WK - s0;
                if (st >= to - s0) break;
                f4 dq[NT];
#pragma unroll
                for (int y = 0; y < NT; y++) {
                    q4_exchange(w[u][y]);
                    if constexpr (GB == 1) dq[y] = q4_quarters(d[u][y]);
                }
                const char *xs = xt + st * 256 + c * 16;
#pragma unroll
                for (int x = 0; x < MT; x++)
#pragma unroll
                    for (int y = 0; y < NT; y++) mid[x][y] = f4{};
                if constexpr (CORR) {
                    // the inputs' block sums times what every code is off by, four blocks in one product
#pragma unroll
                    for (int x = 0; x < MT; x++) {
                        const float t = sums[(st * 4 + c) * MT * 16 + x * 16 + lr];
#pragma unroll
                        for (int y = 0; y < NT; y++)
                            (F32 ? mid[x][y] : acc[x][y]) =
                                __builtin_amdgcn_mfma_f32_16x16x4f32(t, e[u][y], F32 ? mid[x][y] : acc[x][y], 0, 0, 0);
                    }
                }
                f4 dot[MT][NT];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    u4 b[NT];
#pragma unroll
                    for (int y = 0; y < NT; y++) b[y] = BF ? q4_codes_bf16(w[u][y][i]) : q4_codes_f16<MIN>(w[u][y][i]);
#pragma unroll
                    for (int x = 0; x < MT; x++) {
                        const int r = min(x * 16 + lr, rows - 1);
                        const u4 a = *(const u4 *)(xs + r * xrow + i * 64);
                        u4 al;
                        if constexpr (F32) al = *(const u4 *)(xs + plane + r * xrow + i * 64);
#pragma unroll
                        for (int y = 0; y < NT; y++) {
                            f4 z = GB == 4 && i ? dot[x][y] : f4{};
                            if constexpr (BF)
                                z = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b8, a), __builtin_bit_cast(b8, b[y]), z, 0, 0, 0);
                            else {
                                if constexpr (F32)
                                    z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, al), __builtin_bit_cast(h8, b[y]), z, 0, 0, 0);
                                z = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h8, a), __builtin_bit_cast(h8, b[y]), z, 0, 0, 0);
                            }
                            dot[x][y] = z;
                            if (GB == 1 || i == 3) {
                                const float f = GB == 1 ? dq[y][i] : d[u][y];
                                f4 &to_acc = F32 ? mid[x][y] : acc[x][y];
#pragma unroll
                                for (int j = 0; j < 4; j++) to_acc[j] = fmaf(f, z[j], to_acc[j]);
                            }
                        }
                    }
                }
                if constexpr (F32) {
#pragma unroll
                    for (int x = 0; x < MT; x++) {
                        const f4 f = *(const f4 *)(scal + st * MT * 16 + x * 16 + 4 * c);
#pragma unroll
                        for (int y = 0; y < NT; y++)
#pragma unroll
                            for (int j = 0; j < 4; j++)
                                acc[x][y][j] = fmaf(f[j], mid[x][y][j], acc[x][y][j]);
                    }
                }
            }
        }
    }

    // the waves that shared outputs add up, in order
    if constexpr (WK > 1) {
        __syncthreads();
        f4 *part = (f4 *)xt; // [wave][x][y][lane]
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
                // sums of inputs that are not finite do not come apart again: product by product
                if (CORR && odd[r]) v = q4_one<T, MIN>(p, m0 + r, n);
                ((T *)p.y)[(int64_t)(m0 + r) * p.ldy + n] = fw_cvt<T>(v + bias);
            }
    }
}

template <typename T, bool MIN, int GB, int MT, int NT, int WN, int WK, int U>
static void q4_go(hipStream_t st, Q4P p) {
    constexpr bool CORR = MIN || std::is_same<T, fw_bf16>::value, F32 = std::is_same<T, float>::value;
    const int rows = std::min(p.m, MT * 16);
    // as many inputs a stage as fit 64 KiB of LDS, a whole number of turns of the waves
    const int step = Q4X<T>::PARTS * rows * 256 + (CORR ? 256 * MT : 0) + (F32 ? 64 * MT : 0);
    const int fixed = Q4X<T>::PARTS * rows * 16 + 64 * MT, join = 64 * MT + (WK > 1 ? WN * WK * MT * NT * 1024 : 0);
    int steps = std::max(1, (65536 - fixed) / step);
    steps = std::min(steps, (p.k + 127) / 128);
    if (steps > WK) steps = steps / WK * WK;
    p.chunk = steps * 128;
    p.lds = std::max(steps * step + fixed, join);
    const Q4P all = p;
    for (int64_t at = 0; at < all.m; at += 65535 * 16 * MT) { // the grid's reach in rows
        p.m = (int)std::min<int64_t>(all.m - at, 65535 * 16 * MT);
        p.x = (const T *)all.x + at * all.ldx;
        p.y = (T *)all.y + at * all.ldy;
        const dim3 grid((unsigned)((p.n + 16 * NT * WN - 1) / (16 * NT * WN)), (unsigned)((p.m + 16 * MT - 1) / (16 * MT)));
        hipLaunchKernelGGL((k_q4<T, MIN, GB, MT, NT, WN, WK, U>), grid, dim3(64 * WN * WK), p.lds, st, p);
    }
}
template <typename T, bool MIN, int GB>
static void q4_rows(hipStream_t st, const Q4P &p) {
    const bool wide = p.n >= 16384;
    if (p.m <= 16) {
        if (wide) q4_go<T, MIN, GB, 1, 1, 4, 2, 2>(st, p);
        else q4_go<T, MIN, GB, 1, 1, 1, 8, 2>(st, p);
    } else if (p.m <= 32) q4_go<T, MIN, GB, 2, 1, 4, 1, 2>(st, p);
    else q4_go<T, MIN, GB, 4, 2, 4, 1, 1>(st, p);
}
template <typename T>
static void q4_type(hipStream_t st, const Q4P &p) {
    if (p.group == 128) {
        if (p.minimum) q4_rows<T, true, 4>(st, p);
        else q4_rows<T, false, 4>(st, p);
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
    if (a->ldx < a->k || a->ldy < a->n) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: ldx < k or ldy < n");
    if (a->m && a->n) {
        if (!a->x || !a->q || !a->scale || !a->y) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: NULL argument");
        const int eb = fw_dtype_bytes(a->dtype), sb = fw_dtype_bytes(a->scale_dtype);
        if (!fw_aligned(a->q, 16)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: q must be 16-byte aligned");
        if (!fw_aligned(a->x, eb) || !fw_aligned(a->y, eb) || !fw_aligned(a->scale, sb) || !fw_aligned(a->minimum, sb) ||
            !fw_aligned(a->bias, 4))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: an address is not a multiple of its element's size");
        if (fw_overlap(a->y, ((a->m - 1) * a->ldy + a->n) * eb, a->x, ((a->m - 1) * a->ldx + a->k) * eb) &&
            (a->ldx != a->ldy || a->x == a->y))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: y must not overlap x");
    }
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_q4_linear: NULL ctx");
    if (a->m == 0 || a->n == 0) return FWHIP_OK;
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_q4_linear: hipSetDevice failed");
    const int eb = fw_dtype_bytes(a->dtype), vb = 4 * eb;
    const int vec = fw_aligned(a->x, vb) && (a->m == 1 || a->ldx * eb % vb == 0);
    const Q4P p = {a->m, a->n, a->k, a->group, a->ldx, a->ldy, a->x, a->q, a->scale, a->minimum, a->bias, a->y,
                   a->scale_dtype == FWHIP_T_F32, vec, a->group == 32 ? 0 : a->group == 64 ? 1 : 2, 0, 0};
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
