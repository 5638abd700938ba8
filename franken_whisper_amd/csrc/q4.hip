// q4.hip — linears with 4-bit weights and group scales (fwhip_q4_linear), and
// the planes they read from a ggml payload (fwhip_q4_planes).
//
// y[m][n] = sum_g d[n][g] (sum_{k in g} x[m][k] c[n][k]) + lo[n][g] (sum_{k in g} x[m][k]) + b[n]
// with codes c in 0..15 (lo = the minimum) or c - 8 (no minimum): the group's
// inner sums need whole-number codes only, and the scales enter once a group.
#include <algorithm>

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
};

// One wave per output: lanes over the row's 32-weight blocks.
template <typename T, typename S, bool MIN>
__global__ void __launch_bounds__(256) k_q4_linear(Q4P p) {
    const int lane = threadIdx.x & 63;
    const int64_t at = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (at >= (int64_t)p.m * p.n) return;
    const int row = (int)(at / p.n), n = (int)(at % p.n);
    const T *x = (const T *)p.x + row * p.ldx;
    float acc = 0.0f;
    for (int b = lane; b < p.k / 32; b += 64) {
        const uint4 w = *(const uint4 *)(p.q + (int64_t)n * (p.k / 2) + b * 16);
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
        float dot = 0.0f, sum = 0.0f;
        for (int j = 0; j < 16; j++) {
            const uint32_t byte = u[j >> 2] >> (8 * (j & 3)) & 255;
            const float a = fw_to_f32(x[b * 32 + j]), c = fw_to_f32(x[b * 32 + 16 + j]);
            dot = fmaf(a, (float)(byte & 15) - (MIN ? 0.0f : 8.0f), dot);
            dot = fmaf(c, (float)(byte >> 4) - (MIN ? 0.0f : 8.0f), dot);
            sum += a + c;
        }
        const int64_t g = (int64_t)n * (p.k / p.group) + b * 32 / p.group;
        acc = fmaf(fw_to_f32(((const S *)p.scale)[g]), dot, acc);
        if (MIN) acc = fmaf(fw_to_f32(((const S *)p.minimum)[g]), sum, acc);
    }
    acc = fw_wave_sum(acc);
    if (lane == 0) ((T *)p.y)[row * p.ldy + n] = fw_cvt<T>(p.bias ? acc + p.bias[n] : acc);
}

template <typename T, typename S>
static void q4_launch(hipStream_t st, const Q4P &p) {
    const unsigned blocks = (unsigned)(((int64_t)p.m * p.n + 3) / 4);
    if (p.minimum) hipLaunchKernelGGL((k_q4_linear<T, S, true>), dim3(blocks), dim3(256), 0, st, p);
    else hipLaunchKernelGGL((k_q4_linear<T, S, false>), dim3(blocks), dim3(256), 0, st, p);
}
template <typename T>
static void q4_scale(hipStream_t st, int dtype, const Q4P &p) {
    if (dtype == FWHIP_T_F32) q4_launch<T, float>(st, p);
    else q4_launch<T, fw_f16>(st, p);
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
    const Q4P p = {a->m, a->n, a->k, a->group, a->ldx, a->ldy, a->x, a->q, a->scale, a->minimum, a->bias, a->y};
    if (a->dtype == FWHIP_T_F32) q4_scale<float>(c->stream, a->scale_dtype, p);
    else if (a->dtype == FWHIP_T_F16) q4_scale<fw_f16>(c->stream, a->scale_dtype, p);
    else q4_scale<fw_bf16>(c->stream, a->scale_dtype, p);
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
