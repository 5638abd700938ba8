// fw_serve.h — what the serving operators (paged.hip, tree_attn.hip, q4.hip)
// share: element types, argument checks, the device of a call.
#pragma once
#include "fw_internal.h"

// Storage types: the bits of a binary16 / bfloat16 number.
struct fw_f16 {
    uint16_t b;
};
struct fw_bf16 {
    uint16_t b;
};

__device__ __forceinline__ float fw_to_f32(float v) { return v; }
__device__ __forceinline__ float fw_to_f32(fw_f16 v) { return (float)__builtin_bit_cast(_Float16, v.b); }
__device__ __forceinline__ float fw_to_f32(fw_bf16 v) { return __uint_as_float((uint32_t)v.b << 16); }

// Rounding to nearest, ties to even; NaN stays NaN (quiet).
template <typename T>
__device__ __forceinline__ T fw_cvt(float f);
template <>
__device__ __forceinline__ float fw_cvt<float>(float f) {
    return f;
}
template <>
__device__ __forceinline__ fw_f16 fw_cvt<fw_f16>(float f) {
    return {__builtin_bit_cast(uint16_t, (_Float16)f)};
}
template <>
__device__ __forceinline__ fw_bf16 fw_cvt<fw_bf16>(float f) {
    return {__builtin_bit_cast(uint16_t, (__bf16)f)};
}

static inline bool fw_is_dtype(int32_t t) { return t >= FWHIP_T_F32 && t <= FWHIP_T_BF16; }
static inline int fw_dtype_bytes(int32_t t) { return t == FWHIP_T_F32 ? 4 : 2; }
static inline bool fw_aligned(const void *p, int64_t bytes) { return (uintptr_t)p % (uint64_t)bytes == 0; }
static inline bool fw_overlap(const void *a, int64_t na, const void *b, int64_t nb) {
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return na > 0 && nb > 0 && x < y + (uint64_t)nb && y < x + (uint64_t)na;
}

// Two arrays of `rows` rows of na and nb elements (of `bytes` bytes each): whether
// they share an element.  Columns of one wider array (equal strides) lie between
// each other and share none.
static inline bool fw_rows_overlap(const void *a, int64_t lda, int64_t na, const void *b, int64_t ldb, int64_t nb,
                                   int64_t rows, int bytes) {
    if (!fw_overlap(a, ((rows - 1) * lda + na) * bytes, b, ((rows - 1) * ldb + nb) * bytes)) return false;
    if (rows == 1 || lda != ldb || na > lda || nb > lda) return true;
    const int64_t row = lda * bytes, d = (((int64_t)((uintptr_t)b - (uintptr_t)a)) % row + row) % row; // b's columns begin d behind a's
    return d < na * bytes || row - d < nb * bytes;
}

// The context's device for the length of a call; the caller's comes back.
struct FwOnDevice {
    int before = -1;
    bool ok = true;
    explicit FwOnDevice(const fwhip_ctx *c) {
        int now = -1;
        if (hipGetDevice(&now) != hipSuccess) ok = false;
        else if (now != c->device) {
            ok = hipSetDevice(c->device) == hipSuccess;
            before = now;
        }
    }
    ~FwOnDevice() {
        if (before >= 0) (void)hipSetDevice(before);
    }
};

static inline fwhip_status fw_launched(const char *what) {
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fw_fail(FWHIP_ERR_GENERIC, std::string(what) + ": " + hipGetErrorString(e));
    return FWHIP_OK;
}
