// fw_paged.h — index arithmetic of the paged cache, shared by the kernels and
// by the host (the CPU tests compile this header alone).
#pragma once
#include <stdint.h>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define FWP_HD __host__ __device__ __forceinline__
#else
#define FWP_HD static inline
#endif

// Status bits of a request (fwhip_paged_plan_args.status).
#define FWP_NO_PAGES 1
#define FWP_BAD_LENGTH 2
#define FWP_BAD_PARENT 4

#define FWP_MASK_WORDS 4 // mask words a request's tree may have
#define FWP_MAX_NODES (64 * FWP_MASK_WORDS)

// n / d for n < 2^31 without a divide: multiply, add, shift (Granlund and
// Montgomery's round-up method: m = floor(2^32 (2^s - d) / d) + 1 with
// s = ceil(log2 d) gives q = (mulhi(n, m) + n) >> s exactly).
struct FwDiv {
    uint32_t d, m, s;
};
static inline struct FwDiv fw_div_make(uint32_t d) {
    struct FwDiv v;
    uint32_t s = 0;
    while (s < 32 && ((uint64_t)1 << s) < d) s++;
    v.d = d;
    v.s = s;
    v.m = (uint32_t)((((uint64_t)1 << 32) * ((((uint64_t)1 << s) - d))) / d + 1);
    return v;
}
FWP_HD uint32_t fw_div(uint32_t n, struct FwDiv v) {
    const uint32_t hi = (uint32_t)(((uint64_t)n * v.m) >> 32);
    return (hi + n) >> v.s;
}

// What one request asks of the plan, from what the device holds about it.
struct FwReq {
    int64_t rows; // its rows (n_new, 0 if negative)
    int64_t need; // pages it needs and its table row has room for
    int status;   // what already stands against it
};
FWP_HD struct FwReq fw_plan_req(int32_t len, int32_t n_new, int32_t held, int32_t width, struct FwDiv page) {
    struct FwReq r;
    r.status = 0;
    r.need = 0;
    r.rows = n_new > 0 ? n_new : 0;
    if (len < 0 || n_new < 0 || held < 0 || held > width || (int64_t)len + r.rows > 0x7fffffff - (int64_t)page.d) {
        r.status = FWP_BAD_LENGTH;
        return r;
    }
    // (len + rows + page - 1) stays below 2^31
    const int64_t want = (int64_t)fw_div((uint32_t)(len + r.rows + page.d - 1), page) - held;
    if (want > width - held) r.status = FWP_NO_PAGES;
    else if (want > 0) r.need = want;
    return r;
}

// The slot of a request's cached token t, -1 where its page is not in the table.
FWP_HD int64_t fw_slot(int32_t page_id, uint32_t t, uint32_t page_index, struct FwDiv page) {
    if (page_id < 0) return -1;
    return (int64_t)page_id * page.d + (t - page_index * page.d);
}
