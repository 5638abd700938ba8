// tree_attn.hip — attention of drafted trees (or causal chains of new tokens)
// over a paged K/V cache (fwhip_tree_attn).
//
// out_i = sum_j softmax_j(s q_i.k_j) v_j over the keys row i sees: the request's
// cached tokens, and those of its new tokens that the mask row names.  One pass
// over the keys with a running maximum m and sum l:
//   m' = max(m, max_j z_j),  l' = l e^(m-m') + sum_j e^(z_j-m'),  o' likewise.
#include <algorithm>

#include "fw_device.h"
#include "fw_paged.h"
#include "fw_serve.h"

struct TreeP {
    int n_req, n_rows, heads, kv_heads, n_pages, width, max_new, max_len, words;
    float scale;
    FwDiv page;
    int64_t table_stride, q_row, q_head, out_row, out_head, page_stride, token_stride, head_stride;
    const void *q, *kc, *vc;
    const int32_t *table, *len, *row_start;
    const uint64_t *mask;
    void *out;
};

// One wave per (row, head): a lane per key for the scores, a lane per output
// feature (D / 64 of them) for the sum.
template <typename T, int D>
__global__ void __launch_bounds__(64) k_tree_attn(TreeP p) {
    __shared__ float sq[D], sp[64];
    __shared__ int64_t sat[64];
    const int lane = threadIdx.x, h = blockIdx.y, i = blockIdx.x;
    const int r = blockIdx.z, kvh = h / (p.heads / p.kv_heads);
    const int row0 = min(max(p.row_start[r], 0), p.n_rows), row1 = min(p.row_start[r + 1], p.n_rows);
    const int n = row1 - row0, len = p.len[r];
    // rows of this request past max_new are marked too
    for (int row = row0 + i; row < row1; row += gridDim.x) {
        T *out = (T *)p.out + (int64_t)row * p.out_row + (int64_t)h * p.out_head;
        if (len < 0 || n > p.max_new || (int64_t)len + n > p.max_len) {
            for (int e = lane; e < D; e += 64) out[e] = fw_cvt<T>(__builtin_nanf(""));
            continue;
        }
        const int me = row - row0;
        __syncthreads();
        for (int e = lane; e < D; e += 64)
            sq[e] = fw_to_f32(((const T *)p.q)[(int64_t)row * p.q_row + (int64_t)h * p.q_head + e]);
        float m = -INFINITY, l = 0.0f, o[D / 64] = {};
        bool any = false;
        __syncthreads();
        for (int j0 = 0; j0 < len + n; j0 += 64) {
            const int j = j0 + lane;
            bool sees = j < len + n;
            if (sees && j >= len) {
                const int t = j - len;
                sees = p.mask ? (p.mask[(int64_t)row * p.words + (t >> 6)] >> (t & 63)) & 1 : t <= me;
            }
            float z = -INFINITY;
            int64_t at = 0;
            if (sees) {
                const uint32_t pi = fw_div((uint32_t)j, p.page);
                const int id = p.table[(int64_t)r * p.table_stride + pi];
                if (id < 0 || id >= p.n_pages) {
                    z = __builtin_nanf("");
                    at = -1;
                } else {
                    at = id * p.page_stride + (j - pi * p.page.d) * p.token_stride + kvh * p.head_stride;
                    const T *k = (const T *)p.kc + at;
                    z = 0.0f;
                    for (int e = 0; e < D; e++) z = fmaf(sq[e], fw_to_f32(k[e]), z);
                    z *= p.scale;
                }
            }
            if (!__any(sees)) continue;
            any = true;
            const float mn = fmaxf(m, fw_wave_max(z)); // NaN scores come back in e^(z - m)
            const float base = mn == -INFINITY ? 0.0f : mn;
            const float e = sees ? expf(z - base) : 0.0f, f = expf(m - base);
            l = l * f + fw_wave_sum(e);
            m = mn;
            sp[lane] = e;
            sat[lane] = sees ? at : -2;
            __syncthreads();
            for (int x = 0; x < D / 64; x++) {
                float acc = o[x] * f;
                for (int t = 0; t < 64; t++) {
                    if (sat[t] < -1) continue;
                    acc = fmaf(sp[t], sat[t] < 0 ? 0.0f : fw_to_f32(((const T *)p.vc)[sat[t] + x * 64 + lane]), acc);
                }
                o[x] = acc;
            }
            __syncthreads();
        }
        for (int x = 0; x < D / 64; x++) out[x * 64 + lane] = fw_cvt<T>(any ? o[x] / l : 0.0f);
    }
}

template <typename T, int D>
static void tree_launch(hipStream_t st, const TreeP &p) {
    hipLaunchKernelGGL((k_tree_attn<T, D>), dim3((unsigned)std::min(p.max_new, 65535), p.heads, p.n_req), dim3(64), 0,
                       st, p);
}
template <typename T>
static void tree_dim(hipStream_t st, int d, const TreeP &p) {
    if (d == 64) tree_launch<T, 64>(st, p);
    else tree_launch<T, 128>(st, p);
}

extern "C" fwhip_status fwhip_tree_attn_workspace(int32_t n_req, int32_t n_heads, int32_t n_kv_heads, int32_t head_dim,
                                                  int32_t max_new, int32_t max_len, uint64_t *bytes) {
    if (!bytes) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn_workspace: bytes is NULL");
    if (n_req < 0 || n_heads < 1 || n_kv_heads < 1 || n_heads % n_kv_heads || max_new < 0 || max_len < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn_workspace: bad size");
    if (head_dim != 64 && head_dim != 128)
        return fw_fail(FWHIP_ERR_UNSUPPORTED, "fwhip_tree_attn_workspace: head_dim must be 64 or 128");
    *bytes = 0;
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
        const int eb = fw_dtype_bytes(a->dtype);
        if (!fw_aligned(a->q, 16) || !fw_aligned(a->k_cache, 16) || !fw_aligned(a->v_cache, 16) || !fw_aligned(a->out, 16))
            return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: q, the caches and out must be 16-byte aligned");
        for (int k = 1; k < 8; k++)
            if (strides[k] * eb % 16)
                return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: strides must be multiples of 16 bytes");
        if (a->out == a->q) return fw_fail(FWHIP_ERR_INVALID, "fwhip_tree_attn: out must not be q");
    }
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
    p.page_stride = a->page_stride;
    p.token_stride = a->token_stride;
    p.head_stride = a->head_stride;
    p.q = a->q;
    p.kc = a->k_cache;
    p.vc = a->v_cache;
    p.table = a->table;
    p.len = a->len;
    p.row_start = a->row_start;
    p.mask = a->mask;
    p.out = a->out;
    if (a->dtype == FWHIP_T_F32) tree_dim<float>(c->stream, a->head_dim, p);
    else if (a->dtype == FWHIP_T_F16) tree_dim<fw_f16>(c->stream, a->head_dim, p);
    else tree_dim<fw_bf16>(c->stream, a->head_dim, p);
    return fw_launched("fwhip_tree_attn");
}
