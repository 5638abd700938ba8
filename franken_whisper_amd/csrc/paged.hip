// paged.hip — the step plan of a paged K/V cache and the cache's writes
// (fwhip_paged_plan, fwhip_paged_append).
#include <algorithm>

#include "fw_device.h"
#include "fw_paged.h"
#include "fw_serve.h"

// ---------------------------------------------------------------------------
// plan
//
// One launch: a request's place in the rows and in the free list is a prefix
// sum over the requests before it, and every block sums those itself (three
// ints a request from the caches) instead of waiting for another block.  Block
// (x, y) handles requests x * rpb .. + rpb - 1 one after another, and slice y
// of each request's rows and table columns.  10 requests: 5.6 us; 1,024 requests of 64
// drafted tokens with tables of 2,048 columns: 9.5 us, 1.9 TB/s (one block a request, the
// trees' six rounds of pointer jumping the longest chain).
struct PlanP {
    int n_req, width, n_rows, n_free, words, rpb;
    int quads; // table rows in 16-byte pieces
    FwDiv page;
    const int32_t *len, *n_new, *parents, *table, *held, *free_pages, *free_count;
    int32_t *table_out, *held_out, *count_out, *row_start, *row_req, *pos;
    int64_t *slot;
    uint64_t *mask;
    int32_t *status;
};

#define PLAN_T 256

// The ancestors of every node of one request: pointer jumping doubles the
// reach of each node's set a round (sets of the same size n_words per node).
__device__ static int plan_tree(const PlanP &p, int64_t row0, int n, int32_t len, uint64_t (*set)[FWP_MASK_WORDS],
                                int16_t *up, int *bad) {
    const int t = threadIdx.x; // one node per thread: n <= PLAN_T
    if (t == 0) *bad = 0;
    __syncthreads();
    if (t < n) {
        int par = p.parents[row0 + t];
        if (par < -1 || par >= t) {
            par = -1;
            *bad = 1;
        }
        up[t] = (int16_t)par;
        for (int w = 0; w < FWP_MASK_WORDS; w++) set[t][w] = (t >> 6) == w ? 1ull << (t & 63) : 0;
    }
    __syncthreads();
    for (int reach = 1; reach < n; reach *= 2) {
        uint64_t s[FWP_MASK_WORDS];
        int u = -1;
        if (t < n) {
            u = up[t];
            for (int w = 0; w < FWP_MASK_WORDS; w++) s[w] = set[t][w] | (u >= 0 ? set[u][w] : 0);
            u = u >= 0 ? up[u] : -1;
        }
        __syncthreads();
        if (t < n) {
            up[t] = (int16_t)u;
            for (int w = 0; w < FWP_MASK_WORDS; w++) set[t][w] = s[w];
        }
        __syncthreads();
    }
    if (t < n) {
        int depth = -1;
        for (int w = 0; w < FWP_MASK_WORDS; w++) {
            depth += __popcll(set[t][w]);
            if (w < p.words) p.mask[(row0 + t) * p.words + w] = set[t][w];
        }
        p.pos[row0 + t] = len + depth;
    }
    const int b = *bad;
    __syncthreads();
    return b;
}

__global__ void __launch_bounds__(PLAN_T) k_paged_plan(PlanP p) {
    __shared__ int64_t sh[PLAN_T / FW_WAVE];
    __shared__ uint64_t set[PLAN_T][FWP_MASK_WORDS];
    __shared__ int16_t up[PLAN_T];
    __shared__ int bad;
    const int t = threadIdx.x, r0 = blockIdx.x * p.rpb, r1 = min(p.n_req, r0 + p.rpb);
    const bool first = blockIdx.y == 0; // the slice that writes what a request has once
    const int64_t count = min(max(p.free_count[0], 0), p.n_free);

    int64_t rows = 0, pages = 0;
    for (int r = t; r < r0; r += PLAN_T) {
        const FwReq q = fw_plan_req(p.len[r], p.n_new[r], p.held[r], p.width, p.page);
        rows += q.rows;
        pages += q.need;
    }
    rows = fw_block_sum(rows, sh);
    pages = fw_block_sum(pages, sh);
    if (blockIdx.x == 0 && first && t == 0) {
        p.row_start[0] = 0;
        if (p.n_req == 0) p.count_out[0] = (int32_t)count;
    }
    for (int r = r0; r < r1; r++) {
        const int32_t len = p.len[r], held = p.held[r];
        const FwReq q = fw_plan_req(len, p.n_new[r], held, p.width, p.page);
        const int64_t end = pages + q.need;
        int status = q.status;
        if (q.need > 0 && end > count) status |= FWP_NO_PAGES;
        const int64_t row0 = min(rows, (int64_t)p.n_rows), row1 = min(rows + q.rows, (int64_t)p.n_rows);
        if (row1 - row0 < q.rows) status |= FWP_BAD_LENGTH;
        const bool ok = !(status & FWP_NO_PAGES) && !(q.status & FWP_BAD_LENGTH);
        const int take = ok ? (int)q.need : 0;
        const int n = (int)(row1 - row0);
        // pages are taken from the top of the free list
        const int32_t *fresh = p.free_pages + (count - 1 - pages);

        const int32_t *trow = p.table + (int64_t)r * p.width;
        int32_t *orow = p.table_out + (int64_t)r * p.width;
        if (p.table != p.table_out) {
            if (p.quads)
                for (int64_t c = blockIdx.y * PLAN_T + t; c < p.width / 4; c += gridDim.y * PLAN_T) {
                    int4 v = ((const int4 *)trow)[c];
                    if (take && 4 * c + 3 >= held && 4 * c < held + take) {
                        int e[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int i = 0; i < 4; i++)
                            if (4 * c + i >= held && 4 * c + i < held + take) e[i] = fresh[-(4 * c + i - held)];
                        v = make_int4(e[0], e[1], e[2], e[3]);
                    }
                    ((int4 *)orow)[c] = v;
                }
            else
                for (int64_t c = blockIdx.y * PLAN_T + t; c < p.width; c += gridDim.y * PLAN_T)
                    orow[c] = c >= held && c < held + take ? fresh[-(c - held)] : trow[c];
        } else
            for (int64_t c = blockIdx.y * PLAN_T + t; c < take; c += gridDim.y * PLAN_T) orow[held + c] = fresh[-c];
        const bool tree = p.words > 0;
        const bool fits = !tree || q.rows <= (int64_t)64 * p.words;
        for (int64_t i = blockIdx.y * PLAN_T + t; i < n; i += gridDim.y * PLAN_T) {
            const int64_t row = row0 + i;
            const uint32_t token = (uint32_t)len + (uint32_t)i;
            int64_t slot = -1;
            if (ok) {
                const uint32_t pi = fw_div(token, p.page);
                const int32_t id = (int)pi >= held ? fresh[-((int)pi - held)] : trow[pi];
                slot = fw_slot(id, token, pi, p.page);
            }
            p.slot[row] = slot;
            p.row_req[row] = r;
            if (!tree || !fits) p.pos[row] = (int32_t)token;
            if (tree && !fits)
                for (int w = 0; w < p.words; w++) p.mask[row * p.words + w] = 0;
        }
        if (tree && !fits) status |= FWP_BAD_PARENT;
        if (first && tree && fits && n > 0 && plan_tree(p, row0, n, len, set, up, &bad)) status |= FWP_BAD_PARENT;
        if (first && t == 0) {
            p.row_start[r + 1] = (int32_t)row1;
            p.held_out[r] = held + take;
            p.status[r] = status;
            // the first request past the free pages, or the last one, says what is left
            if (pages <= count && end > count) p.count_out[0] = (int32_t)(count - pages);
            else if (r == p.n_req - 1 && end <= count) p.count_out[0] = (int32_t)(count - end);
        }
        rows += q.rows;
        pages = end;
    }
}

extern "C" fwhip_status fwhip_paged_plan(fwhip_ctx *c, const fwhip_paged_plan_args *a) {
    if (!a) return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: args is NULL");
    if (a->n_req < 0 || a->width < 0 || a->n_rows < 0 || a->n_free < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: negative size");
    if (a->page_size < 1 || a->page_size > (1 << 24))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: page_size must be in 1..2^24");
    if (!a->row_start || !a->count_out || !a->free_count ||
        (a->n_req && (!a->len || !a->n_new || !a->held || !a->held_out || !a->status)) ||
        (a->n_req && a->width && (!a->table || !a->table_out)) || (a->n_rows && (!a->row_req || !a->pos || !a->slot)) ||
        (a->n_free && !a->free_pages))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: NULL argument");
    const bool tree = a->mask_words != 0;
    if (a->mask_words < 0 || a->mask_words > FWP_MASK_WORDS ||
        (tree ? a->n_rows && (!a->parents || !a->mask) : a->parents || a->mask))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: parents and mask go together, with mask_words in 1..4");
    for (const void *v : {(const void *)a->len, (const void *)a->n_new, (const void *)a->parents, (const void *)a->table,
                          (const void *)a->held, (const void *)a->free_pages, (const void *)a->free_count,
                          (const void *)a->table_out, (const void *)a->held_out, (const void *)a->count_out,
                          (const void *)a->row_start, (const void *)a->row_req, (const void *)a->pos, (const void *)a->status})
        if (!fw_aligned(v, 4)) return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: an address is not a multiple of its element's size");
    if (!fw_aligned(a->slot, 8) || !fw_aligned(a->mask, 8))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: an address is not a multiple of its element's size");
    // every block reads the lengths that other blocks' results would replace
    if (a->n_req && (fw_overlap(a->held_out, 4ll * a->n_req, a->held, 4ll * a->n_req) ||
                     fw_overlap(a->held_out, 4ll * a->n_req, a->len, 4ll * a->n_req) ||
                     fw_overlap(a->held_out, 4ll * a->n_req, a->n_new, 4ll * a->n_req)))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: held_out must not overlap len, n_new or held");
    if (fw_overlap(a->count_out, 4, a->free_count, 4))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: count_out must not be free_count");
    const int64_t tb = 4ll * a->n_req * a->width;
    if (a->table != a->table_out && fw_overlap(a->table_out, tb, a->table, tb))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: table_out must be table or lie apart from it");
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_plan: NULL ctx");
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_paged_plan: hipSetDevice failed");

    PlanP p;
    p.n_req = a->n_req;
    p.width = a->width;
    p.n_rows = a->n_rows;
    p.n_free = a->n_free;
    p.words = a->mask_words;
    p.page = fw_div_make((uint32_t)a->page_size);
    p.len = a->len;
    p.n_new = a->n_new;
    p.parents = a->parents;
    p.table = a->table;
    p.held = a->held;
    p.free_pages = a->free_pages;
    p.free_count = a->free_count;
    p.table_out = a->table_out;
    p.held_out = a->held_out;
    p.count_out = a->count_out;
    p.row_start = a->row_start;
    p.row_req = a->row_req;
    p.pos = a->pos;
    p.slot = a->slot;
    p.mask = a->mask;
    p.status = a->status;
    // Few requests with many rows or long tables (prompts): several blocks a
    // request, each with a slice.  Many requests: several a block, which bounds
    // how often the lengths before a block are summed.
    p.quads = a->width % 4 == 0 && fw_aligned(a->table, 16) && fw_aligned(a->table_out, 16);
    p.rpb = 1 + a->n_req / 2048;
    const int blocks = a->n_req ? (a->n_req + p.rpb - 1) / p.rpb : 1;
    const int64_t work = ((int64_t)a->n_rows / std::max(a->n_req, 1) + a->width) / PLAN_T;
    const int slices = (int)std::max<int64_t>(1, std::min<int64_t>(work / 4, std::max(1, 1024 / blocks)));
    hipLaunchKernelGGL(k_paged_plan, dim3(blocks, slices), dim3(PLAN_T), 0, c->stream, p);
    return fw_launched("fwhip_paged_plan");
}

// ---------------------------------------------------------------------------
// append
// A block per row: its K and V in pieces of VEC elements, 16 bytes or more of each
// where the addresses allow (VEC = 8), element by element where not.  Bound by
// the rows' bytes, read once and written once: 16,384 rows of 8 x 128 bf16 28.3 us,
// 4.75 TB/s, what a large copy reaches; 8 rows 3.0 us, a launch.
struct AppendP {
    int rows, pieces, per_head; // pieces of K in a row, and in a head
    FwDiv head;                 // by per_head
    int64_t k_row, k_head, v_row, v_head, page_stride, token_stride, head_stride, slots;
    int page;
    const void *k, *v;
    const int64_t *slot;
    void *kc, *vc;
};

template <typename S, typename D, int VEC>
__device__ __forceinline__ void append_piece(const S *from, D *to) {
    struct alignas(VEC == 1 ? sizeof(S) : 16) In {
        S v[VEC];
    };
    struct alignas(VEC == 1 ? sizeof(D) : 16) Out {
        D v[VEC];
    };
    const In a = *(const In *)from;
    Out b;
#pragma unroll
    for (int i = 0; i < VEC; i++) b.v[i] = fw_cvt<D>(fw_to_f32(a.v[i]));
    *(Out *)to = b;
}
template <typename S, typename D, int VEC>
__global__ void __launch_bounds__(256) k_paged_append(AppendP p) {
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x) {
        const int64_t slot = p.slot[row];
        if (slot < 0 || slot >= p.slots) continue;
        const int64_t to = slot / p.page * p.page_stride + slot % p.page * p.token_stride;
        for (int64_t i = threadIdx.x; i < 2 * (int64_t)p.pieces; i += blockDim.x) {
            const bool v = i >= p.pieces;
            const uint32_t at = (uint32_t)(v ? i - p.pieces : i), h = fw_div(at, p.head);
            const int64_t e = (int64_t)(at - h * p.per_head) * VEC;
            if (v) append_piece<S, D, VEC>((const S *)p.v + row * p.v_row + h * p.v_head + e, (D *)p.vc + to + h * p.head_stride + e);
            else append_piece<S, D, VEC>((const S *)p.k + row * p.k_row + h * p.k_head + e, (D *)p.kc + to + h * p.head_stride + e);
        }
    }
}

template <typename S, typename D, int VEC>
static void append_launch(hipStream_t st, const AppendP &p) {
    const int threads = (int)std::min<int64_t>(256, (2 * (int64_t)p.pieces + 63) / 64 * 64);
    hipLaunchKernelGGL((k_paged_append<S, D, VEC>), dim3((unsigned)std::min(p.rows, 1 << 20)), dim3(threads), 0, st, p);
}
template <typename S, int VEC>
static void append_to(hipStream_t st, int dtype, const AppendP &p) {
    if (dtype == FWHIP_T_F32) append_launch<S, float, VEC>(st, p);
    else if (dtype == FWHIP_T_F16) append_launch<S, fw_f16, VEC>(st, p);
    else append_launch<S, fw_bf16, VEC>(st, p);
}
template <int VEC>
static void append_from(hipStream_t st, int src, int dst, const AppendP &p) {
    if (src == FWHIP_T_F32) append_to<float, VEC>(st, dst, p);
    else if (src == FWHIP_T_F16) append_to<fw_f16, VEC>(st, dst, p);
    else append_to<fw_bf16, VEC>(st, dst, p);
}

extern "C" fwhip_status fwhip_paged_append(fwhip_ctx *c, const fwhip_paged_append_args *a) {
    if (!a) return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: args is NULL");
    if (!fw_is_dtype(a->src_dtype) || !fw_is_dtype(a->cache_dtype))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: unknown element type");
    if (a->n_rows < 0 || a->n_heads < 1 || a->head_dim < 1 || a->n_pages < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: bad size");
    if ((int64_t)a->n_heads * a->head_dim > 0x7fffffff || (int64_t)a->n_rows * a->n_heads * a->head_dim > (1ll << 38))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: too many elements");
    if (a->page_size < 1 || a->page_size > (1 << 24))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: page_size must be in 1..2^24");
    if (a->k_row < 0 || a->k_head < 0 || a->v_row < 0 || a->v_head < 0 || a->page_stride < 0 || a->token_stride < 0 ||
        a->head_stride < 0)
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: negative stride");
    if (a->n_rows && (!a->k || !a->v || !a->slot || (a->n_pages && (!a->k_cache || !a->v_cache))))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: NULL argument");
    if (!fw_aligned(a->k, fw_dtype_bytes(a->src_dtype)) || !fw_aligned(a->v, fw_dtype_bytes(a->src_dtype)) ||
        !fw_aligned(a->k_cache, fw_dtype_bytes(a->cache_dtype)) || !fw_aligned(a->v_cache, fw_dtype_bytes(a->cache_dtype)) ||
        !fw_aligned(a->slot, 8))
        return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: an address is not a multiple of its element's size");
    if (!c) return fw_fail(FWHIP_ERR_INVALID, "fwhip_paged_append: NULL ctx");
    if (a->n_rows == 0 || a->n_pages == 0) return FWHIP_OK;
    FwOnDevice dev(c);
    if (!dev.ok) return fw_fail(FWHIP_ERR_GENERIC, "fwhip_paged_append: hipSetDevice failed");
    // pieces of 8 elements where every address of one is a multiple of 16 bytes
    const int sb = fw_dtype_bytes(a->src_dtype), db = fw_dtype_bytes(a->cache_dtype);
    bool wide = a->head_dim % 8 == 0 && fw_aligned(a->k, 16) && fw_aligned(a->v, 16) && fw_aligned(a->k_cache, 16) &&
                fw_aligned(a->v_cache, 16);
    for (int64_t s : {a->k_row, a->k_head, a->v_row, a->v_head}) wide = wide && s * sb % 16 == 0;
    for (int64_t s : {a->page_stride, a->token_stride, a->head_stride}) wide = wide && s * db % 16 == 0;
    const int vec = wide ? 8 : 1;
    AppendP p;
    p.rows = a->n_rows;
    p.per_head = a->head_dim / vec;
    p.pieces = a->n_heads * p.per_head;
    p.head = fw_div_make((uint32_t)p.per_head);
    p.k_row = a->k_row;
    p.k_head = a->k_head;
    p.v_row = a->v_row;
    p.v_head = a->v_head;
    p.page_stride = a->page_stride;
    p.token_stride = a->token_stride;
    p.head_stride = a->head_stride;
    p.slots = (int64_t)a->n_pages * a->page_size;
    p.page = a->page_size;
    p.k = a->k;
    p.v = a->v;
    p.slot = a->slot;
    p.kc = a->k_cache;
    p.vc = a->v_cache;
    if (wide) append_from<8>(c->stream, a->src_dtype, a->cache_dtype, p);
    else append_from<1>(c->stream, a->src_dtype, a->cache_dtype, p);
    return fw_launched("fwhip_paged_append");
}
