/* The index arithmetic of the paged cache (csrc/fw_paged.h) as a plain C
 * library for the CPU tests. */
#include "fw_paged.h"

uint32_t t_div(uint32_t n, uint32_t d) { return fw_div(n, fw_div_make(d)); }
int64_t t_div_bad(uint32_t d, uint32_t lo, uint32_t hi, uint32_t step) {
    const struct FwDiv v = fw_div_make(d);
    int64_t bad = 0;
    for (uint64_t n = lo; n < hi; n += step) bad += fw_div((uint32_t)n, v) != (uint32_t)n / d;
    return bad;
}
void t_req(int32_t len, int32_t n_new, int32_t held, int32_t width, int32_t page, int64_t *rows, int64_t *need, int *status) {
    const struct FwReq r = fw_plan_req(len, n_new, held, width, fw_div_make((uint32_t)page));
    *rows = r.rows;
    *need = r.need;
    *status = r.status;
}
int64_t t_slot(int32_t id, uint32_t t, uint32_t page) {
    const struct FwDiv v = fw_div_make(page);
    return fw_slot(id, t, fw_div(t, v), v);
}
