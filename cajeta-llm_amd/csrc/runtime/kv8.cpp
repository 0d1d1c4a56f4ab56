// kv8.cpp — the launch seam of the 8-bit K/V pages (kernels/kv8.hip): the
// checks of the arguments and extents, and the choice of the kernels. What
// lives on the device (segments, page tables) is checked by the kernels.
#include "rt.h"
#include <algorithm>

namespace cj {
namespace {

constexpr int64_t ROW_MOST = (int64_t)1 << 40;   // floats between rows, at most

int64_t code_bytes(int64_t n_pages, int64_t n_kv, int64_t hd) { return n_pages * n_kv * 64 * hd; }
int64_t plane_bytes(int64_t n_pages, int64_t n_kv, int64_t hd) { return code_bytes(n_pages, n_kv, hd) + n_pages * n_kv * 16; }

bool shape_ok(int32_t n_q, int32_t n_kv, int32_t hd) {
    return (hd == 64 || hd == 128) && n_kv > 0 && n_kv <= 4096 && n_q > 0 && n_q <= 65536 && n_q % n_kv == 0 && n_q / n_kv <= 64;
}

// `rows` rows of `width` floats, `stride` apart, read and written by 16 bytes.
bool rows_ok(int64_t h, int64_t rows, int64_t stride, int64_t width) {
    return stride >= width && stride <= ROW_MOST && stride % 4 == 0 && (h & 15) == 0 &&
           in_buffer(dptr(h), ((rows - 1) * stride + width) * 4);
}

// What the entry points have in common: planes, page table and segments.
int common(const char *who, cj_kv8_args &a, int64_t kplane, int64_t vplane, int64_t pgtab, int64_t segs, int32_t n_segs,
           int32_t max_rows, int32_t n_rows, int32_t n_pages, int32_t n_slots, int32_t slot_pages, int32_t n_q, int32_t n_kv,
           int32_t hd, int64_t status) {
    if (!shape_ok(n_q, n_kv, hd)) return fail(CJ_ERR_ARG, "%s: heads %d/%d of size %d are not served", who, n_q, n_kv, hd);
    if (n_segs <= 0 || max_rows <= 0 || n_rows <= 0)
        return fail(CJ_ERR_ARG, "%s: %d segments of up to %d rows, %d rows", who, n_segs, max_rows, n_rows);
    if ((int64_t)max_rows * n_q > (1 << 30))
        return fail(CJ_ERR_ARG, "%s: %d rows of %d heads exceed a launch", who, max_rows, n_q);
    if (n_pages <= 0 || n_slots <= 0 || slot_pages <= 0 || slot_pages > 0x7fffffff / 64)
        return fail(CJ_ERR_ARG, "%s: %d pages, %d slots of %d pages", who, n_pages, n_slots, slot_pages);
    if (!ready()) return fail(CJ_ERR_STATE, "cj_init has not run");
    const int64_t plane = plane_bytes(n_pages, n_kv, hd);
    if ((kplane & 15) || (vplane & 15) || !in_buffer(dptr(kplane), plane) || !in_buffer(dptr(vplane), plane))
        return fail(CJ_ERR_ARG, "%s: a plane is not 16-byte aligned or smaller than %d pages", who, n_pages);
    if ((segs & 15) || !in_buffer(dptr(segs), (int64_t)n_segs * 16))
        return fail(CJ_ERR_ARG, "%s: the segments are not 16-byte aligned or fewer than %d", who, n_segs);
    if ((pgtab & 3) || !in_buffer(dptr(pgtab), (int64_t)n_slots * slot_pages * 4))
        return fail(CJ_ERR_ARG, "%s: the page table is smaller than %d slots of %d pages", who, n_slots, slot_pages);
    if (status && ((status & 3) || !in_buffer(dptr(status), 4))) return fail(CJ_ERR_ARG, "%s: status is outside its buffer", who);
    const int64_t codes = code_bytes(n_pages, n_kv, hd);
    a.kc = (uint8_t *)dptr(kplane); a.vc = (uint8_t *)dptr(vplane);
    a.ks = (float *)dptr(kplane + codes); a.vs = (float *)dptr(vplane + codes);
    a.pgtab = (const int32_t *)dptr(pgtab); a.segs = (const int32_t *)dptr(segs); a.status = (int32_t *)dptr(status);
    a.n_segs = n_segs; a.max_rows = max_rows; a.n_rows = n_rows; a.limit = slot_pages * 64;
    a.n_pages = n_pages; a.n_slots = n_slots; a.slot_pages = slot_pages; a.n_q = n_q; a.n_kv = n_kv;
    return CJ_OK;
}

// Blocks of 16 positions that max_rows rows reach at most.
int64_t blocks_of(int32_t max_rows) { return ((int64_t)max_rows + 14) / 16 + 1; }

// (A launch holds fewer than 2^32 threads.)
int run(const char *kernel, int32_t hd, int64_t grid, uint32_t block, const cj_kv8_args &a) {
    if (grid > 0xffffffffll / block) return fail(CJ_ERR_ARG, "%s: %lld workgroups exceed a launch", kernel, (long long)grid);
    return launch((std::string(kernel) + "_h" + std::to_string(hd)).c_str(), (uint32_t)grid, block, 0, a);
}

// How a call runs. A column is a row and a query head of one kv head's group;
// a workgroup takes 16, 32 or 128 of a segment's and, up to 32, a part of the
// positions (a wave a page at a time), whose parts a second launch joins.
// Measured on 256 CUs at head size 128, 4 heads a kv head, 8 kv heads (us):
//  - 128 columns a workgroup convert a page once for four waves, but keep the
//    chip busy only where there are enough of them (32 → 128; 1024 rows behind
//    1033, 256 workgroups of 128: 73 → 81 stays; 1536 rows, 384: 117 → 112;
//    2048 rows, 512: 162 → 150);
//  - the positions are split for one workgroup a CU (for one and for two; 32
//    sequences of 2048: 25 and 29; of 4096: 46 and 52; 8 of 65500: 170 and
//    172; one: 30 and 31; 24 of 8192: 69 and 76), and not where it saves a
//    wave two pages or less for the join's 3 us (one sequence of 513, no split
//    and one: 8.8 and 9.6; of 1025, 12.2 and 10.5);
//  - a little over one workgroup a CU would leave a few CUs two of them: long
//    ones are split in three (none and three; 33 sequences of 6000: 93 and 81,
//    40: 97 and 88, but 50: 106 and 115; 33 of 2048: 34 and 35).
struct Plan {
    int64_t tile_cols, col_tiles, splits, split_pages, bytes;
};
Plan plan_attend(int64_t n_segs, int64_t max_rows, int64_t max_count, int64_t n_q, int64_t n_kv, int64_t hd, int64_t window) {
    Plan p;
    const int64_t cols = max_rows * (n_q / n_kv), cus = std::max(1, device_cus()), heads = n_segs * n_kv;
    p.tile_cols = cols <= 16 ? 16 : 4 * heads * ((cols + 127) / 128) < 5 * cus ? 32 : 128;
    p.col_tiles = (cols + p.tile_cols - 1) / p.tile_cols;
    int64_t pages = (max_count + 63) / 64;
    if (window) pages = std::min(pages, (window + max_rows) / 64 + 2);   // what a tile's rows see together
    const int64_t units = heads * p.col_tiles;
    int64_t want = std::max<int64_t>(1, cus / units);
    if (p.tile_cols == 16 && units > cus && 3 * units <= 4 * cus && pages >= 64) want = 3;
    p.split_pages = std::max<int64_t>(4, (pages + want - 1) / want);
    if (p.tile_cols == 128 || pages <= p.split_pages + 8) p.split_pages = pages;
    p.splits = (pages + p.split_pages - 1) / p.split_pages;
    p.bytes = p.splits > 1 ? units * p.splits * p.tile_cols * (hd + 2) * 4 : 0;
    return p;
}

}  // namespace
}  // namespace cj

using namespace cj;

extern "C" {

int64_t cj_kv8_plane_bytes(int32_t n_pages, int32_t n_kv, int32_t head_dim) {
    if (n_pages <= 0 || !shape_ok(n_kv, n_kv, head_dim))
        return fail(CJ_ERR_ARG, "cj_kv8_plane_bytes: %d pages of %d heads of size %d", n_pages, n_kv, head_dim);
    return plane_bytes(n_pages, n_kv, head_dim);
}

int32_t cj_kv8_append(int64_t q_out, int64_t q, int64_t k, int64_t v, int64_t kplane, int64_t vplane, int64_t qw, int64_t kw,
                      int64_t rope, int64_t pgtab, int64_t segs, int32_t n_segs, int32_t max_rows, int32_t n_rows,
                      int32_t rope_ctx, int32_t n_pages, int32_t n_slots, int32_t slot_pages, int32_t n_q, int32_t n_kv,
                      int32_t head_dim, int64_t q_out_stride, int64_t q_stride, int64_t kv_stride, int32_t norm, float eps,
                      int32_t form, int64_t status) {
    cj_kv8_args a{};
    if (int rc = common("cj_kv8_append", a, kplane, vplane, pgtab, segs, n_segs, max_rows, n_rows, n_pages, n_slots, slot_pages,
                        n_q, n_kv, head_dim, status))
        return rc;
    const int64_t qn = (int64_t)n_q * head_dim, kn = (int64_t)n_kv * head_dim;
    if (!rows_ok(k, n_rows, kv_stride, kn) || !rows_ok(v, n_rows, kv_stride, kn))
        return fail(CJ_ERR_ARG, "cj_kv8_append: k or v is not %d rows of %lld floats, 16-byte aligned", n_rows, (long long)kn);
    if ((q != 0) != (q_out != 0) || (q && (!rows_ok(q, n_rows, q_stride, qn) || !rows_ok(q_out, n_rows, q_out_stride, qn))))
        return fail(CJ_ERR_ARG, "cj_kv8_append: q or q_out is not %d rows of %lld floats, 16-byte aligned", n_rows, (long long)qn);
    if (rope_ctx <= 0 || (rope & 15) || !in_buffer(dptr(rope), (int64_t)rope_ctx * head_dim * 4))
        return fail(CJ_ERR_ARG, "cj_kv8_append: the rope table is smaller than %d positions", rope_ctx);
    if (norm && (!in_buffer(dptr(kw), head_dim * 4) || (q && !in_buffer(dptr(qw), head_dim * 4)) || (kw & 3) || (qw & 3)))
        return fail(CJ_ERR_ARG, "cj_kv8_append: a norm weight is smaller than %d floats", head_dim);
    a.q = (const float *)dptr(q); a.k = (const float *)dptr(k); a.v = (const float *)dptr(v); a.q_out = (float *)dptr(q_out);
    a.qw = (const float *)dptr(qw); a.kw = (const float *)dptr(kw); a.rope_cs = (const float *)dptr(rope);
    a.q_stride = q_stride; a.kv_stride = kv_stride; a.out_stride = q_out_stride;
    a.limit = std::min(a.limit, rope_ctx);
    a.norm = norm != 0; a.form = form; a.eps = eps;
    const int64_t kv = blocks_of(max_rows) * n_segs * n_kv, items = KV8_QS * 2048 / head_dim, per = q ? ((int64_t)max_rows * n_q + items - 1) / items : 0;
    if (kv > 0x7fffffff || per > 0x7fffffff) return fail(CJ_ERR_ARG, "cj_kv8_append: %d x %d rows exceed a launch", n_segs, max_rows);
    a.kv_wgs = (int32_t)kv; a.per_seg = (int32_t)per;
    return run("cj_kv8_append", head_dim, kv + per * n_segs, 256, a);
}

int32_t cj_kv8_read(int64_t k_out, int64_t v_out, int64_t kplane, int64_t vplane, int64_t pgtab, int64_t segs, int32_t n_segs,
                    int32_t max_rows, int32_t n_rows, int32_t n_pages, int32_t n_slots, int32_t slot_pages, int32_t n_kv,
                    int32_t head_dim, int64_t out_stride, int64_t status) {
    cj_kv8_args a{};
    if (int rc = common("cj_kv8_read", a, kplane, vplane, pgtab, segs, n_segs, max_rows, n_rows, n_pages, n_slots, slot_pages,
                        n_kv, n_kv, head_dim, status))
        return rc;
    const int64_t kn = (int64_t)n_kv * head_dim;
    if ((!k_out && !v_out) || (k_out && !rows_ok(k_out, n_rows, out_stride, kn)) || (v_out && !rows_ok(v_out, n_rows, out_stride, kn)))
        return fail(CJ_ERR_ARG, "cj_kv8_read: k_out or v_out is not %d rows of %lld floats, 16-byte aligned", n_rows, (long long)kn);
    a.out = (float *)dptr(k_out); a.out2 = (float *)dptr(v_out); a.out_stride = out_stride;
    return run("cj_kv8_read", head_dim, blocks_of(max_rows) * n_segs * n_kv, 256, a);
}

int64_t cj_kv8_attend_bytes(int32_t n_segs, int32_t max_rows, int32_t max_count, int32_t n_q, int32_t n_kv, int32_t head_dim,
                            int32_t window) {
    if (!shape_ok(n_q, n_kv, head_dim) || n_segs <= 0 || max_rows <= 0 || (int64_t)max_rows * n_q > (1 << 30) || max_count <= 0 || window < 0)
        return fail(CJ_ERR_ARG, "cj_kv8_attend_bytes: %d segments of %d rows, %d positions, heads %d/%d of size %d", n_segs,
                    max_rows, max_count, n_q, n_kv, head_dim);
    if (!ready()) return fail(CJ_ERR_STATE, "cj_init has not run");   // the split follows the device's size
    return plan_attend(n_segs, max_rows, max_count, n_q, n_kv, head_dim, window).bytes;
}

int32_t cj_kv8_attend(int64_t out, int64_t q, int64_t kplane, int64_t vplane, int64_t pgtab, int64_t segs, int64_t part,
                      int32_t n_segs, int32_t max_rows, int32_t n_rows, int32_t max_count, int32_t n_pages, int32_t n_slots,
                      int32_t slot_pages, int32_t n_q, int32_t n_kv, int32_t head_dim, int64_t q_stride, int64_t out_stride,
                      int32_t window, float scale, int64_t status) {
    cj_kv8_args a{};
    if (int rc = common("cj_kv8_attend", a, kplane, vplane, pgtab, segs, n_segs, max_rows, n_rows, n_pages, n_slots, slot_pages,
                        n_q, n_kv, head_dim, status))
        return rc;
    const int64_t qn = (int64_t)n_q * head_dim;
    if (max_count <= 0 || window < 0) return fail(CJ_ERR_ARG, "cj_kv8_attend: %d positions, window %d", max_count, window);
    if (!rows_ok(q, n_rows, q_stride, qn) || !rows_ok(out, n_rows, out_stride, qn))
        return fail(CJ_ERR_ARG, "cj_kv8_attend: q or out is not %d rows of %lld floats, 16-byte aligned", n_rows, (long long)qn);
    a.q = (const float *)dptr(q); a.out = (float *)dptr(out); a.q_stride = q_stride; a.out_stride = out_stride;
    a.limit = std::min(a.limit, max_count); a.window = window; a.scale = scale;
    const Plan p = plan_attend(n_segs, max_rows, max_count, n_q, n_kv, head_dim, window);
    if (p.bytes && ((part & 15) || !in_buffer(dptr(part), p.bytes)))
        return fail(CJ_ERR_ARG, "cj_kv8_attend: part is not 16-byte aligned or smaller than %lld bytes", (long long)p.bytes);
    // the join: as many threads over a column's splits as there are splits, of the W that a workgroup has for its columns
    int64_t ways = 1, W = 1024 / head_dim;
    while (ways < W && ways < p.splits) ways *= 2;
    const int64_t units = (int64_t)n_segs * n_kv * p.splits, per = W / ways, cols = (int64_t)max_rows * (n_q / n_kv);
    const int64_t wgs = (p.tile_cols == 32 ? (units + 7) / 8 * 8 : units) * p.col_tiles, join = (int64_t)n_segs * n_kv * ((cols + per - 1) / per);
    if (wgs > 0x7fffffff || join > 0x7fffffff)
        return fail(CJ_ERR_ARG, "cj_kv8_attend: %d x %d rows of %d heads exceed a launch", n_segs, max_rows, n_q);
    a.part = (float *)dptr(part); a.col_tiles = (int32_t)p.col_tiles; a.tile_cols = (int32_t)p.tile_cols;
    a.splits = (int32_t)p.splits; a.split_pages = (int32_t)p.split_pages; a.join_ways = (int32_t)ways;
    const int rc = run(p.tile_cols == 16 ? "cj_kv8_attend_c16" : p.tile_cols == 32 ? "cj_kv8_attend_c32" : "cj_kv8_attend_c128", head_dim, wgs, 256, a);
    return rc || p.splits == 1 ? rc : run("cj_kv8_join", head_dim, join, 256, a);
}

}  // extern "C"
