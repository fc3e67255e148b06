// Attention over a quantised key / value cache (layout: qmv_kv.cuh; C-ABI declarations: include/nemicli_qmv.h).
#include <cmath>

#include "qmv_attn_tc.cuh"

using namespace qmv;

namespace {
constexpr int kMostKeys = 1 << 30;        // tokens a table may hold, query rows, rows a key head (max_new times its heads):
                                          // positions, windows and tiles' ends stay in 31 bits
bool bad_table(const KvView& c, int width, int window) { return width <= 0 || width > kMostKeys >> c.page_shift || window < 0; }
// a window no shorter than the table is none
int real_window(const KvView& c, int width, int window) { return window >= width << c.page_shift ? 0 : window; }
int few_rows(const AttnParams& P, int dtype, const AttnPlan& pl, cudaStream_t s) {
    switch (P.c.J) {
    case 2: return attn_dispatch<2>(P, dtype, pl, s);
    case 3: return attn_dispatch<3>(P, dtype, pl, s);
    case 4: return attn_dispatch<4>(P, dtype, pl, s);
    case 8: return attn_dispatch<8>(P, dtype, pl, s);
    }
    return ST_BAD_SHAPE;
}
}  // namespace

extern "C" {

int64_t qmv_kv_attend_workspace_bytes(const qmv_kv_cache* cache, int n_heads, int n_seq, int max_new, int dtype,
                                      int table_width, int window) {
    KvView c{};
    if (kv_view(cache, c) || n_heads <= 0 || n_heads > 65535 || n_heads % c.n_kv || n_seq <= 0 || n_seq > 65535 || max_new <= 0)
        return 0;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return 0;
    if (bad_table(c, table_width, window) || max_new > kMostKeys / (n_heads / c.n_kv)) return 0;
    window = real_window(c, table_width, window);
    const AttnTcPlan tc = attn_tc_plan(c, dtype, n_heads, n_seq, max_new, table_width, window);
    if (tc.used) return tc.grid > 0x7FFFFFFF ? 0 : tc.bytes + 1;      // (no workspace: one byte)
    const AttnPlan p = attn_plan(c, dtype, n_heads, n_seq, max_new, table_width, window);
    return p.grid ? p.bytes : 0;
}

int qmv_kv_attend(const qmv_kv_cache* cache, const void* q, int dtype, long long q_stride, int n_heads,
                  const int* tables, int table_width, const int* lens, const int* starts, int n_seq, long long n_rows,
                  int max_new, float scale, int window, void* out, void* workspace, long long workspace_bytes,
                  void* stream) {
    AttnParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!q || !tables || !lens || !out || !workspace) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (n_heads <= 0 || n_heads > 65535 || n_heads % P.c.n_kv || bad_table(P.c, table_width, window)) return ST_BAD_SHAPE;
    if (!std::isfinite(scale)) return ST_BAD_SHAPE;           // (its kernels would take NaN for the smallest scale)
    window = real_window(P.c, table_width, window);
    if (n_seq <= 0 || n_seq > 65535 || n_rows < 0 || n_rows > kMostKeys || max_new <= 0 || (!starts && n_rows < n_seq))
        return ST_BAD_TOKENS;
    if (q_stride < (long long)n_heads * P.c.dim) return ST_BAD_SHAPE;
    const uintptr_t four = 4 * elem_bytes(dtype);
    if (!aligned(q, four) || q_stride % 4 || !aligned(out, 16) || !aligned(tables, 4) || !aligned(lens, 4) ||
        !aligned(starts, 4) || !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    if (!starts) max_new = 1;
    if (max_new > kMostKeys / (n_heads / P.c.n_kv)) return ST_BAD_TOKENS;
    const AttnTcPlan tc = attn_tc_plan(P.c, dtype, n_heads, n_seq, max_new, table_width, window);
    const AttnPlan pl = attn_plan(P.c, dtype, n_heads, n_seq, max_new, table_width, window);
    if (tc.used ? tc.grid > 0x7FFFFFFF || workspace_bytes < tc.bytes : !pl.grid || workspace_bytes < pl.bytes) return ST_BAD_SHAPE;
    if (n_rows == 0) return ST_OK;
    P.q = q, P.q_stride = q_stride, P.out = out;
    P.tables = tables, P.row_entries = table_width, P.lens = lens, P.starts = starts;
    P.width = table_width, P.n_seq = n_seq, P.n_heads = n_heads, P.n_rows = int(n_rows);
    P.max_new = max_new, P.window = window, P.scale = scale;
    P.row_tiles = pl.row_tiles, P.split = pl.split, P.by_segment = pl.by_segment;
    P.parts = static_cast<float*>(workspace);
    P.desc = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + pl.part_bytes);
    P.status = device_status_ptr();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (tc.used) {
        P.row_tiles = tc.row_tiles, P.split = tc.split;
        switch (P.c.J) {
        case 2: return attn_tc_dispatch<2>(P, dtype, s);
        case 3: return attn_tc_dispatch<3>(P, dtype, s);
        case 4: return attn_tc_dispatch<4>(P, dtype, s);
        case 8: return attn_tc_dispatch<8>(P, dtype, s);
        }
    }
    return few_rows(P, dtype, pl, s);
}

int64_t qmv_kv_attend_chosen_workspace_bytes(const qmv_kv_cache* cache, int n_heads, long long n_rows, int dtype, int keep) {
    KvView c{};
    if (kv_view(cache, c) || n_heads <= 0 || n_heads > 65535 || n_heads % c.n_kv || n_rows <= 0 || n_rows > 65535) return 0;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return 0;
    if (bad_table(c, keep, 0)) return 0;
    const AttnPlan p = attn_plan(c, dtype, n_heads, int(n_rows), 1, keep, 0);
    return p.grid ? p.bytes : 0;
}

int qmv_kv_attend_chosen(const qmv_kv_cache* cache, const void* q, int dtype, long long q_stride, int n_heads, const int* chosen, int keep,
                         const int* held, long long n_rows, float scale, void* out, void* workspace, long long workspace_bytes,
                         void* stream) {
    AttnParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!q || !chosen || !held || !out || !workspace) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (n_heads <= 0 || n_heads > 65535 || n_heads % P.c.n_kv || bad_table(P.c, keep, 0) || !std::isfinite(scale)) return ST_BAD_SHAPE;
    if (n_rows < 0 || n_rows > 65535) return ST_BAD_TOKENS;
    if (q_stride < (long long)n_heads * P.c.dim) return ST_BAD_SHAPE;
    if (!aligned(q, 4 * elem_bytes(dtype)) || q_stride % 4 || !aligned(out, 16) || !aligned(chosen, 4) || !aligned(held, 4) || !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    if (n_rows == 0) return ST_OK;
    const AttnPlan pl = attn_plan(P.c, dtype, n_heads, int(n_rows), 1, keep, 0);
    if (!pl.grid || workspace_bytes < pl.bytes) return ST_BAD_SHAPE;
    P.q = q, P.q_stride = q_stride, P.out = out;
    P.tables = chosen, P.row_entries = (long long)P.c.n_kv * keep, P.head_entries = keep, P.lens = held;
    P.width = keep, P.n_seq = int(n_rows), P.n_heads = n_heads, P.n_rows = int(n_rows);
    P.max_new = 1, P.scale = scale;
    P.row_tiles = pl.row_tiles, P.split = pl.split, P.by_segment = pl.by_segment;
    P.parts = static_cast<float*>(workspace);
    P.desc = reinterpret_cast<int4*>(static_cast<uint8_t*>(workspace) + pl.part_bytes);
    P.status = device_status_ptr();
    return few_rows(P, dtype, pl, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
