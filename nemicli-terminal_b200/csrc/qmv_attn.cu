// Attention over a quantised key / value cache (layout: qmv_kv.cuh; C-ABI declarations: include/nemicli_qmv.h).
#include <type_traits>

#include "qmv_kv.cuh"

using namespace qmv;

namespace {

struct AttnParams {
    KvView c;
    const void* q;
    long long q_stride;                   // values between query rows
    void* out;                            // [n_rows][n_heads][dim]
    const int* tables;                    // [n_seq][width] page of each run of P tokens
    const int* lens;                      // [n_seq] tokens in the cache, the new ones among them
    const int* starts;                    // [n_seq + 1] first query row (null: row b is sequence b's)
    int width, n_seq, n_heads, n_rows, max_new, window;
    float scale;
    int* status;
};

// One warp per (query row, head), lane e of it value e of every block; keys one after another.
template <int DT, int J>
__global__ void __launch_bounds__(128) attn_row_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int b = blockIdx.z, head = blockIdx.y, i = blockIdx.x * 4 + warp;
    int row0 = b, row1 = b + 1;
    if (P.starts) {
        row0 = min(max(P.starts[b], 0), P.n_rows);
        row1 = min(max(P.starts[b + 1], row0), P.n_rows);
    }
    const int cap = P.width << P.c.page_shift;
    if (i == 0 && lane == 0 && P.status && (P.lens[b] < 0 || P.lens[b] > cap || row1 - row0 > P.max_new)) atomicOr(P.status, DEV_BAD_ADDRESS);
    if (i >= min(row1 - row0, P.max_new)) return;
    const int len = min(max(P.lens[b], 0), cap);
    const int pos = len - (row1 - row0) + i;
    const int hk = head / (P.n_heads / P.c.n_kv);
    const T* q = static_cast<const T*>(P.q) + (row0 + i) * P.q_stride + head * 32 * J;
    float x[J], o[J];
#pragma unroll
    for (int j = 0; j < J; ++j) x[j] = to_float(q[32 * j + lane]) * P.scale, o[j] = 0.f;
    float top = -INFINITY, sum = 0.f;
    const int first = P.window > 0 ? max(0, pos - P.window + 1) : 0;
    const int kt = lane >> 3, ke = lane & 7, vg = lane >> 2, ve = lane & 3;
    for (int t = first; t <= pos; ++t) {
        const long long page = P.tables[(long long)b * P.width + (t >> P.c.page_shift)];
        if (page < 0 || page >= P.c.n_pages) {
            if (P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
            continue;
        }
        const int at = t & (P.c.page() - 1);
        const uint8_t* kr = P.c.k + P.c.k_row(page, hk, at);
        const uint8_t* vr = P.c.v + P.c.v_pair(page, hk, at >> 1);
        const __half* sc = P.c.sc + P.c.scale_row(page, hk, at);
        float s = 0.f, v[J];
#pragma unroll
        for (int j = 0; j < J; ++j) {
            int code;
            if (P.c.kb == 4) code = ((kr[(kt * J + j) * 4 + 2 * (ke & 1) + (ke >> 2)] >> (4 * ((ke >> 1) & 1))) & 15) - 8;
            else code = int(kr[(kt * J + j) * 8 + 4 * (ke >> 2) + 2 * (ke & 1) + ((ke & 3) >> 1)]) - 128;
            s += x[j] * (__half2float(sc[j]) * float(code));
            if (P.c.vb == 4) code = ((vr[(vg * J + j) * 4 + 2 * (at & 1) + (ve >> 1)] >> (4 * (ve & 1))) & 15) - 8;
            else code = int(vr[(vg * J + j) * 8 + 4 * (ve >> 1) + 2 * (at & 1) + (ve & 1)]) - 128;
            v[j] = __half2float(sc[J + j]) * float(code);
        }
        s = warp_sum(s);
        const float m = fmaxf(top, s), f = expf(top - m), p = expf(s - m);
        sum = sum * f + p;
#pragma unroll
        for (int j = 0; j < J; ++j) o[j] = o[j] * f + p * v[j];
        top = m;
    }
    T* out = static_cast<T*>(P.out) + ((long long)(row0 + i) * P.n_heads + head) * 32 * J;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        T r;
        from_float(r, sum > 0.f ? o[j] / sum : 0.f);
        out[32 * j + lane] = r;
    }
}

}  // namespace

extern "C" {

int64_t qmv_kv_attend_workspace_bytes(const qmv_kv_cache* cache, int n_heads, int n_seq, int max_new, int dtype) {
    KvView c{};
    if (kv_view(cache, c) || n_heads <= 0 || n_heads % c.n_kv || n_seq <= 0 || max_new <= 0) return 0;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return 0;
    return 256;
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
    if (n_heads <= 0 || n_heads > 65535 || n_heads % P.c.n_kv || table_width <= 0 ||
        table_width > (0x7FFFFFFF >> P.c.page_shift) || window < 0)
        return ST_BAD_SHAPE;
    if (n_seq <= 0 || n_seq > 65535 || n_rows < 0 || n_rows > 0x7FFFFFFFLL || max_new <= 0 || (!starts && n_rows < n_seq))
        return ST_BAD_TOKENS;
    if (q_stride < (long long)n_heads * P.c.dim) return ST_BAD_SHAPE;
    const uintptr_t four = 4 * elem_bytes(dtype);
    if (!aligned(q, four) || q_stride % 4 || !aligned(out, 16) || !aligned(tables, 4) || !aligned(lens, 4) ||
        !aligned(starts, 4) || !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    if (workspace_bytes < qmv_kv_attend_workspace_bytes(cache, n_heads, n_seq, max_new, dtype)) return ST_BAD_SHAPE;
    if (n_rows == 0) return ST_OK;
    P.q = q, P.q_stride = q_stride, P.out = out;
    P.tables = tables, P.lens = lens, P.starts = starts;
    P.width = table_width, P.n_seq = n_seq, P.n_heads = n_heads, P.n_rows = int(n_rows);
    P.max_new = starts ? max_new : 1, P.window = window, P.scale = scale;
    P.status = device_status_ptr();
    const dim3 grid((P.max_new + 3) / 4, n_heads, n_seq);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return by_elem(dtype, [&](auto c) {
        constexpr int DT = decltype(c)::value;
        switch (P.c.J) {
        case 2: attn_row_kernel<DT, 2><<<grid, 128, 0, s>>>(P); break;
        case 3: attn_row_kernel<DT, 3><<<grid, 128, 0, s>>>(P); break;
        case 4: attn_row_kernel<DT, 4><<<grid, 128, 0, s>>>(P); break;
        case 8: attn_row_kernel<DT, 8><<<grid, 128, 0, s>>>(P); break;
        default: return int(ST_BAD_SHAPE);
        }
        return launched();
    });
}

}  // extern "C"
