// Pages of the quantised cache that a query needs: boxes around each page's keys, their scores, the choice; and attention over the
// chosen pages (cache layout: qmv_kv.cuh; C-ABI declarations: include/nemicli_qmv.h).
//
//   lo[c], hi[c]   the least and largest key of the page, channel by channel
//   s = max over the query heads h of a key head of  sum_c max(q_h[c] lo[c], q_h[c] hi[c])   >= q_h . k for every key k of the page
//
// A box takes 4 bytes a channel where a page of 64 keys takes 36 (Q4_0), so the choice reads a ninth of the cache's keys and the
// attention the chosen pages.
#include <algorithm>
#include <climits>
#include <cmath>

#include "qmv_attn_tc.cuh"

using namespace qmv;

namespace {

constexpr int kThreads = 256;

// ---- boxes -----------------------------------------------------------------------------------------------------

struct BoxParams {
    KvView c;
    __half* bounds;                       // [n_pages][n_kv][2][dim]
    const int* tables;
    const int* lens;
    const int* starts;                    // (null: one new token a sequence)
    int width, n_seq, most;               // most: pages a sequence completes, at most
    int* status;
};

// eight codes of a key as values without scale
template <int KB>
__device__ __forceinline__ void codes8(const uint32_t* w, float (&v)[8]) {
#pragma unroll
    for (int n = 0; n < 8; ++n) {
        const uint32_t c = KB == 4 ? w[0] >> (16 * (n & 1) + 4 * (n >> 1)) & 15u : w[KB == 4 ? 0 : n >> 2] >> (8 * (2 * (n & 1) + ((n & 3) >> 1))) & 255u;
        v[n] = float(int(c) - (KB == 4 ? 8 : 128));
    }
}

// A warp a page and key head: lane (token, unit) takes the 8 values of one unit (block j, run t) of every kTok-th token.  Bound by
// reading K's codes and scales once (V's scales lie in the same sectors).
template <int J, int KB>
__global__ void __launch_bounds__(kThreads) box_kernel(const __grid_constant__ BoxParams P) {
    constexpr int kUnits = 4 * J, kTok = 32 / kUnits, D = 32 * J;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const long long item = id / P.c.n_kv;
    const int head = int(id - item * P.c.n_kv), seq = int(item / P.most), nth = int(item - (long long)seq * P.most);
    if (seq >= P.n_seq) return;                                   // whole warps
    const int cap = P.width << P.c.page_shift, len = __ldg(P.lens + seq), held = min(max(len, 0), cap);
    int fresh = P.starts ? __ldg(P.starts + seq + 1) - __ldg(P.starts + seq) : 1;
    fresh = min(max(fresh, 0), held);
    const int page_i = ((held - fresh) >> P.c.page_shift) + nth, end = held >> P.c.page_shift;
    if (nth == 0 && head == 0 && lane == 0 && P.status && (held != len || end - page_i > P.most)) atomicOr(P.status, DEV_BAD_ADDRESS);
    if (page_i >= end) return;
    const int page = __ldg(P.tables + (long long)seq * P.width + page_i);
    if (page < 0 || page >= P.c.n_pages) {
        if (lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
        return;
    }
    const int unit = lane % kUnits, tok = lane / kUnits, t = unit / J, j = unit - t * J;
    const uint8_t* k = P.c.k + P.c.k_row(page, head, 0) + unit * KB;
    const __half* sc = P.c.sc + P.c.scale_row(page, head, 0) + j;
    float lo[8], hi[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    if (tok < kTok) {
#pragma unroll 8
        for (int x = tok; x < P.c.page(); x += kTok) {
            uint32_t w[2];
            if constexpr (KB == 4) {
                w[0] = __ldg(reinterpret_cast<const uint32_t*>(k + x * (kUnits * KB)));
            } else {
                const uint2 both = __ldg(reinterpret_cast<const uint2*>(k + x * (kUnits * KB)));
                w[0] = both.x, w[1] = both.y;
            }
            const float d = __half2float(sc[x * 2 * J]);
            float v[8];
            codes8<KB>(w, v);
#pragma unroll
            for (int i = 0; i < 8; ++i) lo[i] = fminf(lo[i], d * v[i]), hi[i] = fmaxf(hi[i], d * v[i]);
        }
    }
    // the other tokens of the unit
#pragma unroll
    for (int o = 1; o < kTok; ++o)
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float a = __shfl_sync(0xffffffffu, lo[i], (lane + o * kUnits) % (kTok * kUnits)), b = __shfl_sync(0xffffffffu, hi[i], (lane + o * kUnits) % (kTok * kUnits));
            // (o by o of the lanes as they were: a and b are the partial results, which only grow)
            lo[i] = fminf(lo[i], a), hi[i] = fmaxf(hi[i], b);
        }
    if (tok) return;
    // outwards to fp16, within its range: the box still holds every key
    uint32_t a[4], b[4];
    auto in = [](float x) { return fminf(fmaxf(x, -kKvMax), kKvMax); };
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[i] = h2_bits(__halves2half2(__float2half_rd(in(lo[2 * i])), __float2half_rd(in(lo[2 * i + 1]))));
        b[i] = h2_bits(__halves2half2(__float2half_ru(in(hi[2 * i])), __float2half_ru(in(hi[2 * i + 1]))));
    }
    __half* out = P.bounds + ((long long)page * P.c.n_kv + head) * (2 * D) + 32 * j + 8 * t;
    *reinterpret_cast<uint4*>(out) = make_uint4(a[0], a[1], a[2], a[3]);
    *reinterpret_cast<uint4*>(out + D) = make_uint4(b[0], b[1], b[2], b[3]);
}

// ---- scores ----------------------------------------------------------------------------------------------------

struct ChooseParams {
    const void* q;
    long long q_stride;
    const __half* bounds;
    long long n_pages;
    const int* tables;
    const int* lens;
    const int* starts;
    int n_kv, group, width, shift, n_seq, n_rows, keep, first, last;
    double* scores;                       // workspace: [rows][n_kv][width]
    int* chosen;                          // [rows][n_kv][keep]
    int* held;                            // [rows]
    int* status;
};

struct Row {
    int seq, pos;                         // sequence (-1: none), position in it
};
// the row's sequence and place, by the whole CTA
__device__ __forceinline__ Row find_row(const ChooseParams& P, int row, int* s_seq, bool tell) {
    if (threadIdx.x == 0) *s_seq = P.starts ? -1 : row < P.n_seq ? row : -1;
    __syncthreads();
    if (P.starts)
        for (int b = threadIdx.x; b < P.n_seq; b += kThreads)
            if (__ldg(P.starts + b) <= row && row < __ldg(P.starts + b + 1)) *s_seq = b;
    __syncthreads();
    const int seq = *s_seq;
    if (seq < 0) return Row{-1, -1};
    const int cap = P.width << P.shift, len = __ldg(P.lens + seq), held = min(max(len, 0), cap);
    if (tell && held != len && threadIdx.x == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    return Row{seq, P.starts ? held - (min(__ldg(P.starts + seq + 1), P.n_rows) - row) : held - 1};
}

constexpr int kPagesCta = 64;             // pages a CTA scores

// Eight lanes a page, each J runs of 4 channels; heads four at a time.  In fp64: products of a query and an fp16 bound are exact, and
// pages next to the border between chosen and left have to come out the same way whatever the order of the sums.
template <int DT, int J>
__global__ void __launch_bounds__(kThreads) score_kernel(const __grid_constant__ ChooseParams P) {
    using T = typename Elem<DT>::type;
    constexpr int D = 32 * J;
    extern __shared__ __align__(16) double s_q[];                 // [group up to 4s][J][2][8][2]
    __shared__ int s_seq;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, l = lane & 7;
    const int head = blockIdx.y, row = blockIdx.z;
    const Row r = find_row(P, row, &s_seq, false);
    const int at = r.pos >> P.shift;                              // the query's own page
    const int begin = P.first + blockIdx.x * kPagesCta, end = min(at + 1 - P.last, begin + kPagesCta);
    if (r.pos < 0 || at + 1 <= P.keep || begin >= end) return;
    const int groups = (P.group + 3) / 4;
    for (int i = tid; i < groups * 4 * D; i += kThreads) {
        const int h = i / D, c = i - h * D;
        const double v = h < P.group ? double(to_float(static_cast<const T*>(P.q)[row * P.q_stride + (long long)(head * P.group + h) * D + c])) : 0.0;
        s_q[h * D + ((c / 32 * 2 + (c & 2) / 2) * 8 + (c % 32) / 4) * 2 + (c & 1)] = v;
    }
    __syncthreads();
    for (int i0 = begin + 4 * warp; i0 < end; i0 += 4 * (kThreads / 32)) {
        const int i = i0 + (lane >> 3);
        const int page = i < end ? __ldg(P.tables + (long long)r.seq * P.width + i) : -1;
        const bool there = page >= 0 && page < P.n_pages;
        uint2 lo[J], hi[J];
        const __half* box = P.bounds + ((long long)(there ? page : 0) * P.n_kv + head) * (2 * D) + 4 * l;
#pragma unroll
        for (int p = 0; p < J; ++p) {
            lo[p] = there ? __ldg(reinterpret_cast<const uint2*>(box + 32 * p)) : make_uint2(0, 0);
            hi[p] = there ? __ldg(reinterpret_cast<const uint2*>(box + D + 32 * p)) : make_uint2(0, 0);
        }
        double best = -INFINITY;
        for (int g = 0; g < groups; ++g) {
            double acc[4] = {0.0, 0.0, 0.0, 0.0};
            const double* q = s_q + 4 * g * D + 2 * l;
#pragma unroll
            for (int p = 0; p < J; ++p)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const float2 a = unpack_h2(h ? lo[p].y : lo[p].x), b = unpack_h2(h ? hi[p].y : hi[p].x);
                    const double a0 = a.x, a1 = a.y, b0 = b.x, b1 = b.y;
#pragma unroll
                    for (int n = 0; n < 4; ++n) {
                        const double2 v = *reinterpret_cast<const double2*>(q + n * D + (p * 2 + h) * 16);
                        acc[n] = fma(v.x, v.x > 0.0 ? b0 : a0, acc[n]);
                        acc[n] = fma(v.y, v.y > 0.0 ? b1 : a1, acc[n]);
                    }
                }
#pragma unroll
            for (int o = 1; o < 8; o *= 2)
#pragma unroll
                for (int n = 0; n < 4; ++n) acc[n] += __shfl_xor_sync(0xffffffffu, acc[n], o);
#pragma unroll
            for (int n = 0; n < 4; ++n)
                if (4 * g + n < P.group) best = fmax(best, acc[n]);
        }
        if (i < end && l == 0) P.scores[((long long)row * P.n_kv + head) * P.width + i] = there ? best : -INFINITY;
    }
}

// ---- the choice ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t ordered64(double x) {
    if (!(x == x)) return 0;
    const uint64_t b = __double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// A CTA a row and key head.  The k-th largest score by digits of 8 bits from the top: a histogram of those that agree with
// the digits so far; then the pages from it on, in order.
__global__ void __launch_bounds__(kThreads) choose_kernel(const __grid_constant__ ChooseParams P) {
    __shared__ int s_seq, s_hist[256], s_digit, s_need, s_warp[kThreads / 32];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.x % P.n_kv, row = blockIdx.x / P.n_kv;
    const Row r = find_row(P, row, &s_seq, head == 0);
    int* out = P.chosen + (long long)blockIdx.x * P.keep;
    const int* table = P.tables + (long long)max(r.seq, 0) * P.width;
    const int n = r.pos < 0 ? 0 : (r.pos >> P.shift) + 1, kept = min(n, P.keep);
    if (head == 0 && tid == 0) P.held[row] = n ? ((kept - 1) << P.shift) + (r.pos & ((1 << P.shift) - 1)) + 1 : 0;
    if (n <= P.keep) {
        for (int i = tid; i < P.keep; i += kThreads) out[i] = i < n ? __ldg(table + i) : -1;
        return;
    }
    const int begin = P.first, end = n - P.last, k = P.keep - P.first - P.last;
    for (int i = tid; i < P.first; i += kThreads) out[i] = __ldg(table + i);
    for (int i = tid; i < P.last; i += kThreads) out[P.keep - P.last + i] = __ldg(table + end + i);
    if (k == 0) return;
    const double* scores = P.scores + (long long)blockIdx.x * P.width;
    uint64_t prefix = 0, mask = 0;
    int need = k;                                                 // of those that agree with prefix
    bool tied = true;
    for (int shift = 56; shift >= 0; shift -= 8) {
        s_hist[tid] = 0;
        __syncthreads();
        for (int i = begin + tid; i < end; i += kThreads) {
            const uint64_t key = ordered64(scores[i]);
            if ((key & mask) == prefix) atomicAdd(&s_hist[key >> shift & 255], 1);
        }
        __syncthreads();
        if (warp == 0) {
            int own[8], sum = 0;                                  // lane: digits 255 - 8 lane .. 248 - 8 lane
#pragma unroll
            for (int i = 0; i < 8; ++i) own[i] = s_hist[255 - 8 * lane - i], sum += own[i];
            int inc = sum;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const int y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            int above = inc - sum;
            if (above < need && need <= inc) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (above < need && need <= above + own[i]) s_digit = 255 - 8 * lane - i, s_need = need - above;
                    above += own[i];
                }
            }
        }
        __syncthreads();
        prefix |= uint64_t(s_digit) << shift, mask |= 255ull << shift;
        need = s_need;
        if (s_hist[s_digit] == need) {                            // all of them
            tied = false;
            break;
        }
        __syncthreads();
    }
    // above the prefix every one, with it the first `need`
    int base = P.first, equal = 0;
    for (int i0 = begin; i0 < end; i0 += kThreads) {
        const int i = i0 + tid;
        const uint64_t key = i < end ? ordered64(scores[i]) & mask : 0;
        const bool same = i < end && key == prefix;
        bool take = i < end && key > prefix;
        const uint32_t ties = __ballot_sync(0xffffffffu, same);
        __syncthreads();
        if (lane == 0) s_warp[warp] = __popc(ties);
        __syncthreads();
        int before = equal;
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) before += s_warp[w];
            equal += s_warp[w];
        }
        if (same && (!tied || before + __popc(ties & ((1u << lane) - 1)) < need)) take = true;
        const uint32_t taken = __ballot_sync(0xffffffffu, take);
        __syncthreads();
        if (lane == 0) s_warp[warp] = __popc(taken);
        __syncthreads();
        int to = base + __popc(taken & ((1u << lane) - 1));
        for (int w = 0; w < kThreads / 32; ++w) {
            if (w < warp) to += s_warp[w];
            base += s_warp[w];
        }
        if (take) out[to] = __ldg(table + i);
    }
}

bool bad_type(int dtype) { return dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16; }
constexpr int kMostKeys = 1 << 30;        // tokens a table may hold

}  // namespace

extern "C" {

int qmv_kv_bounds(const qmv_kv_cache* cache, const int* tables, int table_width, const int* lens, const int* starts, int n_seq,
                  int max_new, void* bounds, void* stream) {
    BoxParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!tables || !lens || !bounds) return ST_NULL;
    if (table_width <= 0 || table_width > kMostKeys >> P.c.page_shift) return ST_BAD_SHAPE;
    if (n_seq <= 0 || n_seq > 65535 || max_new <= 0) return ST_BAD_TOKENS;
    if (!aligned(tables, 4) || !aligned(lens, 4) || !aligned(starts, 4) || !aligned(bounds, 16)) return ST_BAD_ALIGN;
    if (!starts) max_new = 1;
    P.bounds = static_cast<__half*>(bounds), P.tables = tables, P.lens = lens, P.starts = starts;
    P.width = table_width, P.n_seq = n_seq;
    P.most = int(std::min<long long>(table_width, ((long long)max_new + P.c.page() - 1) >> P.c.page_shift));
    P.status = device_status_ptr();
    const long long ctas = ((long long)n_seq * P.most * P.c.n_kv + kThreads / 32 - 1) / (kThreads / 32);
    if (ctas > 0x7FFFFFFFLL) return ST_BAD_TOKENS;
    auto go = [&](auto j) {
        constexpr int J = decltype(j)::value;
        return P.c.kb == 4 ? launch_pdl(box_kernel<J, 4>, dim3(unsigned(ctas)), dim3(kThreads), static_cast<cudaStream_t>(stream), P)
                           : launch_pdl(box_kernel<J, 8>, dim3(unsigned(ctas)), dim3(kThreads), static_cast<cudaStream_t>(stream), P);
    };
    switch (P.c.J) {
    case 2: return go(std::integral_constant<int, 2>{});
    case 3: return go(std::integral_constant<int, 3>{});
    case 4: return go(std::integral_constant<int, 4>{});
    case 8: return go(std::integral_constant<int, 8>{});
    }
    return ST_BAD_SHAPE;
}

int64_t qmv_kv_choose_workspace_bytes(const qmv_kv_cache* cache, int table_width, long long n_rows, int keep) {
    KvView c{};
    if (kv_view(cache, c) || table_width <= 0 || table_width > kMostKeys >> c.page_shift || n_rows <= 0 || n_rows > 65535 || keep <= 0) return 0;
    return table_width <= keep ? 8 : 8LL * n_rows * c.n_kv * table_width;
}

int qmv_kv_choose(const qmv_kv_cache* cache, const void* q, int dtype, long long q_stride, int n_heads, const void* bounds,
                  const int* tables, int table_width, const int* lens, const int* starts, int n_seq, long long n_rows, int keep, int first,
                  int last, int* chosen, int* held, void* workspace, long long workspace_bytes, void* stream) {
    KvView c{};
    const int st = kv_view(cache, c);
    if (st) return st;
    if (!q || !bounds || !tables || !lens || !chosen || !held || !workspace) return ST_NULL;
    if (bad_type(dtype) || n_heads <= 0 || n_heads > 65535 || n_heads % c.n_kv || n_heads / c.n_kv > 64) return ST_BAD_SHAPE;
    if (table_width <= 0 || table_width > kMostKeys >> c.page_shift) return ST_BAD_SHAPE;
    if (n_seq <= 0 || n_seq > 65535 || n_rows < 0 || n_rows > 65535 || (!starts && n_rows < n_seq)) return ST_BAD_TOKENS;
    if (first < 0 || last < 1 || keep <= 0 || (long long)first + last > keep || keep > kMostKeys >> c.page_shift) return ST_BAD_SHAPE;
    if (q_stride < (long long)n_heads * c.dim) return ST_BAD_SHAPE;
    if (!aligned(q, 4 * elem_bytes(dtype)) || q_stride % 4 || !aligned(bounds, 16) || !aligned(tables, 4) || !aligned(lens, 4) || !aligned(starts, 4) ||
        !aligned(chosen, 4) || !aligned(held, 4) || !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    if (n_rows == 0) return ST_OK;
    if (workspace_bytes < qmv_kv_choose_workspace_bytes(cache, table_width, n_rows, keep)) return ST_BAD_SHAPE;
    ChooseParams P{};
    P.q = q, P.q_stride = q_stride, P.bounds = static_cast<const __half*>(bounds), P.n_pages = c.n_pages;
    P.tables = tables, P.lens = lens, P.starts = starts;
    P.n_kv = c.n_kv, P.group = n_heads / c.n_kv, P.width = table_width, P.shift = c.page_shift, P.n_seq = n_seq, P.n_rows = int(n_rows);
    P.keep = keep, P.first = first, P.last = last;
    P.scores = static_cast<double*>(workspace), P.chosen = chosen, P.held = held;
    P.status = device_status_ptr();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int middle = table_width - first - last;                // pages to score, at most
    if (table_width > keep && middle > 0) {
        const dim3 grid((middle + kPagesCta - 1) / kPagesCta, c.n_kv, unsigned(n_rows));
        const size_t smem = size_t((P.group + 3) / 4 * 4) * c.dim * 8;
        auto go = [&](auto dt, auto j) {
            constexpr int DT = decltype(dt)::value, J = decltype(j)::value;
            static SmemGrant grant;
            if (const int e = grant(score_kernel<DT, J>, 64 * 256 * 8)) return e;
            return launch_pdl_smem(score_kernel<DT, J>, grid, dim3(kThreads), smem, s, P);
        };
        const int e = by_elem(dtype, [&](auto dt) {
            switch (c.J) {
            case 2: return go(dt, std::integral_constant<int, 2>{});
            case 3: return go(dt, std::integral_constant<int, 3>{});
            case 4: return go(dt, std::integral_constant<int, 4>{});
            case 8: return go(dt, std::integral_constant<int, 8>{});
            }
            return int(ST_BAD_SHAPE);
        });
        if (e) return e;
    }
    return launch_behind(choose_kernel, dim3(unsigned(n_rows * c.n_kv)), dim3(kThreads), s, P);
}

}  // extern "C"
