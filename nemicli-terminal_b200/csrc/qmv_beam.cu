// Beam search's choice over the beams and the vocabulary (C-ABI declarations: include/nemicli_qmv.h).
//
//   s[k][v] = scores[k] + x[k][v] - max_k - log sum_v exp(x[k][v] - max_k);   the n largest of a request's K V, the lowest
//   k V + v first among equals
//
// One pass over the logits: a beam's order is that of its logits, so each part of a row gives its n best, its largest logit and its
// sum of exponentials, and a second launch joins the parts, with logarithm and scores in fp64 (candidates of different beams may lie
// nearer than fp32 tells apart).  Bound by reading the logits, 12 lane-instructions a bf16 value at the HBM's rate: the exponential
// costs 8 of them (16 a clock and SM), so candidates must cost nothing: a lane compares the maximum of 16 or 32 values, which the
// softmax needs anyway, with a bound that n values seen so far reach.
#include <algorithm>

#include "qmv_kv.cuh"

using namespace qmv;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kMostBest = 64;             // candidates kept
constexpr int kRoom = 128;                // keys a warp holds before it sorts out: kMostBest + a value of every lane, at least
constexpr float kMost = 3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f;

struct BeamParams {
    const void* x;                        // [rows][vocab], rows stride values apart
    long long stride;
    const float* scores;                  // [n_req][K]
    int vocab, K, n, splits, n_req;
    float* scores_out;                    // [n_req][n]
    int* parents;
    int* tokens;
    uint64_t* keys;                       // workspace: [rows][splits][n], best first
    double* sums;                         // [rows][splits]
    float* tops;
};

// 32 bits that order as the floats do; back
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) { return __uint_as_float(o >> 31 ? o & 0x7FFFFFFFu : ~o); }
__device__ __forceinline__ uint64_t ordered64(double x) {
    const uint64_t b = __double_as_longlong(x);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
// NaN counts as -inf, +inf as the largest float
__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), kMost); }
// a value and its place as one number: larger value, then lower place
__device__ __forceinline__ uint64_t key_of(float x, int place) { return uint64_t(ordered(clean(x) + 0.f)) << 32 | uint32_t(~place); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int DT> struct Piece;           // 16 bytes of logits
template <> struct Piece<QMV_OUT_F32> {
    static constexpr int N = 4;
    static __device__ __forceinline__ float get(const uint4& w, int i) { return __uint_as_float((&w.x)[i]); }
};
template <> struct Piece<QMV_OUT_BF16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float get(const uint4& w, int i) {
        const uint32_t v = (&w.x)[i / 2];
        return __uint_as_float(i & 1 ? v & 0xFFFF0000u : v << 16);
    }
};
template <> struct Piece<QMV_OUT_F16> {
    static constexpr int N = 8;
    static __device__ __forceinline__ float get(const uint4& w, int i) {
        const __half2 h = *reinterpret_cast<const __half2*>(&(&w.x)[i / 2]);
        return i & 1 ? __high2float(h) : __low2float(h);
    }
};

// The best keys of a warp in shared memory: at most kRoom, of which only those from `bound` on can be among the n best.
struct Held {
    uint64_t* keys;
    int count;
};
// keeps the n best, in order
__device__ __forceinline__ void sort_out(Held& H, int n, uint64_t& bound) {
    const int lane = threadIdx.x & 31;
    __syncwarp();
    uint64_t own[kRoom / 32];
    int rank[kRoom / 32];
#pragma unroll
    for (int i = 0; i < kRoom / 32; ++i) own[i] = 32 * i + lane < H.count ? H.keys[32 * i + lane] : 0, rank[i] = 0;
    for (int j = 0; j < H.count; ++j) {
        const uint64_t o = H.keys[j];
#pragma unroll
        for (int i = 0; i < kRoom / 32; ++i) rank[i] += o > own[i];
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < kRoom / 32; ++i)
        if (own[i] && rank[i] < n) H.keys[rank[i]] = own[i];
    __syncwarp();
    H.count = min(H.count, n);
    if (H.count == n) bound = max(bound, H.keys[n - 1]);
}
// takes each lane's key where it reaches the bound (whole warps)
__device__ __forceinline__ void take(Held& H, int n, uint64_t& bound, uint64_t key) {
    uint32_t who = __ballot_sync(0xffffffffu, key >= bound && key);
    if (!who) return;
    if (H.count + __popc(who) > kRoom) {
        sort_out(H, n, bound);
        who = __ballot_sync(0xffffffffu, key >= bound && key);
    }
    if (who >> (threadIdx.x & 31) & 1) H.keys[H.count + __popc(who & ((1u << (threadIdx.x & 31)) - 1))] = key;
    H.count += __popc(who);
}

template <int DT>
__global__ void __launch_bounds__(kThreads) beam_part_kernel(const __grid_constant__ BeamParams P) {
    using T = typename Elem<DT>::type;
    using Pc = Piece<DT>;
    constexpr int N = Pc::N, U = 4;       // pieces in flight
    __shared__ uint64_t s_keys[kWarps][kRoom];
    __shared__ uint64_t s_bound;
    __shared__ double s_sum[kWarps];
    __shared__ float s_top[kWarps];
    __shared__ int s_count[kWarps];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = P.n;
    if (tid == 0) s_bound = 0;
    __syncthreads();
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = blockIdx.x / P.splits;
    const int split = int(blockIdx.x - row * P.splits);
    const T* x = static_cast<const T*>(P.x) + row * P.stride;
    // the row's 16-byte pieces; the values before and behind them are the first part's
    const int head = min(P.vocab, int((16 - (reinterpret_cast<uintptr_t>(x) & 15)) & 15) / int(sizeof(T)));
    const int pieces = (P.vocab - head) / N, tail = P.vocab - head - pieces * N;
    const int first = int((long long)pieces * split / P.splits), last = int((long long)pieces * (split + 1) / P.splits);
    const uint4* body = reinterpret_cast<const uint4*>(x + head);

    Held H{s_keys[warp], 0};
    uint64_t bound = 0;                   // n values seen are at least this
    float top = -kMost;
    double sum = 0.0;
    auto reaches = [&](float m) { return ordered(m) >= uint32_t(bound >> 32); };

    if (split == 0 && warp == 0) {        // at most 14 values
        const int i = lane < head ? lane : P.vocab - tail + lane - head;
        const bool there = lane < head + tail;
        const float v = there ? clean(to_float(x[i])) : -INFINITY;
        if (there) top = fmaxf(v, -kMost), sum = double(ex2((v - top) * kLog2e));
        take(H, n, bound, there ? key_of(v, i) : 0);
    }
    bool primed = false;
    for (int p0 = first + 32 * U * warp; p0 < last; p0 += 32 * U * kWarps) {
        uint4 w[U];
        bool there[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + 32 * u + lane;
            there[u] = p < last;
            w[u] = there[u] ? __ldg(body + p) : make_uint4(0, 0, 0, 0);
        }
        float best = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            float m = -INFINITY;
#pragma unroll
            for (int i = 0; i < N; ++i) m = fmaxf(m, Pc::get(w[u], i));
            best = fmaxf(best, there[u] ? m : -INFINITY);
        }
        if (best > top) {
            best = fminf(best, kMost);
            sum *= double(ex2((top - best) * kLog2e));
            top = best;
        }
        float part = 0.f;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) part += there[u] ? ex2((Pc::get(w[u], i) - top) * kLog2e) : 0.f;
        if (!(part == part) || part > 3e38f) {                    // a NaN or an infinity among them
            part = 0.f;
            for (int u = 0; u < U; ++u)
                for (int i = 0; i < N; ++i) part += there[u] ? ex2((clean(Pc::get(w[u], i)) - top) * kLog2e) : 0.f;
        }
        sum += double(part);
        if (!primed) {
            // the first bound: of 64 maxima (two a lane) the n-th
            primed = true;
            uint64_t two[2] = {0, 0};
            int rank[2] = {0, 0};
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (there[u]) two[u & 1] = max(two[u & 1], key_of(Pc::get(w[u], i), head + (p0 + 32 * u + lane) * N + i));
            for (int o = 0; o < 32; ++o)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint64_t k = __shfl_sync(0xffffffffu, two[h], o);
                    rank[0] += k > two[0], rank[1] += k > two[1];
                }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t who = __ballot_sync(0xffffffffu, two[h] && rank[h] == n - 1);
                if (who) bound = max(bound, __shfl_sync(0xffffffffu, two[h], __ffs(who) - 1));
            }
        }
        bound = max(bound, *static_cast<volatile uint64_t*>(&s_bound));       // the other warps'
        if (__any_sync(0xffffffffu, reaches(best))) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    take(H, n, bound, there[u] ? key_of(Pc::get(w[u], i), head + (p0 + 32 * u + lane) * N + i) : 0);
            if (lane == 0) atomicMax(reinterpret_cast<unsigned long long*>(&s_bound), (unsigned long long)bound);
        }
        bound = __shfl_sync(0xffffffffu, bound, 0);
    }
    // ---- the warps' together
    {
        float m = top;
#pragma unroll
        for (int o = 16; o; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        sum *= double(ex2((top - m) * kLog2e));
#pragma unroll
        for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        top = m;
    }
    if (H.count > n) sort_out(H, n, bound);
    if (lane == 0) s_sum[warp] = sum, s_top[warp] = top, s_count[warp] = H.count;
    __syncthreads();
    uint64_t* out = P.keys + (long long)blockIdx.x * n;
    int total = 0;
    for (int w = 0; w < kWarps; ++w) total += s_count[w];
    for (int i = total + tid; i < n; i += kThreads) out[i] = 0;
    for (int i = tid; i < kWarps * kMostBest; i += kThreads) {
        const int w = i / kMostBest, at = i % kMostBest;
        if (at >= s_count[w]) continue;
        const uint64_t key = s_keys[w][at];
        int rank = 0;
        for (int o = 0; o < kWarps; ++o)
            for (int j = 0; j < s_count[o]; ++j) rank += s_keys[o][j] > key;
        if (rank < n) out[rank] = key;
    }
    if (tid == 0) {
        float m = s_top[0];
        for (int w = 1; w < kWarps; ++w) m = fmaxf(m, s_top[w]);
        double s = 0.0;
        for (int w = 0; w < kWarps; ++w) s += s_sum[w] * double(ex2((s_top[w] - m) * kLog2e));
        P.sums[blockIdx.x] = s, P.tops[blockIdx.x] = m;
    }
}

// Joins a request's parts: K * splits lists of n.  Candidates are numbers (score, place), ordered by score, then by the lower place.
struct Cand {
    uint64_t score;                       // ordered64
    int64_t place;                        // k V + v
};
__device__ __forceinline__ bool before(const Cand& a, const Cand& b) { return a.score > b.score || (a.score == b.score && a.place < b.place); }

constexpr int kList = 1024;

__global__ void __launch_bounds__(kThreads) beam_join_kernel(const __grid_constant__ BeamParams P) {
    __shared__ double s_off[kMostBest], s_score[kMostBest];        // of a beam: largest logit; score - log of the sum
    __shared__ Cand s_list[kList];
    __shared__ int s_count;
    __shared__ Cand s_limit;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, req = blockIdx.x, n = P.n, per = P.splits * n, all = P.K * per;
    if (tid < P.K) {
        const long long r = (long long)req * P.K + tid;
        float m = -kMost;
        for (int s = 0; s < P.splits; ++s) m = fmaxf(m, P.tops[r * P.splits + s]);
        double sum = 0.0;
        for (int s = 0; s < P.splits; ++s) sum += P.sums[r * P.splits + s] * exp(double(P.tops[r * P.splits + s]) - double(m));
        s_off[tid] = double(m);
        s_score[tid] = double(P.scores[r]) - log(max(sum, 1e-300));
    }
    if (tid == 0) s_count = 0, s_limit = Cand{0, INT64_MAX};
    __syncthreads();
    const uint64_t* keys = P.keys + (long long)req * all;
    auto cand = [&](int i) {
        const uint64_t key = keys[i];
        if (!key) return Cand{0, INT64_MAX};                      // none
        const int k = i / per;
        double s = (double(unordered(uint32_t(key >> 32))) - s_off[k]) + s_score[k];
        if (!(s == s)) s = -INFINITY;
        return Cand{ordered64(s + 0.0), (long long)k * P.vocab + int(~uint32_t(key))};
    };
    // with many candidates a limit first: of the threads' best ones the n-th
    if (all > kThreads) {
        Cand best{0, INT64_MAX};
        for (int i = tid; i < all; i += kThreads) {
            const Cand c = cand(i);
            if (before(c, best)) best = c;
        }
        s_list[tid] = best;
        __syncthreads();
        int rank = 0;
        for (int j = 0; j < kThreads; ++j) rank += before(s_list[j], best);
        if (rank == n - 1 && best.place != INT64_MAX) s_limit = best;
        __syncthreads();
    }
    const Cand limit = s_limit;
    // Those that reach it: at most n threads' candidates.  More than the list holds are taken in turns, the n best of each kept.
    int done = 0;                         // candidates looked at, by all threads
    while (done < all) {
        const int end = min(all, done + kList - n);
        for (int i = done + tid; i < end; i += kThreads) {
            const Cand c = cand(i);
            if (c.place != INT64_MAX && !before(limit, c)) s_list[atomicAdd(&s_count, 1)] = c;
        }
        __syncthreads();
        done = end;
        const int count = s_count;
        Cand own[kList / kThreads];
        int rank[kList / kThreads];
#pragma unroll
        for (int i = 0; i < kList / kThreads; ++i) {
            rank[i] = kList;
            if (kThreads * i + tid >= count) continue;
            own[i] = s_list[kThreads * i + tid];
            int r = 0;
            for (int j = 0; j < count; ++j) r += before(s_list[j], own[i]);
            rank[i] = r;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < kList / kThreads; ++i)
            if (rank[i] < n) s_list[rank[i]] = own[i];
        if (tid == 0) s_count = min(count, n);
        __syncthreads();
    }
    for (int i = tid; i < n; i += kThreads) {
        const Cand c = s_list[i];
        const uint64_t o = c.score;
        const double s = __longlong_as_double(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o);
        const long long at = (long long)req * n + i;
        P.scores_out[at] = float(s);
        P.parents[at] = int(c.place / P.vocab);
        P.tokens[at] = int(c.place % P.vocab);
    }
}

// Parts a row: two CTAs an SM over all rows, of 2048 values at least.
int splits_of(int n_req, int K, int vocab) {
    const long long rows = (long long)n_req * K;
    const long long want = (4LL * sm_count() + rows - 1) / rows;
    return int(std::max<long long>(1, std::min<long long>(want, vocab / 2048)));
}
bool bad_sizes(int n_req, int K, int vocab, int n) {
    return n_req <= 0 || K <= 0 || K > kMostBest || n_req > 65535 / K || vocab <= 0 || vocab > (1 << 30) || n <= 0 || n > kMostBest || n > (long long)K * vocab;
}

}  // namespace

extern "C" {

int64_t qmv_beam_workspace_bytes(int n_req, int beams, int vocab, int n) {
    if (bad_sizes(n_req, beams, vocab, n)) return 0;
    return (long long)n_req * beams * splits_of(n_req, beams, vocab) * (8LL * n + 8 + 4);
}

int qmv_beam_select(const void* logits, int dtype, long long row_stride, int n_req, int beams, int vocab, const float* scores, int n,
                    float* scores_out, int* parents, int* tokens, void* workspace, long long workspace_bytes, void* stream) {
    if (!logits || !scores || !scores_out || !parents || !tokens || !workspace) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (bad_sizes(n_req, beams, vocab, n) || row_stride < vocab) return ST_BAD_SHAPE;
    if (workspace_bytes < qmv_beam_workspace_bytes(n_req, beams, vocab, n)) return ST_BAD_SHAPE;
    if (!aligned(logits, elem_bytes(dtype)) || !aligned(scores, 4) || !aligned(scores_out, 4) || !aligned(parents, 4) || !aligned(tokens, 4) ||
        !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    BeamParams P{};
    P.x = logits, P.stride = row_stride, P.scores = scores;
    P.vocab = vocab, P.K = beams, P.n = n, P.n_req = n_req, P.splits = splits_of(n_req, beams, vocab);
    P.scores_out = scores_out, P.parents = parents, P.tokens = tokens;
    const long long parts = (long long)n_req * beams * P.splits;
    P.keys = static_cast<uint64_t*>(workspace);
    P.sums = reinterpret_cast<double*>(P.keys + parts * n);
    P.tops = reinterpret_cast<float*>(P.sums + parts);
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const int e = by_elem(dtype, [&](auto c) { return launch_pdl(beam_part_kernel<decltype(c)::value>, dim3(unsigned(parts)), dim3(kThreads), st, P); });
    if (e) return e;
    return launch_pdl(beam_join_kernel, dim3(n_req), dim3(kThreads), st, P);
}

}  // extern "C"
