// Beam search's choice over the beams and the vocabulary (C-ABI declarations: include/nemicli_qmv.h).
//
//   s[k][v] = scores[k] + x[k][v] - max_k - log sum_v exp(x[k][v] - max_k);   the n largest of a request's K V, the lowest
//   k V + v first among equals
//
// A beam whose score is -inf or NaN has -inf throughout, so its part is its first places, whatever its logits.
//
// One pass over the logits: a beam's order is that of its logits, so each part of a row gives its n best, its largest logit and its
// sum of exponentials, and a second launch joins the parts, with logarithm and scores in fp64 (candidates of different beams may lie
// nearer than fp32 tells apart).  Bound by reading the logits: at the HBM's rate an SM sees 12 bf16 values a clock, and of exponentials it
// makes 16.  So candidates must cost nothing on the way: a lane notes the largest of its values of each step, which the softmax needs anyway,
// and behind the last step a bound that n values reach leaves a few of these to be read again (looked for on the way they took twice the
// instructions).  512 rows of 128256 bf16 logits, 16 candidates of 64 x 8 beams: 40.9 us both kernels (floor 20.1); without the look at the
// candidates 35.5, without exponentials too 27.  4 rows of fp32 logits: 10.9 to 11.4, of which the join 4.6.
#include <algorithm>
#include <climits>

#include "qmv_kv.cuh"

using namespace qmv;

namespace {

constexpr int kThreads = 256, kWarps = kThreads / 32;
constexpr int kResident = 4;              // CTAs an SM
constexpr int kStep = 8192, kSteps = 16;  // values of a CTA's step, steps of a part
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

// 16 bytes of logits
template <int DT> struct Piece {
    static constexpr int N = 16 / elem_bytes(DT);
    static __device__ __forceinline__ float get(const uint4& w, int i) {
        if constexpr (DT == QMV_OUT_F32) {
            return __uint_as_float((&w.x)[i]);
        } else if constexpr (DT == QMV_OUT_BF16) {
            const uint32_t v = (&w.x)[i / 2];
            return __uint_as_float(i & 1 ? v & 0xFFFF0000u : v << 16);
        } else {
            const __half2 h = *reinterpret_cast<const __half2*>(&(&w.x)[i / 2]);
            return i & 1 ? __high2float(h) : __low2float(h);
        }
    }
    // the largest of a piece's values; NaN only where all are
    static __device__ __forceinline__ float top(const uint4& w) {
        if constexpr (DT == QMV_OUT_F32) {
            return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
        } else if constexpr (DT == QMV_OUT_BF16) {
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&w.x);
            const __nv_bfloat162 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(__low2float(m), __high2float(m));
        } else {
            const __half2* h = reinterpret_cast<const __half2*>(&w.x);
            const __half2 m = __hmax2(__hmax2(h[0], h[1]), __hmax2(h[2], h[3]));
            return fmaxf(__low2float(m), __high2float(m));
        }
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
// the lanes' values from the largest down (bitonic exchange)
__device__ __forceinline__ float sorted_down(float x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int k = 2; k <= 32; k *= 2)
#pragma unroll
        for (int j = k / 2; j; j /= 2) {
            const float y = __shfl_xor_sync(0xffffffffu, x, j);
            x = ((lane & j) == 0) == ((lane & k) == 0) ? fmaxf(x, y) : fminf(x, y);
        }
    return x;
}

// A CTA takes a part of a row: pieces of 16 bytes, U in flight a lane; counted from the row's start whatever its alignment (a shifted row puts
// each piece together from two), so equal rows have equal sums to the last bit and their candidates tie.
// (x - top before the product with log2 e, not a fused x log2 e - c: logits of 1e4 would carry log2 e's own rounding into the sum.)
template <int DT, bool SHIFTED>
__global__ void __launch_bounds__(kThreads, kResident) beam_part_kernel(const __grid_constant__ BeamParams P) {
    using T = typename Elem<DT>::type;
    using Pc = Piece<DT>;
    constexpr int N = Pc::N, U = DT == QMV_OUT_F32 ? 8 : 4, V = U * N;                  // V values a lane and step
    static_assert(V * kThreads == kStep, "splits_of counts in these");
    __shared__ uint64_t s_keys[kWarps][kRoom];
    __shared__ float s_best[kSteps][kThreads];                    // of a lane's pieces of a step the largest value
    __shared__ uint16_t s_found[kWarps][kSteps * 32];              // lanes and steps with candidates
    __shared__ double s_sum[kWarps];
    __shared__ float s_top[kWarps], s_seen[kWarps][32];
    __shared__ int s_count;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, n = P.n;
    if (tid == 0) s_count = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long row = blockIdx.x / P.splits;
    const int split = int(blockIdx.x - row * P.splits);
    const float score = __ldg(P.scores + row);                    // looked at behind the sums: here it would hold up the logits' loads
    const T* x = static_cast<const T*>(P.x) + row * P.stride;
    const int pieces = P.vocab / N, tail = P.vocab - pieces * N;  // the values behind the last whole piece are the first part's
    const int first = int((long long)pieces * split / P.splits), last = int((long long)pieces * (split + 1) / P.splits);
    const int off = SHIFTED ? int(reinterpret_cast<uintptr_t>(x) & 15) : 0;        // bytes
    const uint4* body = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(x) - off);
    auto load = [&](int p) {
        if constexpr (!SHIFTED) {
            return __ldg(body + p);
        } else {
            // both hold values of the row: the piece ends behind the second one's start (where off is 0 the second is not needed)
            const uint4 a = __ldg(body + p), b = off ? __ldg(body + p + 1) : a;
            const uint32_t w[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
            const int o = off >> 2, bits = 8 * (off & 3);
            uint32_t v[5];
#pragma unroll
            for (int i = 0; i < 5; ++i) v[i] = o == 0 ? w[i] : o == 1 ? w[i + 1] : o == 2 ? w[i + 2] : w[min(i + 3, 7)];
            return make_uint4(__funnelshift_r(v[0], v[1], bits), __funnelshift_r(v[1], v[2], bits), __funnelshift_r(v[2], v[3], bits),
                              __funnelshift_r(v[3], v[4], bits));
        }
    };

    Held H{s_keys[warp], 0};
    uint64_t bound = 0;                   // n values seen are at least this
    float top = -kMost;
    double sum = 0.0;
    if (split == 0 && warp == 0 && tail) {                        // at most 7 values
        const int i = pieces * N + lane;
        const bool there = lane < tail;
        const float v = there ? clean(to_float(x[i])) : -INFINITY;
        if (there) top = fmaxf(v, -kMost), sum = double(ex2((v - top) * kLog2e));
        take(H, n, bound, there ? key_of(v, i) : 0);
    }
    // The bound of all warps: the n-th largest of the lanes' largest so far (of 256, which n values reach); with more than 32 candidates
    // the least of what the warps' lanes all reach.  Each warp's lie in order, the 32 largest of two such lists are the larger ones of one
    // and the other from behind, and seven of these joins are left to each warp.
    float seen = -INFINITY;
    auto tell = [&]() { s_seen[warp][lane] = sorted_down(seen); };
    auto hear = [&]() {
        float m = s_seen[0][lane];
        if (n <= 32) {
#pragma unroll
            for (int w = 1; w < kWarps; ++w) {
                m = fmaxf(m, s_seen[w][31 - lane]);
#pragma unroll
                for (int j = 16; j; j /= 2) {
                    const float y = __shfl_xor_sync(0xffffffffu, m, j);
                    m = lane & j ? fminf(m, y) : fmaxf(m, y);
                }
            }
            m = __shfl_sync(0xffffffffu, m, n - 1);
        } else {
#pragma unroll
            for (int w = 1; w < kWarps; ++w) m = fminf(m, s_seen[w][lane]);
            m = __shfl_sync(0xffffffffu, m, 31);
        }
        if (m > -INFINITY) bound = max(bound, uint64_t(ordered(fminf(m, kMost) + 0.f)) << 32);
        bound = __shfl_sync(0xffffffffu, bound, 0);
    };
    // The candidates of the steps from piece p1 on: a lane's values of a step, read again, where the largest reaches the bound.  They
    // are few (n and some a CTA), so what counts is that their loads go out together.
    auto flush = [&](int p1, int steps) {
        int found = 0;
        // (no value of a lane's step has a larger key than its largest in the first place; none of the lane's one than `seen` in place 0)
        uint32_t lanes = __ballot_sync(0xffffffffu, key_of(seen, 0) >= bound);
        for (; lanes; lanes &= lanes - 1) {
            const int l = __ffs(lanes) - 1, p = p1 + lane * (32 * U * kWarps) + l;
            const uint32_t who = __ballot_sync(0xffffffffu, lane < steps && p < last && key_of(s_best[lane & (kSteps - 1)][32 * warp + l], p * N) >= bound);
            if (who >> lane & 1) s_found[warp][found + __popc(who & ((1u << lane) - 1))] = uint16_t(32 * lane + l);
            found += __popc(who);
        }
        __syncwarp();
        constexpr int kLoads = 4;
        for (int i = 0; i < found; i += kLoads) {
            uint64_t key[kLoads];
#pragma unroll
            for (int y = 0; y < kLoads; ++y) {
                key[y] = 0;
                if (i + y >= found) continue;
                const int at = s_found[warp][i + y], p0 = p1 + (at >> 5) * (32 * U * kWarps), p = p0 + 32 * (lane / N) + (at & 31), place = p * N + lane % N;
                // (since the list was made the bound may have passed all of them)
                if (key_of(s_best[at >> 5][32 * warp + (at & 31)], (p0 + (at & 31)) * N) < bound) continue;
                if (lane < V && p < last) key[y] = key_of(to_float(x[place]), place);
            }
#pragma unroll
            for (int y = 0; y < kLoads; ++y)
                if (i + y < found) take(H, n, bound, key[y]);
        }
        __syncwarp();
    };
    const int begin = first + 32 * U * warp;
    int step = 0;                                                 // (at most kSteps: splits_of)
    for (int p0 = begin; p0 < last; p0 += 32 * U * kWarps) {
        uint4 w[U];
        float best = -INFINITY;
        constexpr uint32_t none = DT == QMV_OUT_F32 ? 0xFF800000u : DT == QMV_OUT_BF16 ? 0xFF80FF80u : 0xFC00FC00u;      // -inf
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + 32 * u + lane;
            w[u] = make_uint4(none, none, none, none);
            if (p < last) w[u] = load(p);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) best = fmaxf(best, Pc::top(w[u]));
        if (best > top) {
            const float m = fminf(best, kMost);
            sum *= double(ex2((top - m) * kLog2e));
            top = m;
        }
        float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int i = 0; i < N; ++i) part[i & 3] += ex2((Pc::get(w[u], i) - top) * kLog2e);
        float all = (part[0] + part[1]) + (part[2] + part[3]);
        if (!(all < 3e38f)) {                                     // a NaN or an infinity among them
            all = 0.f;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int i = 0; i < N; ++i) all += ex2((clean(Pc::get(w[u], i)) - top) * kLog2e);
        }
        sum += double(all);
        seen = fmaxf(seen, best);
        s_best[step][tid] = best;
        ++step;
    }
    if (!(score > -INFINITY)) {                                   // all of the beam's candidates are -inf: the first places (the whole CTA)
        uint64_t* out = P.keys + (long long)blockIdx.x * n;
        for (int i = tid; i < n; i += kThreads) out[i] = split == 0 && i < P.vocab ? key_of(-INFINITY, i) : 0;
        if (tid == 0) P.sums[blockIdx.x] = 1.0, P.tops[blockIdx.x] = -kMost;
        return;
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
    if (lane == 0) s_sum[warp] = sum, s_top[warp] = top;
    tell();
    __syncthreads();
    hear();
    flush(begin, step);
    __syncthreads();
    uint64_t* s_list = reinterpret_cast<uint64_t*>(s_best);
    static_assert(sizeof(s_best) >= sizeof(s_keys), "room for every key");
    for (int i = lane; i < H.count; i += 32)
        if (H.keys[i] >= bound) s_list[atomicAdd(&s_count, 1)] = H.keys[i];
    __syncthreads();
    uint64_t* out = P.keys + (long long)blockIdx.x * n;
    const int total = s_count;
    for (int i = total + tid; i < n; i += kThreads) out[i] = 0;
    for (int i = tid; i < total; i += kThreads) {
        const uint64_t key = s_list[i];
        int rank = 0;
        for (int j = 0; j < total; ++j) rank += s_list[j] > key;
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

// Joins a request's parts: K * splits lists of n.  Candidates are ordered by score, then by the lower beam, then as in their beam's lists: by
// the larger logit (fp64 does not tell logits apart beside a score of 1e30), then by the lower place.
struct Cand {
    uint64_t score, key;                  // ordered64; key_of
    int beam;
};

constexpr int kJoin = 1024, kList = 1024;

// A CTA a request.  The lists are in order, so n candidates reach the r-th largest of their q-th entries, q r >= n: the largest of these for
// q = 1, 2, 4 ... is a limit that a few more than n pass (compared as floats: rounding keeps the order).  Each of those finds its rank by
// looking at all others, four threads a candidate.
__global__ void __launch_bounds__(kJoin) beam_join_kernel(const __grid_constant__ BeamParams P) {
    __shared__ double s_off[kMostBest], s_score[kMostBest];        // of a beam: largest logit; score - log of the sum
    __shared__ uint64_t s_cand[kList], s_key[kList];              // ordered64 of the score; key_of
    __shared__ uint8_t s_beam[kList];
    __shared__ __align__(16) float s_entry[kList];                // [level][list]
    __shared__ int s_count;
    __shared__ uint32_t s_limit;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, req = blockIdx.x, n = P.n, lists = P.K * P.splits, all = lists * n, per = P.splits * n;
    const uint64_t* keys = P.keys + (long long)req * all;
    const uint64_t first = tid < all ? keys[tid] : 0;             // on its way while the sums are made
    for (int k = tid >> 5; k < P.K; k += kJoin / 32) {            // a warp a beam
        const long long r = ((long long)req * P.K + k) * P.splits;
        float m = -kMost;
        for (int i = lane; i < P.splits; i += 32) m = fmaxf(m, P.tops[r + i]);
#pragma unroll
        for (int o = 16; o; o /= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        double sum = 0.0;
        for (int i = lane; i < P.splits; i += 32) sum += P.sums[r + i] * double(ex2((P.tops[r + i] - m) * kLog2e));
#pragma unroll
        for (int o = 16; o; o /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_off[k] = double(m);
            s_score[k] = double(P.scores[(long long)req * P.K + k]) - log(max(sum, 1e-300));
        }
    }
    if (tid == 0) s_count = 0, s_limit = 0;
    __syncthreads();
    auto score = [&](int i, uint64_t key) {
        const int k = i / per;
        const double s = (double(unordered(uint32_t(key >> 32))) - s_off[k]) + s_score[k];
        return s == s ? s + 0.0 : -INFINITY;
    };
    // ---- the limit
    const int padded = (lists + 3) & ~3;
    int levels = 0;
    while (1 << levels <= n && (levels + 1) * padded <= kList) ++levels;
    for (int i = tid; i < levels * padded; i += kJoin) s_entry[i] = -INFINITY;
    __syncthreads();
    for (int i = tid; i < all; i += kJoin) {
        const int list = i / n, q = i - list * n + 1, level = 31 - __clz(q);
        const uint64_t key = i == tid ? first : keys[i];
        if ((q & (q - 1)) == 0 && level < levels && key) s_entry[level * padded + list] = float(score(i, key));
    }
    __syncthreads();
    for (int i = tid; i < levels * padded; i += kJoin) {
        const int level = i / padded, r = (n + (1 << level) - 1) >> level;
        const float mine = s_entry[i];
        int more = 0, equal = 0;
        for (int j = 0; j < padded; j += 4) {
            const float4 o = *reinterpret_cast<const float4*>(s_entry + level * padded + j);
            more += (o.x > mine) + (o.y > mine) + (o.z > mine) + (o.w > mine);
            equal += (o.x == mine) + (o.y == mine) + (o.z == mine) + (o.w == mine);
        }
        if (more < r && r <= more + equal) atomicMax(&s_limit, ordered(mine));
    }
    __syncthreads();
    const uint32_t limit = s_limit;                               // (-inf and nothing: every candidate passes)
    // ---- the ones that reach it.  Where more than the list holds do (scores alike): in turns, of which the n best are kept
    for (int done = 0, turn = all; done < all;) {
        const int kept = s_count;
        __syncthreads();
        for (int i = done + tid; i < min(all, done + turn); i += kJoin) {
            const uint64_t key = i == tid ? first : keys[i];
            if (!key) continue;
            const double s = score(i, key);
            if (ordered(float(s) + 0.f) < limit) continue;
            const int at = atomicAdd(&s_count, 1);
            if (at < kList) s_cand[at] = ordered64(s), s_key[at] = key, s_beam[at] = uint8_t(i / per);
        }
        __syncthreads();
        const int count = s_count;
        if (count > kList) {                                      // (only where turn is all)
            __syncthreads();
            if (tid == 0) s_count = kept;
            turn = kList - n;
            __syncthreads();
            continue;
        }
        done += turn;
        Cand own[4];
        int rank[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            const int i = kJoin / 4 * x + tid / 4;
            rank[x] = kList;
            if (kJoin / 4 * x >= count) continue;
            int r = 0;
            if (i < count) {
                own[x] = Cand{s_cand[i], s_key[i], s_beam[i]};
                for (int j = lane & 3; j < count; j += 4) {
                    const uint64_t o = s_cand[j];
                    if (o > own[x].score) ++r;
                    else if (o == own[x].score) r += s_beam[j] < own[x].beam || (s_beam[j] == own[x].beam && s_key[j] > own[x].key);
                }
            }
            r += __shfl_xor_sync(0xffffffffu, r, 1);
            r += __shfl_xor_sync(0xffffffffu, r, 2);
            if (i < count && (lane & 3) == 0) rank[x] = r;
        }
        if (done >= all) {
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (rank[x] < n) {
                    const uint64_t o = own[x].score;
                    const long long at = (long long)req * n + rank[x];
                    P.scores_out[at] = float(__longlong_as_double(o >> 63 ? o & 0x7FFFFFFFFFFFFFFFull : ~o));
                    P.parents[at] = own[x].beam;
                    P.tokens[at] = int(~uint32_t(own[x].key));
                }
            return;
        }
        __syncthreads();
#pragma unroll
        for (int x = 0; x < 4; ++x)
            if (rank[x] < n) s_cand[rank[x]] = own[x].score, s_key[rank[x]] = own[x].key, s_beam[rank[x]] = uint8_t(own[x].beam);
        if (tid == 0) s_count = min(count, n);
        __syncthreads();
    }
}

// Parts a row: as many as make the fewest steps, with three steps' time for a CTA's start and end, over the CTAs that are resident
// together, and no part longer than kSteps.  (512 rows of 128256: one part, 16 steps, one round of CTAs: 40.9 us; two parts, two rounds of 8
// steps 42.3, three 47.0.  4 rows: 16 parts 10.9, three 13.0, two 14.5.)
int splits_of(int n_req, int K, int vocab) {
    const long long rows = (long long)n_req * K, room = (long long)kResident * sm_count();
    const int steps = (vocab + kStep - 1) / kStep, least = (steps + kSteps - 1) / kSteps;
    long long best = least, cost = LLONG_MAX;
    for (long long s = least; s <= std::min<long long>(steps, least + 1024); ++s) {
        const long long c = (rows * s + room - 1) / room * ((steps + s - 1) / s + 3);
        if (c < cost) cost = c, best = s;
    }
    return int(best);
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
    const bool shifted = !aligned(logits, 16) || row_stride * elem_bytes(dtype) % 16;
    const int e = by_elem(dtype, [&](auto c) {
        constexpr int DT = decltype(c)::value;
        return shifted ? launch_pdl(beam_part_kernel<DT, true>, dim3(unsigned(parts)), dim3(kThreads), st, P)
                       : launch_pdl(beam_part_kernel<DT, false>, dim3(unsigned(parts)), dim3(kThreads), st, P);
    });
    if (e) return e;
    return launch_behind(beam_join_kernel, dim3(n_req), dim3(kJoin), st, P);
}

}  // extern "C"
