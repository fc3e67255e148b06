// Page tables of a paged cache on the device: a step's slots from request lengths, pages given back, the tables of beams
// that part and join (C-ABI declarations: include/nemicli_qmv.h).  Pages come from a stack: free[0 .. counts[0]), the last first.
//
// Whole numbers and a few kilobytes: bound by latency, that is by launches and by dependent reads.  So plan and release are one
// launch, in which every CTA makes the sums over the sequences again (they lie in L2) and takes its share of the rows.  No atomics:
// every place follows from the sums, and the same call gives the same numbers.
#include <algorithm>

#include "qmv_host.cuh"
#include "../../include/nemicli_qmv.h"

using namespace qmv;

namespace {

constexpr int kThreads = 256, kPer = 4, kChunk = kThreads * kPer;    // sequences looked at together
constexpr int kMostSeqs = 65535, kMostTokens = 1 << 30;              // sequences, tokens a table may hold

// exclusive sums over the CTA's threads; total: of all
template <int THREADS = kThreads>
__device__ __forceinline__ long long block_sums(long long x, long long* s_warp, long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    long long inc = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const long long y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();                                              // s_warp may still be read
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    total = 0;
    long long before = 0;
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += s_warp[w];
        total += s_warp[w];
    }
    return before + inc - x;
}
// the last i of 0 .. n - 1 with start[i] <= x (start ascending, start[0] <= x)
template <class T>
__device__ __forceinline__ int last_at(const T* start, int n, T x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (start[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ void report(int* status) {
    if (status) atomicOr(status, DEV_BAD_ADDRESS);
}

struct PlanParams {
    const int* lens;                      // [n_seq] tokens held
    const int* add;                       // [n_seq] new ones (plan)
    const uint8_t* done;                  // [n_seq] (release)
    int* tables;                          // [n_seq][width]
    int* free;                            // [n_pages]
    const int* counts;                    // free pages, pages missing so far
    int n_pages, n_seq, width, shift;
    int rows;
    long long* slots;                     // [rows]
    long long* positions;
    int* starts;                          // [n_seq + 1]
    int* lens_out;
    int* counts_out;
    int* status;
};

template <bool RELEASE>
__global__ void __launch_bounds__(kThreads) plan_kernel(const __grid_constant__ PlanParams P) {
    __shared__ long long s_row[kChunk], s_page[kChunk], s_warp[kThreads / 32];
    __shared__ int s_held[kChunk], s_had[kChunk];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, cap = P.width << P.shift;
    const long long mine = (long long)blockIdx.x * kThreads + tid, all = (long long)gridDim.x * kThreads;
    const int given = __ldg(P.counts), n_free = min(max(given, 0), P.n_pages);
    if (mine == 0 && given != n_free) report(P.status);
    // Where pages were asked for in vain, tables may hold entries of -1, which are no pages to give back: then the entries are
    // counted, a warp a sequence, by every CTA (else only lengths are read: 4.4 us for a quarter of 1021 sequences of up to 512 pages, counted 50,
    // for all of them 6.1 and 118).
    const bool holes = RELEASE && __ldg(P.counts + 1) != 0;
    const int lane = tid & 31, warp = tid >> 5;
    auto entry = [&](int b, int i, int had) { return i < had ? __ldg(P.tables + (long long)b * P.width + i) : -1; };
    long long row0 = 0, page0 = 0;                                // rows and pages of the sequences before this chunk
    for (int b0 = 0, turn = 0; b0 < P.n_seq; b0 += kChunk, ++turn) {
        int held[kPer], take[kPer], need[kPer];
        const int here = min(kChunk, P.n_seq - b0);
        long long rows = 0, pages = 0;
        const bool writes = turn % gridDim.x == blockIdx.x;       // this CTA writes the chunk's lengths
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int b = b0 + tid * kPer + i;
            held[i] = take[i] = need[i] = 0;
            if (b >= P.n_seq) continue;
            const int len = __ldg(P.lens + b);
            held[i] = min(max(len, 0), cap);
            const int had = (held[i] + (1 << P.shift) - 1) >> P.shift;
            bool odd = held[i] != len;
            if constexpr (RELEASE) {
                need[i] = P.done[b] ? had : 0;
                if (writes) P.lens_out[b] = P.done[b] ? 0 : held[i];
            } else {
                const int add = __ldg(P.add + b);
                take[i] = min(max(add, 0), cap - held[i]);
                odd |= take[i] != add;
                need[i] = ((held[i] + take[i] + (1 << P.shift) - 1) >> P.shift) - had;
                if (writes) P.lens_out[b] = held[i] + take[i];
            }
            if (writes && odd) report(P.status);
            rows += take[i], pages += need[i];
        }
        if (holes) {
            for (int at = warp; at < here; at += kThreads / 32) {
                const int had = P.done[b0 + at] ? (min(max(__ldg(P.lens + b0 + at), 0), cap) + (1 << P.shift) - 1) >> P.shift : 0;
                int n = 0;
                for (int i = lane; i < had; i += 32) {
                    const int page = entry(b0 + at, i, had);
                    n += page >= 0 && page < P.n_pages;
                }
                n = __reduce_add_sync(0xffffffffu, n);
                if (lane == 0) s_had[at] = n;
            }
            __syncthreads();
            pages = 0;
#pragma unroll
            for (int i = 0; i < kPer; ++i) pages += need[i] = b0 + tid * kPer + i < P.n_seq ? s_had[tid * kPer + i] : 0;
        }
        long long n_rows = 0, n_need;
        long long r = RELEASE ? 0 : row0 + block_sums(rows, s_warp, n_rows), p = page0 + block_sums(pages, s_warp, n_need);
#pragma unroll
        for (int i = 0; i < kPer; ++i) {
            const int at = tid * kPer + i;
            s_row[at] = r, s_page[at] = p, s_held[at] = held[i], s_had[at] = (held[i] + (1 << P.shift) - 1) >> P.shift;
            if (!RELEASE && writes && b0 + at < P.n_seq) P.starts[b0 + at] = int(min(r, (long long)P.rows));
            r += take[i], p += need[i];
        }
        __syncthreads();
        if (holes) {
            for (long long at = blockIdx.x * (kThreads / 32) + warp; at < here; at += all / 32) {
                const int had = P.done[b0 + at] ? s_had[at] : 0;
                long long to = n_free + s_page[at];
                for (int i0 = 0; i0 < had; i0 += 32) {
                    const int page = entry(b0 + at, i0 + lane, had);
                    const bool there = page >= 0 && page < P.n_pages;
                    const uint32_t who = __ballot_sync(0xffffffffu, there);
                    const long long spot = to + __popc(who & ((1u << lane) - 1));
                    if (there && spot < P.n_pages) P.free[spot] = page;
                    if (there ? spot >= P.n_pages : page != -1) report(P.status);
                    to += __popc(who);
                }
            }
        }
        // pages that change hands: the e-th of this call
        for (long long e = page0 + mine; e < page0 + n_need && !holes; e += all) {
            const int i = last_at(s_page, here, e), in = int(e - s_page[i]);
            int* row = P.tables + (long long)(b0 + i) * P.width;
            if constexpr (RELEASE) {
                const int page = row[in];
                const bool fits = n_free + e < P.n_pages;         // more pages than there are: one was given back twice
                if (fits) P.free[n_free + e] = page;
                if (!fits || page < 0 || page >= P.n_pages) report(P.status);
            } else {
                int page = e < n_free ? P.free[n_free - 1 - e] : -1;
                if (page < 0 || page >= P.n_pages) page = -1, report(P.status);
                row[s_had[i] + in] = page;
            }
        }
        if constexpr (!RELEASE) {
            for (long long x = row0 + mine; x < row0 + n_rows && x < P.rows; x += all) {
                const int i = last_at(s_row, here, x), pos = s_held[i] + int(x - s_row[i]), at = pos >> P.shift;
                const long long e = s_page[i] + at - s_had[i];    // its page: held already, or the e-th of this call
                int page;
                if (at < s_had[i]) page = __ldg(P.tables + (long long)(b0 + i) * P.width + at);
                else page = e < n_free ? __ldg(P.free + n_free - 1 - e) : -1;
                const bool there = page >= 0 && page < P.n_pages;
                if (!there) report(P.status);
                P.slots[x] = there ? ((long long)page << P.shift) + (pos & ((1 << P.shift) - 1)) : -1;
                P.positions[x] = pos;
            }
        }
        row0 += n_rows, page0 += n_need;
        __syncthreads();
    }
    if constexpr (!RELEASE) {
        for (long long x = row0 + mine; x < P.rows; x += all) P.slots[x] = -1, P.positions[x] = 0;
        if (mine == 0) {
            P.starts[P.n_seq] = int(min(row0, (long long)P.rows));
            if (row0 > P.rows) report(P.status);
        }
    }
    if (mine == 0) {
        const long long n = RELEASE ? n_free + page0 : n_free - page0;
        P.counts_out[0] = int(min(max(n, 0LL), (long long)P.n_pages));
        P.counts_out[1] = P.counts[1] + (n < 0 ? int(min(-n, 0x7FFFFFFFLL - max(P.counts[1], 0))) : 0);
    }
}

// ---- beams -----------------------------------------------------------------------------------------------------

struct ReorderParams {
    const int* parents;                   // [n_req][K] -1: no beam
    const int* lens;                      // [n_req][K]
    const int* tables;                    // [n_req][K][width]
    const int* own;                       // [n_req] leading pages that are not the request's own (or null)
    int* free;
    const int* counts;
    int n_pages, n_req, K, width, shift;
    int* tables_out;
    int* lens_out;
    int* src;                             // [n_req][K] pages to copy, -1: none
    int* dst;
    int* used;                            // tokens of them
    int* counts_out;
    int* freed;                           // workspace: [n_req][K * width] pages that fell free, [n_req][2] how many, how many copies
    int* numbers;
    int* status;
};
constexpr int kMostBeams = 64;

// What a request's beams go on from, in shared memory.
struct Beams {
    int pages[kMostBeams], parent[kMostBeams], len[kMostBeams], end[kMostBeams], copy[kMostBeams], asked[kMostBeams];
    unsigned long long chosen;            // old beams that some new one goes on from
    int wants;                            // copies
};
// Beam j copies its last, partly filled page where that is not the request's own or an earlier beam j' writes to the same one.
__device__ __forceinline__ void read_beams(const ReorderParams& P, int req, Beams& B, bool tell) {
    const int j = threadIdx.x, cap = P.width << P.shift, own = P.own ? __ldg(P.own + req) : 0;
    if (j == 0) B.chosen = 0, B.wants = 0;
    __syncthreads();
    if (j < P.K) {
        const int len = __ldg(P.lens + req * P.K + j), held = min(max(len, 0), cap);
        B.pages[j] = (held + (1 << P.shift) - 1) >> P.shift;
        int parent = __ldg(P.parents + req * P.K + j);
        if (tell && (held != len || parent < -1 || parent >= P.K)) report(P.status);
        if (parent < 0 || parent >= P.K) parent = -1;
        B.parent[j] = parent;
        int from = 0;
        if (parent >= 0) {
            atomicOr(&B.chosen, 1ull << parent);
            from = min(max(__ldg(P.lens + req * P.K + parent), 0), cap);
        }
        B.len[j] = from;
        B.end[j] = (from & ((1 << P.shift) - 1)) ? __ldg(P.tables + (long long)(req * P.K + parent) * P.width + (from >> P.shift)) : -1;
    }
    __syncthreads();
    if (j < P.K) {
        bool copy = B.end[j] >= 0 && (B.len[j] >> P.shift) < own;
        for (int o = 0; o < j; ++o) copy |= B.end[j] >= 0 && B.end[o] == B.end[j];
        B.copy[j] = copy;
    }
    __syncthreads();
    if (j < P.K) {
        int before = 0;
        for (int o = 0; o < j; ++o) before += B.copy[o];
        B.asked[j] = before;
        if (j == P.K - 1) B.wants = before + B.copy[j];
    }
    __syncthreads();
}

// Pages that no beam holds any more, in the order of place, then beam.  The beams of a request share a page at the same place of
// their tables only (they part by copies of tables), so a place is looked at alone: a thread an entry, as many whole places as fit the
// CTA, the next ones on their way meanwhile.  (A thread a place, which read the other beams' entries one after the other: 31 us for 16
// requests of 16 beams of 64 pages, both kernels, where this takes 13.6.)
constexpr int kFreers = 1024;
__global__ void __launch_bounds__(kFreers) reorder_free_kernel(const __grid_constant__ ReorderParams P) {
    __shared__ Beams B;
    __shared__ long long s_warp[kFreers / 32];
    __shared__ int s_page[kFreers];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int req = blockIdx.x, tid = threadIdx.x, K = P.K, places = kFreers / K, at = tid / K, k = tid - at * K;
    read_beams(P, req, B, true);
    int most = 0;
    for (int o = 0; o < K; ++o) most = max(most, B.pages[o]);
    const int* table = P.tables + (long long)req * K * P.width;
    int* list = P.freed + (long long)req * K * P.width;
    long long base = 0;
    auto entry = [&](int i) { return at < places && i < B.pages[k] ? __ldg(table + (long long)k * P.width + i) : -1; };
    const int first = P.own ? min(max(__ldg(P.own + req), 0), P.width) : 0;      // (any number there: first + at stays an int)
    int next = entry(first + at);
    for (int i0 = first; i0 < most; i0 += places) {
        const int page = next;
        s_page[tid] = page;
        next = entry(i0 + places + at);
        __syncthreads();
        bool gone = page >= 0 && page < P.n_pages && !(B.chosen >> k & 1);
        if (gone)
            for (int o = 0; o < K; ++o) gone &= !(o != k && (o < k || (B.chosen >> o & 1)) && s_page[at * K + o] == page);
        long long total;
        const long long to = base + block_sums<kFreers>(gone, s_warp, total);
        if (gone) list[to] = page;
        base += total;
    }
    if (tid == 0) P.numbers[2 * req] = int(base), P.numbers[2 * req + 1] = B.wants;
}

// The tables of the next step.  A copy goes to a page of its own request that fell free, in order, or one from the stack, onto which
// all the other freed pages went before.
__global__ void __launch_bounds__(kThreads) reorder_kernel(const __grid_constant__ ReorderParams P) {
    __shared__ Beams B;
    __shared__ long long s_warp[kThreads / 32], s_left[kChunk];
    __shared__ int s_target[kMostBeams];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int req = blockIdx.x, tid = threadIdx.x;
    read_beams(P, req, B, false);
    const int given = __ldg(P.counts), n_free = min(max(given, 0), P.n_pages);
    const int freed = P.numbers[2 * req];
    // pages that other requests leave and lack, the ones before this request and all
    long long left_before = 0, short_before = 0, left = 0, lacks = 0, mine = 0, mine_short = 0;
    for (int g = tid; g < P.n_req; g += kThreads) {
        const int d = P.numbers[2 * g] - P.numbers[2 * g + 1];
        if (g < req) mine += max(d, 0), mine_short += max(-d, 0);
        left += max(d, 0), lacks += max(-d, 0);
    }
    block_sums(mine, s_warp, left_before);
    block_sums(mine_short, s_warp, short_before);
    long long x = left;
    block_sums(x, s_warp, left);
    x = lacks;
    block_sums(x, s_warp, lacks);
    const long long size = n_free + left;
    const int* list = P.freed + (long long)req * P.K * P.width;
    for (int f = B.wants + tid; f < freed; f += kThreads) {
        const long long at = n_free + left_before + f - B.wants;
        if (at < P.n_pages) P.free[at] = list[f];
        else report(P.status);
    }
    // where the copies go: pages of the request, of the stack as it was, or (from >= 0) the from-th that others leave
    long long from = -1;
    if (tid < P.K) {
        int target = -1;
        if (B.copy[tid]) {
            const int a = B.asked[tid];
            const long long s = size - 1 - (short_before + a - freed);
            if (a < freed) target = list[a];
            else if (s >= n_free) from = s - n_free;
            else if (s >= 0) target = __ldg(P.free + s);
        }
        s_target[tid] = target;
    }
    if (__syncthreads_or(from >= 0)) {
        long long base = 0;
        for (int g0 = 0; g0 < P.n_req; g0 += kChunk) {
            long long n[kPer], sum = 0, total;
#pragma unroll
            for (int i = 0; i < kPer; ++i) {
                const int g = g0 + tid * kPer + i;
                n[i] = g < P.n_req ? max(P.numbers[2 * g] - P.numbers[2 * g + 1], 0) : 0;
                sum += n[i];
            }
            long long at = base + block_sums(sum, s_warp, total);
#pragma unroll
            for (int i = 0; i < kPer; ++i) s_left[tid * kPer + i] = at, at += n[i];
            __syncthreads();
            if (from >= base && from < base + total) {
                const int i = last_at(s_left, kChunk, from), g = g0 + i;
                s_target[tid] = P.freed[(long long)g * P.K * P.width + P.numbers[2 * g + 1] + (from - s_left[i])];
            }
            base += total;
            __syncthreads();
        }
    }
    if (tid < P.K) {
        int target = s_target[tid];
        if (B.copy[tid] && (target < 0 || target >= P.n_pages)) target = -1, report(P.status);
        s_target[tid] = target;
        const int at = req * P.K + tid;
        P.lens_out[at] = B.len[tid];
        P.src[at] = B.copy[tid] ? B.end[tid] : -1;
        P.dst[at] = target;
        P.used[at] = B.copy[tid] ? B.len[tid] & ((1 << P.shift) - 1) : 0;
    }
    __syncthreads();
    int* out = P.tables_out + (long long)req * P.K * P.width;
    const int* old = P.tables + (long long)req * P.K * P.width;
#pragma unroll 4
    for (int e = tid; e < P.K * P.width; e += kThreads) {
        const int j = e / P.width, i = e - j * P.width, pages = (B.len[j] + (1 << P.shift) - 1) >> P.shift;
        out[e] = i >= pages ? -1 : B.copy[j] && i == pages - 1 ? s_target[j] : __ldg(old + (long long)B.parent[j] * P.width + i);
    }
    if (req == 0 && tid == 0) {
        if (given != n_free) report(P.status);
        P.counts_out[0] = int(min(max(size - lacks, 0LL), (long long)P.n_pages));
        P.counts_out[1] = P.counts[1] + int(max(lacks - size, 0LL));
    }
}

// The same in one launch for few beams: a warp a request, in a cluster of up to eight CTAs (one SM alone was bound by its own instructions:
// 1400 a warp, 9.2 us for 32 requests), the sums over the requests behind the cluster's barrier.  Bound by dependent reads: lengths and
// parents, the tables, the freed pages.  Calls in a graph: 4 beams of 14 pages 4.0 us (two launches 9.3), 32 requests of
// 8 beams of 21 pages 5.9 (15.4); with more entries a warp walks its request alone (8 x 8 x 130: 15.0, two launches 14.0).
constexpr int kFewReqs = 32, kFewBeams = 8, kFewEntries = 1 << 13;    // requests, beams of each, entries of all tables
__global__ void __launch_bounds__(32 * kFewReqs / 8) reorder_few_kernel(const __grid_constant__ ReorderParams P) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, req = blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5), K = P.K, cap = P.width << P.shift, tokens = 1 << P.shift;
    const bool here = req < P.n_req;                              // (warps behind the last request only meet the barrier)
    const int given = __ldg(P.counts), n_free = min(max(given, 0), P.n_pages);
    // ---- lane j: beam j
    const bool live = here && lane < K;
    const int own = here && P.own ? max(__ldg(P.own + req), 0) : 0;
    const int len = live ? __ldg(P.lens + req * K + lane) : 0, held = min(max(len, 0), cap), pages = (held + tokens - 1) >> P.shift;
    int parent = live ? __ldg(P.parents + req * K + lane) : -1;
    if (held != len || parent < -1 || parent >= K) report(P.status);
    if (parent >= K) parent = -1;
    const uint32_t chosen = __reduce_or_sync(0xffffffffu, parent >= 0 ? 1u << parent : 0u);
    const int from = __shfl_sync(0xffffffffu, held, max(parent, 0)), mine = parent >= 0 ? from : 0;
    const int* table = P.tables + (long long)req * K * P.width;
    const int end = mine & (tokens - 1) ? __ldg(table + (long long)parent * P.width + (mine >> P.shift)) : -1;
    bool copy = end >= 0 && (mine >> P.shift) < own;
#pragma unroll
    for (int o = 0; o < kFewBeams - 1; ++o) {
        const int other = __shfl_sync(0xffffffffu, end, o);       // (by all lanes)
        copy |= lane > o && end >= 0 && other == end;
    }
    const uint32_t copies = __ballot_sync(0xffffffffu, copy);
    const int asked = copy ? __popc(copies & ((1u << lane) - 1)) : -1, wants = __popc(copies);
    int n[kFewBeams];                                             // pages of the old beams
#pragma unroll
    for (int k = 0; k < kFewBeams; ++k) n[k] = __shfl_sync(0xffffffffu, pages, k);       // (0 from K on)
    // ---- pages that no beam holds any more, a place a lane
    const int most = __reduce_max_sync(0xffffffffu, pages);
    int* list = P.freed + (long long)req * K * P.width;
    int freed = 0;
    for (int i0 = own; i0 < most; i0 += 32) {
        const int i = i0 + lane;
        int at[kFewBeams];
#pragma unroll
        for (int k = 0; k < kFewBeams; ++k) at[k] = i < n[k] ? __ldg(table + (long long)k * P.width + i) : -1;
        uint32_t gone = 0;
#pragma unroll
        for (int k = 0; k < kFewBeams; ++k) {
            bool kept = at[k] < 0 || at[k] >= P.n_pages || (chosen >> k & 1);
#pragma unroll
            for (int o = 0; o < kFewBeams; ++o)
                if (o != k) kept |= (o < k || (chosen >> o & 1)) && at[o] == at[k];
            gone |= (kept ? 0u : 1u) << k;
        }
        int inc = __popc(gone);
#pragma unroll
        for (int o = 1; o < 32; o *= 2) {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        int to = freed + inc - __popc(gone);
#pragma unroll
        for (int k = 0; k < kFewBeams; ++k)
            if (gone >> k & 1) list[to++] = at[k];
        freed += __shfl_sync(0xffffffffu, inc, 31);
    }
    if (here && lane == 0) P.numbers[2 * req] = freed, P.numbers[2 * req + 1] = wants;
    // every CTA's numbers and lists are written before any is read
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (!here) return;
    // ---- what the requests leave and lack, a request a lane, summed up
    const int2 its = lane < P.n_req ? __ldcg(reinterpret_cast<const int2*>(P.numbers) + lane) : make_int2(0, 0);
    const int spare = its.x - its.y;
    int left = max(spare, 0), lack = max(-spare, 0);
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int x = __shfl_up_sync(0xffffffffu, left, o), y = __shfl_up_sync(0xffffffffu, lack, o);
        if (lane >= o) left += x, lack += y;
    }
    const int all_left = __shfl_sync(0xffffffffu, left, 31), all_lack = __shfl_sync(0xffffffffu, lack, 31);
    const int left_before = __shfl_sync(0xffffffffu, left, req) - max(freed - wants, 0), lack_before = __shfl_sync(0xffffffffu, lack, req) - max(wants - freed, 0);
    const int size = n_free + all_left;
    for (int f = wants + lane; f < freed; f += 32) {
        const int at = n_free + left_before + f - wants;
        if (at < P.n_pages) P.free[at] = list[f];
        else report(P.status);
    }
    // ---- lane j: where beam j's copy goes
    const int s = size - 1 - (lack_before + asked - freed);
    int other = 0, before = 0, its_wants = 0;                     // the request whose left page that is, those before it, its copies
    if (__any_sync(0xffffffffu, asked >= freed && s >= n_free))
        for (int r = 0; r < P.n_req; ++r) {
            const int up_to = __shfl_sync(0xffffffffu, left, r), w = __shfl_sync(0xffffffffu, its.y, r);
            if (up_to <= s - n_free) other = r + 1, before = up_to;
            else if (other == r) its_wants = w;
        }
    int target = -1;
    if (asked >= 0) {
        if (asked < freed) target = list[asked];
        else if (s >= n_free) target = __ldcg(P.freed + (long long)other * K * P.width + its_wants + s - n_free - before);
        else if (s >= 0) target = __ldg(P.free + s);
        if (target < 0 || target >= P.n_pages) target = -1, report(P.status);
    }
    if (live) {
        const int beam = req * K + lane;
        P.lens_out[beam] = mine;
        P.src[beam] = asked >= 0 ? end : -1;
        P.dst[beam] = target;
        P.used[beam] = asked >= 0 ? mine & (tokens - 1) : 0;
    }
    for (int j = 0; j < K; ++j) {
        const int have = (__shfl_sync(0xffffffffu, mine, j) + tokens - 1) >> P.shift, to = __shfl_sync(0xffffffffu, target, j);
        const int copied = __shfl_sync(0xffffffffu, asked, j), old = __shfl_sync(0xffffffffu, parent, j);
        const int* row = table + (long long)max(old, 0) * P.width;
        int* out = P.tables_out + (long long)(req * K + j) * P.width;
        for (int i = lane; i < P.width; i += 32) out[i] = i >= have ? -1 : copied >= 0 && i == have - 1 ? to : __ldg(row + i);
    }
    if (req == 0 && lane == 0) {
        if (given != n_free) report(P.status);
        P.counts_out[0] = min(max(size - all_lack, 0), P.n_pages);
        P.counts_out[1] = P.counts[1] + max(all_lack - size, 0);
    }
}

// log2 of the tokens a page, or -1
int page_shift(int page) {
    for (int s = 4; s <= 10; ++s)
        if (1 << s == page) return s;
    return -1;
}
bool bad_table(int width, int shift) { return shift < 0 || width <= 0 || width > kMostTokens >> shift; }

int plan_launch(PlanParams& P, bool release, cudaStream_t st) {
    P.status = device_status_ptr();
    // CTAs for the rows, and for the pages that change hands: some a sequence, of those given back up to all, up to two CTAs an SM
    // (1021 sequences that give back 66000 pages: 48 us with a thread a sequence)
    const long long work = release ? (long long)P.n_seq * std::min(P.width, 64) : std::max<long long>(P.rows, P.n_seq);
    const int grid = int(std::min<long long>((work + kThreads - 1) / kThreads, 2LL * sm_count()));
    return release ? launch_pdl(plan_kernel<true>, dim3(grid), dim3(kThreads), st, P)
                   : launch_pdl(plan_kernel<false>, dim3(grid), dim3(kThreads), st, P);
}

}  // namespace

extern "C" {

int qmv_page_plan(const int* lens, const int* add, int* tables, int n_seq, int table_width, int page, const int* free_pages,
                  int n_pages, const int* counts, long long rows, long long* slots, long long* positions, int* starts,
                  int* lens_out, int* counts_out, void* stream) {
    if (!lens || !add || !tables || !free_pages || !counts || !starts || !lens_out || !counts_out) return ST_NULL;
    if (rows > 0 && (!slots || !positions)) return ST_NULL;
    const int shift = page_shift(page);
    if (bad_table(table_width, shift) || n_pages <= 0) return ST_BAD_SHAPE;
    if (n_seq <= 0 || n_seq > kMostSeqs || rows < 0 || rows > kMostTokens) return ST_BAD_TOKENS;
    if (lens_out == lens || counts_out == counts) return ST_BAD_SHAPE;       // read by every CTA while some writes it
    if (!aligned(lens, 4) || !aligned(add, 4) || !aligned(tables, 4) || !aligned(free_pages, 4) || !aligned(counts, 4) || !aligned(slots, 8) ||
        !aligned(positions, 8) || !aligned(starts, 4) || !aligned(lens_out, 4) || !aligned(counts_out, 4))
        return ST_BAD_ALIGN;
    PlanParams P{};
    P.lens = lens, P.add = add, P.tables = tables, P.free = const_cast<int*>(free_pages), P.counts = counts;
    P.n_pages = n_pages, P.n_seq = n_seq, P.width = table_width, P.shift = shift, P.rows = int(rows);
    P.slots = slots, P.positions = positions, P.starts = starts, P.lens_out = lens_out, P.counts_out = counts_out;
    return plan_launch(P, false, static_cast<cudaStream_t>(stream));
}

int qmv_page_release(const uint8_t* done, const int* lens, const int* tables, int n_seq, int table_width, int page, int* free_pages,
                     int n_pages, const int* counts, int* lens_out, int* counts_out, void* stream) {
    if (!done || !lens || !tables || !free_pages || !counts || !lens_out || !counts_out) return ST_NULL;
    const int shift = page_shift(page);
    if (bad_table(table_width, shift) || n_pages <= 0) return ST_BAD_SHAPE;
    if (n_seq <= 0 || n_seq > kMostSeqs) return ST_BAD_TOKENS;
    if (lens_out == lens || counts_out == counts) return ST_BAD_SHAPE;
    if (!aligned(lens, 4) || !aligned(tables, 4) || !aligned(free_pages, 4) || !aligned(counts, 4) || !aligned(lens_out, 4) || !aligned(counts_out, 4))
        return ST_BAD_ALIGN;
    PlanParams P{};
    P.lens = lens, P.done = done, P.tables = const_cast<int*>(tables), P.free = free_pages, P.counts = counts;
    P.n_pages = n_pages, P.n_seq = n_seq, P.width = table_width, P.shift = shift;
    P.lens_out = lens_out, P.counts_out = counts_out;
    return plan_launch(P, true, static_cast<cudaStream_t>(stream));
}

int64_t qmv_page_reorder_workspace_bytes(int n_req, int beams, int table_width) {
    if (n_req <= 0 || beams <= 0 || beams > kMostBeams || n_req > kMostSeqs / beams || table_width <= 0 || table_width > kMostTokens / 16 / beams) return 0;
    return 4LL * n_req * beams * table_width + 8LL * n_req;
}

int qmv_page_reorder(const int* parents, const int* lens, const int* tables, const int* own, int n_req, int beams, int table_width,
                     int page, int* free_pages, int n_pages, const int* counts, int* tables_out, int* lens_out, int* src,
                     int* dst, int* used, int* counts_out, void* workspace, long long workspace_bytes, void* stream) {
    if (!parents || !lens || !tables || !free_pages || !counts || !tables_out || !lens_out || !src || !dst || !used || !counts_out || !workspace)
        return ST_NULL;
    const int shift = page_shift(page);
    if (bad_table(table_width, shift) || n_pages <= 0 || beams <= 0 || beams > kMostBeams || table_width > kMostTokens / 16 / beams) return ST_BAD_SHAPE;
    if (n_req <= 0 || n_req > kMostSeqs / beams) return ST_BAD_TOKENS;
    if (tables_out == tables || lens_out == lens || counts_out == counts) return ST_BAD_SHAPE;
    if (workspace_bytes < qmv_page_reorder_workspace_bytes(n_req, beams, table_width)) return ST_BAD_SHAPE;
    if (!aligned(parents, 4) || !aligned(lens, 4) || !aligned(tables, 4) || !aligned(own, 4) || !aligned(free_pages, 4) || !aligned(counts, 4) ||
        !aligned(tables_out, 4) || !aligned(lens_out, 4) || !aligned(src, 4) || !aligned(dst, 4) || !aligned(used, 4) || !aligned(counts_out, 4) ||
        !aligned(workspace, 256))
        return ST_BAD_ALIGN;
    ReorderParams P{};
    P.parents = parents, P.lens = lens, P.tables = tables, P.own = own, P.free = free_pages, P.counts = counts;
    P.n_pages = n_pages, P.n_req = n_req, P.K = beams, P.width = table_width, P.shift = shift;
    P.tables_out = tables_out, P.lens_out = lens_out, P.src = src, P.dst = dst, P.used = used, P.counts_out = counts_out;
    P.numbers = static_cast<int*>(workspace);
    P.freed = P.numbers + 2LL * n_req;
    P.status = device_status_ptr();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (beams <= kFewBeams && n_req <= kFewReqs && (long long)n_req * beams * table_width <= kFewEntries) {
        const int ctas = std::min(n_req, 8);
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas);
        cfg.blockDim = dim3(32 * ((n_req + ctas - 1) / ctas));
        cfg.stream = s;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas, attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        cudaLaunchKernelEx(&cfg, reorder_few_kernel, P);
        return launched();
    }
    if (const int e = launch_pdl(reorder_free_kernel, dim3(n_req), dim3(kFreers), s, P)) return e;
    return launch_behind(reorder_kernel, dim3(n_req), dim3(kThreads), s, P);
}

}  // extern "C"
