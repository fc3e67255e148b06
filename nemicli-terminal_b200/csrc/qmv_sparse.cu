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

// Eight codes of a key times its scale d, exactly: a code's bits below the exponent of 2^e are the float 2^e + code, and
// d (2^e + code) - d (2^e + offset) is one fused multiply-add without a rounding (d has 11 bits, 2^e + offset at most 13).  (Converted
// from integers the codes took 16 a clock and SM: 18 us for the pages of 32000 tokens.)
template <int KB>
__device__ __forceinline__ void keys8(const uint32_t* w, float d, float (&v)[8]) {
    if constexpr (KB == 4) {
        const float d7 = d * -136.f, d11 = d * -2056.f, d15 = d * -32776.f;      // the code at bits 16, 12, 8: 2^7, 2^11, 2^15
        auto at16 = [&](uint32_t x) { return fmaf(d, __uint_as_float((x & 0x000F0000u) | 0x43000000u), d7); };
        auto at12 = [&](uint32_t x) { return fmaf(d, __uint_as_float((x & 0x0000F000u) | 0x45000000u), d11); };
        auto at8 = [&](uint32_t x) { return fmaf(d, __uint_as_float((x & 0x00000F00u) | 0x47000000u), d15); };
        const uint32_t up = w[0] << 8, down = w[0] >> 8;          // value n at bit 16 (n & 1) + 4 (n >> 1)
        v[0] = at8(up), v[2] = at12(up), v[4] = at8(w[0]), v[6] = at12(w[0]);
        v[1] = at16(w[0]), v[3] = at12(down), v[5] = at16(down), v[7] = at16(w[0] >> 12);
    } else {
        const float d15 = d * -32896.f;                           // the code at bit 8: 2^15
#pragma unroll
        for (int i = 0; i < 2; ++i) {                             // bytes n0 n2 n1 n3
            auto at8 = [&](uint32_t x) { return fmaf(d, __uint_as_float((x & 0x0000FF00u) | 0x47000000u), d15); };
            v[4 * i] = at8(w[i] << 8), v[4 * i + 2] = at8(w[i]), v[4 * i + 1] = at8(w[i] >> 8), v[4 * i + 3] = at8(w[i] >> 16);
        }
    }
}

// the words of a lane's run of codes or scales, as wide as they are aligned
template <int N>
__device__ __forceinline__ void load_words(uint32_t (&w)[N], const void* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = __ldg(static_cast<const uint4*>(p) + i / 4);
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = __ldg(static_cast<const uint2*>(p) + i / 2);
            w[i] = x.x, w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __ldg(static_cast<const uint32_t*>(p) + i);
    }
}

// A warp a page and key head; a lane takes run t of C blocks (8 to 24 bytes of codes, C scales) of every kTok-th token, two tokens at a time.
// 500 pages of 64 keys, 8 heads of 128 in Q4_0 (18.5 MB): 10.6 us.  Bound by latency (lengths, table, two rounds of loads) and by the minima
// and maxima (ALU 44 %).  4 bytes a load, eight dependent rounds: 13.4; 16 bytes, whose registers leave half the warps: 13.0; CTAs of 256: 11.7.
constexpr int kBoxers = 128;
template <int J, int KB>
__global__ void __launch_bounds__(kBoxers) box_kernel(const __grid_constant__ BoxParams P) {
    constexpr int C = J == 3 ? 3 : 2, kLanes = 4 * J / C, kTok = 32 / kLanes, D = 32 * J, W = C * KB / 4, S = (C + 1) / 2;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31;
    const long long id = (long long)blockIdx.x * (kBoxers / 32) + (threadIdx.x >> 5);
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
    const int part = lane % kLanes, tok = lane / kLanes, t = part / (J / C), j0 = (part - t * (J / C)) * C;
    const uint8_t* k = P.c.k + P.c.k_row(page, head, tok) + (t * J + j0) * KB;
    const __half* sc = P.c.sc + P.c.scale_row(page, head, tok) + j0;
    float lo[8 * C], hi[8 * C];
#pragma unroll
    for (int i = 0; i < 8 * C; ++i) lo[i] = INFINITY, hi[i] = -INFINITY;
    constexpr int kAhead = 8 / C;                                 // pairs of tokens whose loads go out together
    for (int x0 = 0; x0 < P.c.page(); x0 += 2 * kAhead * kTok) {
        uint32_t w[2 * kAhead][W], d[2 * kAhead][S];
#pragma unroll
        for (int a = 0; a < 2 * kAhead; ++a) {
            const int x = x0 + a * kTok;
            if (a >= 2 && x >= P.c.page()) continue;              // (a page holds 16 tokens at least: whole pairs)
            load_words<W>(w[a], k + (long long)x * (4 * J * KB));
            const __half* at = sc + (long long)x * (2 * J);
            if constexpr (C == 3) load_words<1>(*reinterpret_cast<uint32_t(*)[1]>(d[a]), at), load_words<1>(*reinterpret_cast<uint32_t(*)[1]>(d[a] + 1), at + 2);      // rows of 12 bytes
            else load_words<S>(d[a], at);
        }
#pragma unroll
        for (int a = 0; a < 2 * kAhead; a += 2) {
            if (a >= 2 && x0 + a * kTok >= P.c.page()) continue;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float u[8], v[8];
                const float2 du = unpack_h2(d[a][c / 2]), dv = unpack_h2(d[a + 1][c / 2]);
                keys8<KB>(&w[a][c * KB / 4], c & 1 ? du.y : du.x, u);
                keys8<KB>(&w[a + 1][c * KB / 4], c & 1 ? dv.y : dv.x, v);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    lo[8 * c + i] = fminf(fminf(lo[8 * c + i], u[i]), v[i]), hi[8 * c + i] = fmaxf(fmaxf(hi[8 * c + i], u[i]), v[i]);
            }
        }
    }
    // the other tokens: at each exchange a lane keeps half of its values (the two halves of each 8, then of each 4, then of each 2)
    int n = 0;                                                    // the first of the values of each 8 that this lane holds
#pragma unroll
    for (int half = 4, o = kLanes; half >= 1 && o < 32; half /= 2, o *= 2) {
        const bool up = lane & o;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int i = 0; i < half; ++i) {
                const float a = up ? lo[8 * c + i] : lo[8 * c + half + i], b = up ? hi[8 * c + i] : hi[8 * c + half + i];
                lo[8 * c + i] = fminf(up ? lo[8 * c + half + i] : lo[8 * c + i], __shfl_xor_sync(0xffffffffu, a, o));
                hi[8 * c + i] = fmaxf(up ? hi[8 * c + half + i] : hi[8 * c + i], __shfl_xor_sync(0xffffffffu, b, o));
            }
        n += up ? half : 0;
    }
    // outwards to fp16, within its range: the box still holds every key
    constexpr int kLeft = 8 * kLanes / 32;                        // values of each 8: 1, with 8 lanes a token 2
    auto in = [](float x) { return fminf(fmaxf(x, -kKvMax), kKvMax); };
    __half* out = P.bounds + ((long long)page * P.c.n_kv + head) * (2 * D) + 32 * j0 + 8 * t + n;
#pragma unroll
    for (int c = 0; c < C; ++c)
#pragma unroll
        for (int i = 0; i < kLeft; ++i) {
            out[32 * c + i] = __float2half_rd(in(lo[8 * c + i]));
            out[D + 32 * c + i] = __float2half_ru(in(hi[8 * c + i]));
        }
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
    int n_kv, group, dim, width, shift, n_seq, n_rows, keep, first, last;
    float* near;                          // workspace, each [rows][n_kv][width]: a page's score, nearly
    float* sizes;                         // what its error is measured by
    double* scores;                       // in fp64, where many lie next to the border
    int* chosen;                          // [rows][n_kv][keep]
    int* held;                            // [rows]
    int* status;
};

// the larger one, NaN where one is
__device__ __forceinline__ float larger(float a, float b) { return b > a || b != b ? b : a; }

struct Row {
    int seq, pos;                         // sequence (-1: none), position in it
};
// the row's sequence and place, by each warp
__device__ __forceinline__ Row find_row(const ChooseParams& P, int row, bool tell) {
    const int lane = threadIdx.x & 31;
    int seq = row < P.n_seq ? row : -1, past = 0;
    if (P.starts) {
        seq = -1;
        for (int b0 = 0; b0 < P.n_seq && seq < 0; b0 += 32) {
            const int b = b0 + lane;
            const int s0 = b < P.n_seq ? __ldg(P.starts + b) : INT_MAX, s1 = b < P.n_seq ? __ldg(P.starts + b + 1) : 0;
            const uint32_t who = __ballot_sync(0xffffffffu, s0 <= row && row < s1);
            if (who) seq = b0 + __ffs(who) - 1, past = __shfl_sync(0xffffffffu, s1, __ffs(who) - 1);
        }
    }
    if (seq < 0) return Row{-1, -1};
    const int cap = P.width << P.shift, len = __ldg(P.lens + seq), held = min(max(len, 0), cap);
    if (tell && held != len && threadIdx.x == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    return Row{seq, P.starts ? held - (min(past, P.n_rows) - row) : held - 1};
}

constexpr int kScorers = 128;             // threads a CTA
constexpr int kTiles = 2, kPagesWarp = 16 * kTiles;              // pages a warp scores

// A warp 16 pages, the rows of mma.m16n8k16 over the 2 dim halves of a box: lo against the queries' negative parts, hi against the
// positive ones, the key head's query heads as columns (eight at a time).  A lane's 16 bytes of a box are two steps' operands as they
// lie; the queries are laid out to match.  Queries are fp16 after a power of two a head, fp32 ones two fp16 parts.  So a score is near:
// off by less than 2^-15 sum_c |q_c| max(|box|, 2^-14): 2^-20 of it for the queries' parts, and in each of four chains at most 16 steps of 17
// terms cut off at 2^-24 of the chain's share of that sum (a denormal side of a box counts there as 2^-14: with all sides 2^-24 scores were
// off by 7 times 2^-15 of the sum with the sides' own size).  The choice computes those that lie nearer to its border again, in fp64.
// 64 sequences of 154 pages on average, 8 key heads (40 MB of boxes): 9.8 us, bound by latency (lengths, table, boxes: dependent reads; DRAM
// 31 %); 47 instructions a page and key head.  (All in fp64 on the CUDA cores: 27 to 46 us, 184 instructions.)
template <int DT, int J>
__global__ void __launch_bounds__(kScorers) score_kernel(const __grid_constant__ ChooseParams P) {
    using T = typename Elem<DT>::type;
    constexpr int D = 32 * J, kParts = DT == QMV_OUT_F32 ? 2 : 1, kPieces = 2 * J, kAhead = J == 3 ? 3 : 4;
    static_assert(kPieces % kAhead == 0, "whole rounds of pieces");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, head = blockIdx.y, row = blockIdx.z;
    const Row r = find_row(P, row, false);
    const int at = r.pos >> P.shift;                              // the query's own page
    const int begin = P.first + (blockIdx.x * (kScorers / 32) + warp) * kPagesWarp, end = min(at + 1 - P.last, begin + kPagesWarp);
    if (r.pos < 0 || at + 1 <= P.keep || begin >= end) return;
    // the boxes of pages begin + g and begin + g + 8 of each tile: this lane's runs of 8 halves
    bool there[kTiles][2];
    const uint4* box[kTiles][2];
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int i = begin + 16 * y + g + 8 * x, page = i < end ? __ldg(P.tables + (long long)r.seq * P.width + i) : -1;
            there[y][x] = page >= 0 && page < P.n_pages;
            box[y][x] = reinterpret_cast<const uint4*>(P.bounds + ((long long)(there[y][x] ? page : 0) * P.n_kv + head) * (2 * D)) + t;
        }
    uint4 a[kAhead][2];
    auto load = [&](int y, int s0) {
#pragma unroll
        for (int s = 0; s < kAhead; ++s)
#pragma unroll
            for (int x = 0; x < 2; ++x) a[s][x] = there[y][x] ? __ldg(box[y][x] + 4 * (s0 + s)) : make_uint4(0, 0, 0, 0);
    };
    load(0, 0);
    float best[kTiles][2], size = 0.f;                            // of the pages; the heads' largest sum of |q|
    uint32_t wide[kTiles][2];                                     // largest |half| of the boxes' runs
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
        for (int x = 0; x < 2; ++x) best[y][x] = -INFINITY, wide[y][x] = 0;
    for (int h0 = 0; h0 < P.group; h0 += 8) {
        // ---- column g: query head h0 + g
        const bool live = h0 + g < P.group;
        const T* src = static_cast<const T*>(P.q) + row * P.q_stride + (long long)(head * P.group + (live ? h0 + g : 0)) * D + 8 * t;
        float4 q[J][2];
        float top = 0.f, sum = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float4 v = q[j][m] = live ? load4(src + 32 * j + 4 * m) : make_float4(0.f, 0.f, 0.f, 0.f);
                top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
                sum += (fabsf(v.x) + fabsf(v.y)) + (fabsf(v.z) + fabsf(v.w));
            }
#pragma unroll
        for (int o = 1; o < 4; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o)), sum += __shfl_xor_sync(0xffffffffu, sum, o);
        size = larger(size, sum);
        if (top > 0.f && top < 1e-24f) size = INFINITY;           // below what the powers of two here lift: all of it in fp64
        // 2^14 <= top 2^-e < 2^15; a head of zeros or with an infinity keeps its size
        const int ex = int((__float_as_uint(top) >> 23) & 255u), e = ex == 0 || ex == 255 ? 0 : max(-100, ex - 127 - 14);
        const float down = __uint_as_float(uint32_t(127 - e) << 23);
        uint32_t b[kPieces][2][kParts][2];                        // [piece: lo's, hi's][step][part][half of the step]
#pragma unroll
        for (int j = 0; j < J; ++j)
#pragma unroll
            for (int m = 0; m < 2; ++m) {
                const float v[4] = {q[j][m].x * down, q[j][m].y * down, q[j][m].z * down, q[j][m].w * down};
#pragma unroll
                for (int y = 0; y < 2; ++y) {
                    uint32_t w = pack_h2(v[2 * y], v[2 * y + 1]);
                    const float2 f = unpack_h2(w);
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        if (part) w = pack_h2(v[2 * y] - f.x, v[2 * y + 1] - f.y);
                        // by the sign of the value, not of its second part
                        const uint32_t minus = (v[2 * y] < 0.f ? 0xFFFFu : 0u) | (v[2 * y + 1] < 0.f ? 0xFFFF0000u : 0u);
                        b[j][m][part][y] = w & minus, b[J + j][m][part][y] = w & ~minus;
                    }
                }
            }
        const float back = __uint_as_float(uint32_t(127 + e) << 23);
        const float back0 = __shfl_sync(0xffffffffu, back, 8 * t), back1 = __shfl_sync(0xffffffffu, back, 8 * t + 4);
#pragma unroll
        for (int y = 0; y < kTiles; ++y) {
            if (begin + 16 * y >= end) continue;
            // ---- the products, in four chains
            float c[4][4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
#pragma unroll
                for (int i = 0; i < 4; ++i) c[x][i] = 0.f;
#pragma unroll
            for (int s0 = 0; s0 < kPieces; s0 += kAhead) {
                if (y || s0 || h0) load(y, s0);
#pragma unroll
                for (int s = 0; s < kAhead; ++s) {
#pragma unroll
                    for (int part = 0; part < kParts; ++part) {
                        mma16816(c[s & 1], a[s][0].x, a[s][1].x, a[s][0].y, a[s][1].y, b[s0 + s][0][part][0], b[s0 + s][0][part][1]);
                        mma16816(c[2 + (s & 1)], a[s][0].z, a[s][1].z, a[s][0].w, a[s][1].w, b[s0 + s][1][part][0], b[s0 + s][1][part][1]);
                    }
                    if (h0 == 0)
#pragma unroll
                        for (int x = 0; x < 2; ++x)
                            wide[y][x] = __vmaxu2(wide[y][x], __vmaxu2(__vmaxu2(a[s][x].x & 0x7FFF7FFFu, a[s][x].y & 0x7FFF7FFFu), __vmaxu2(a[s][x].z & 0x7FFF7FFFu, a[s][x].w & 0x7FFF7FFFu)));
                }
            }
            // ---- columns 2 t, 2 t + 1 of rows g and g + 8: times their heads' powers of two, and the largest
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float u = ((c[0][2 * x] + c[1][2 * x]) + (c[2][2 * x] + c[3][2 * x])) * back0;
                const float v = ((c[0][2 * x + 1] + c[1][2 * x + 1]) + (c[2][2 * x + 1] + c[3][2 * x + 1])) * back1;
                if (h0 + 2 * t < P.group) best[y][x] = fmaxf(best[y][x], u);
                if (h0 + 2 * t + 1 < P.group) best[y][x] = fmaxf(best[y][x], v);
            }
        }
    }
#pragma unroll
    for (int o = 4; o < 32; o *= 2) {
        size = larger(size, __shfl_xor_sync(0xffffffffu, size, o));      // over the columns
    }
    const long long out = ((long long)row * P.n_kv + head) * P.width;
#pragma unroll
    for (int y = 0; y < kTiles; ++y)
#pragma unroll
        for (int x = 0; x < 2; ++x) {
#pragma unroll
            for (int o = 1; o < 4; o *= 2) {
                best[y][x] = fmaxf(best[y][x], __shfl_xor_sync(0xffffffffu, best[y][x], o));
                wide[y][x] = __vmaxu2(wide[y][x], __shfl_xor_sync(0xffffffffu, wide[y][x], o));
            }
            const int i = begin + 16 * y + g + 8 * x;
            const float2 w = unpack_h2(wide[y][x]);
            if (t == x && i < end) {
                P.near[out + i] = there[y][x] ? best[y][x] : -INFINITY;
                P.sizes[out + i] = there[y][x] ? size * larger(6.103515625e-5f, larger(w.x, w.y)) : 0.f;
            }
        }
}

// ---- the choice ------------------------------------------------------------------------------------------------

__device__ __forceinline__ uint64_t ordered64(double x) {
    if (!(x == x)) return 0;
    const uint64_t b = __double_as_longlong(x + 0.0);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}

// exclusive sums over the CTA's threads; total: of all
__device__ __forceinline__ int block_sums(int x, int* s_warp, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int inc = x;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
        const int y = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += y;
    }
    __syncthreads();                                              // s_warp may still be read
    if (lane == 31) s_warp[warp] = inc;
    __syncthreads();
    total = 0;
    int before = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += s_warp[w];
        total += s_warp[w];
    }
    return before + inc - x;
}
constexpr int kMostPer = 4, kList = 512, kHold = 8192;

// Of `per` bins a thread from the top (bin per * kThreads - 1 - per * tid and the ones below) the one in which the count reaches `need`,
// and how many of it are needed.
__device__ __forceinline__ void find_bin(const int* s_hist, int per, int need, int* s_warp, int* s_bin, int* s_need) {
    const int top = per * (kThreads - int(threadIdx.x)) - 1;
    int sum = 0, total;
    for (int i = 0; i < per; ++i) sum += s_hist[top - i];
    int above = block_sums(sum, s_warp, total);
    if (above < need && need <= above + sum)
        for (int i = 0; i < per; ++i) {
            const int n = s_hist[top - i];
            if (above < need && need <= above + n) *s_bin = top - i, *s_need = need - above;
            above += n;
        }
    __syncthreads();
}

// A CTA a row and key head.  A histogram of the near scores in even bins between the least and the largest tells the bin of the k-th
// largest.  Pages whose score lies above that bin by twice the error are taken, those below it by as much are not; the few others are
// computed again in fp64, a warp each, and ranked against one another (more than a list holds, scores alike say: by digits of
// 8 bits).  Then the pages in order.  2048 pages of 8 key heads: 9.3 us, 11 barriers, each phase 1 to 1.8 us; bound by latency and by fetching its
// own instructions (unrolled over scores in registers 16 us), so its loops are rolled, over scores in shared memory.
template <int DT>
__global__ void __launch_bounds__(kThreads) choose_kernel(const __grid_constant__ ChooseParams P) {
    using T = typename Elem<DT>::type;
    __shared__ float s_near[kHold];
    __shared__ int s_hist[kMostPer * kThreads], s_bin, s_need, s_warp[kThreads / 32], s_count;
    __shared__ float s_lo[kThreads / 32], s_hi[kThreads / 32], s_size[kThreads / 32];
    __shared__ uint64_t s_key[kList];
    __shared__ int s_place[kList];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, head = blockIdx.x % P.n_kv, row = blockIdx.x / P.n_kv;
    const Row r = find_row(P, row, head == 0);
    int* out = P.chosen + (long long)blockIdx.x * P.keep;
    const int* table = P.tables + (long long)max(r.seq, 0) * P.width;
    const int n = r.pos < 0 ? 0 : (r.pos >> P.shift) + 1, kept = min(n, P.keep);
    if (head == 0 && tid == 0) P.held[row] = n ? ((kept - 1) << P.shift) + (r.pos & ((1 << P.shift) - 1)) + 1 : 0;
    if (n <= P.keep) {
        for (int i = tid; i < P.keep; i += kThreads) out[i] = i < n ? __ldg(table + i) : -1;
        return;
    }
    const int middle = n - P.last - P.first, k = P.keep - P.first - P.last;
    for (int i = tid; i < P.first; i += kThreads) out[i] = __ldg(table + i);
    for (int i = tid; i < P.last; i += kThreads) out[P.keep - P.last + i] = __ldg(table + n - P.last + i);
    if (k == 0) return;
    table += P.first, out += P.first;
    // ---- the middle's scores, in shared memory where they fit, and their range.  More bins leave fewer pages to compute again: 1024 for 2045
    // pages 14.0 us of both kernels, 256 15.4; for 151 19.1 and 16.9 (64 rows of 8 key heads)
    const int per_thread = middle > 2 * kThreads ? kMostPer : 1, bins = per_thread * kThreads;
    const long long at0 = (long long)blockIdx.x * P.width + P.first;
    float* near = middle <= kHold ? s_near : P.near + at0;
    float lo = INFINITY, hi = -INFINITY, size = 0.f;
#pragma unroll 4
    for (int i = tid; i < middle; i += kThreads) {
        const float s = P.near[at0 + i], y = P.sizes[at0 + i];
        if (middle <= kHold) s_near[i] = s;
        if (fabsf(s) < INFINITY) lo = fminf(lo, s), hi = fmaxf(hi, s);
        size = larger(size, y);
    }
    for (int i = tid; i < bins; i += kThreads) s_hist[i] = 0;
    if (tid == 0) s_count = 0;
#pragma unroll
    for (int o = 16; o; o /= 2) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o)), hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
        size = larger(size, __shfl_xor_sync(0xffffffffu, size, o));
    }
    if (lane == 0) s_lo[warp] = lo, s_hi[warp] = hi, s_size[warp] = size;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) lo = fminf(lo, s_lo[w]), hi = fmaxf(hi, s_hi[w]), size = larger(size, s_size[w]);
    const float per = hi > lo && hi - lo < INFINITY ? bins / (hi - lo) : 0.f;
    const float off = size < 1e30f ? size * (1.f / 16384.f) : INFINITY;      // twice the error; with infinities and NaN every page is computed again
    // grows with the score: each step of it does (NaN: 0)
    auto bin_of = [&](float f) { return !(f > lo) ? 0 : f >= hi ? bins - 1 : min(bins - 1, int((f - lo) * per)); };
#pragma unroll 1
    for (int i = tid; i < middle; i += kThreads) atomicAdd(&s_hist[bin_of(near[i])], 1);
    __syncthreads();
    find_bin(s_hist, per_thread, k, s_warp, &s_bin, &s_need);
    // ---- taken: +inf, not: -inf; the ones to be computed again are listed
    const int bin = s_bin;
    int sure = 0, total;
#pragma unroll 1
    for (int i = tid; i < middle; i += kThreads) {
        const float s = near[i];
        const bool above = off < INFINITY && bin_of(s - off) > bin, below = off < INFINITY && bin_of(s + off) < bin;
        sure += above;
        if (!above && !below) {
            const int at = atomicAdd(&s_count, 1);
            if (at < kList) s_place[at] = i;
        }
        near[i] = above ? INFINITY : below ? -INFINITY : 0.f;
    }
    block_sums(sure, s_warp, total);
    int need = k - total;                                         // of the ones to be computed again: one at least, not more than there are
    const int members = s_count;
    // a page's score in fp64, by a warp, four heads at a time
    auto exact = [&](int i) {
        const int page = __ldg(table + i), D = P.dim;
        if (page < 0 || page >= P.n_pages) return -double(INFINITY);
        const __half* box = P.bounds + ((long long)page * P.n_kv + head) * (2 * D);
        double best = -INFINITY;
#pragma unroll 1
        for (int h0 = 0; h0 < P.group; h0 += 4) {
            const T* q = static_cast<const T*>(P.q) + row * P.q_stride + (long long)(head * P.group + h0) * D;
            double sum[4] = {0.0, 0.0, 0.0, 0.0};
#pragma unroll 2
            for (int c = lane; c < D; c += 32) {
                const float a = __half2float(box[c]), b = __half2float(box[D + c]);
#pragma unroll
                for (int h = 0; h < 4; ++h) {
                    const float x = h0 + h < P.group ? to_float(q[h * D + c]) : 0.f;
                    sum[h] = fma(double(x), double(x > 0.f ? b : a), sum[h]);
                }
            }
#pragma unroll
            for (int o = 16; o; o /= 2)
#pragma unroll
                for (int h = 0; h < 4; ++h) sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], o);
#pragma unroll
            for (int h = 0; h < 4; ++h)
                if (h0 + h < P.group) best = fmax(best, sum[h]);
        }
        return best;
    };
    if (need == members) {
#pragma unroll 1
        for (int i = tid; i < middle; i += kThreads)
            if (near[i] == 0.f) near[i] = INFINITY;
    } else if (members <= kList) {
#pragma unroll 1
        for (int m = warp; m < members; m += kThreads / 32) {
            const double s = exact(s_place[m]);
            if (lane == 0) s_key[m] = ordered64(s);
        }
        __syncthreads();
#pragma unroll 1
        for (int m = tid; m < members; m += kThreads) {
            const uint64_t key = s_key[m];
            const int place = s_place[m];
            int rank = 0;
            for (int j = 0; j < members; ++j) rank += s_key[j] > key || (s_key[j] == key && s_place[j] < place);
            near[place] = rank < need ? INFINITY : -INFINITY;
        }
    } else {
        double* scores = P.scores + at0;
#pragma unroll 1
        for (int i = warp; i < middle; i += kThreads / 32)
            if (near[i] == 0.f) {
                const double s = exact(i);
                if (lane == 0) scores[i] = s;
            }
        uint64_t prefix = 0, mask = 0;
#pragma unroll 1
        for (int shift = 56; shift >= 0; shift -= 8) {
            __syncthreads();
            s_hist[tid] = 0;
            __syncthreads();
            for (int i = tid; i < middle; i += kThreads) {
                if (near[i] != 0.f) continue;
                const uint64_t key = ordered64(scores[i]);
                if ((key & mask) == prefix) atomicAdd(&s_hist[key >> shift & 255], 1);
            }
            __syncthreads();
            find_bin(s_hist, 1, need, s_warp, &s_bin, &s_need);
            prefix |= uint64_t(s_bin) << shift, mask |= 255ull << shift;
            need = s_need;
        }
        // of equal scores the first ones
        int equal = 0;
#pragma unroll 1
        for (int i0 = 0; i0 < middle; i0 += kThreads) {
            const int i = i0 + tid;
            const bool open = i < middle && near[i] == 0.f;
            const uint64_t key = open ? ordered64(scores[i]) : 0;
            const int before = equal + block_sums(open && key == prefix, s_warp, total);
            if (open) near[i] = key > prefix || (key == prefix && before < need) ? INFINITY : -INFINITY;
            equal += total;
        }
    }
    // ---- the pages, a run of places a thread
    __syncthreads();
    const int run = (middle + kThreads - 1) / kThreads, i0 = min(middle, tid * run), i1 = min(middle, i0 + run);
    int count = 0;
#pragma unroll 1
    for (int i = i0; i < i1; ++i) count += near[i] > 0.f;
    int to = block_sums(count, s_warp, total);
#pragma unroll 1
    for (int i = i0; i < i1; ++i)
        if (near[i] > 0.f) out[to++] = __ldg(table + i);
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
    const long long ctas = ((long long)n_seq * P.most * P.c.n_kv + kBoxers / 32 - 1) / (kBoxers / 32);
    if (ctas > 0x7FFFFFFFLL) return ST_BAD_TOKENS;
    auto go = [&](auto j) {
        constexpr int J = decltype(j)::value;
        return P.c.kb == 4 ? launch_pdl(box_kernel<J, 4>, dim3(unsigned(ctas)), dim3(kBoxers), static_cast<cudaStream_t>(stream), P)
                           : launch_pdl(box_kernel<J, 8>, dim3(unsigned(ctas)), dim3(kBoxers), static_cast<cudaStream_t>(stream), P);
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
    if (kv_view(cache, c) || table_width <= 0 || table_width > kMostKeys >> c.page_shift || n_rows <= 0 || n_rows > 65535 || n_rows * c.n_kv > INT_MAX || keep <= 0)
        return 0;
    return table_width <= keep ? 8 : 16LL * n_rows * c.n_kv * table_width;
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
    if (n_seq <= 0 || n_seq > 65535 || n_rows < 0 || n_rows > 65535 || n_rows * c.n_kv > INT_MAX || (!starts && n_rows < n_seq)) return ST_BAD_TOKENS;
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
    P.n_kv = c.n_kv, P.group = n_heads / c.n_kv, P.dim = c.dim, P.width = table_width, P.shift = c.page_shift, P.n_seq = n_seq, P.n_rows = int(n_rows);
    P.keep = keep, P.first = first, P.last = last;
    const long long pages = n_rows * c.n_kv * table_width;
    P.scores = static_cast<double*>(workspace), P.near = reinterpret_cast<float*>(P.scores + pages), P.sizes = P.near + pages;
    P.chosen = chosen, P.held = held;
    P.status = device_status_ptr();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    const int middle = table_width - first - last;                // pages to score, at most
    if (table_width > keep && middle > 0) {
        constexpr int kPagesCta = kPagesWarp * (kScorers / 32);
        const dim3 grid((middle + kPagesCta - 1) / kPagesCta, c.n_kv, unsigned(n_rows));
        auto go = [&](auto dt, auto j) {
            constexpr int DT = decltype(dt)::value, J = decltype(j)::value;
            return launch_pdl(score_kernel<DT, J>, grid, dim3(kScorers), s, P);
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
    return by_elem(dtype, [&](auto dt) { return launch_behind(choose_kernel<decltype(dt)::value>, dim3(unsigned(n_rows * c.n_kv)), dim3(kThreads), s, P); });
}

}  // extern "C"
