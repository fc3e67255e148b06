// Attention of few query rows over the quantised cache (layout: qmv_kv.cuh): decode steps, drafted tokens, and every call
// with fp32 queries.
//
//   s[r][key] = scale * sum_j d_k[key][j] * sum_{i in block j} q[r][i] code_k[key][i]
//   o[r][i]   = sum_key p[r][key] d_v[key][j(i)] code_v[key][i] / sum_key p[r][key],   p = 2^(s log2 e - ref)
//
// Bound by reading the cache once (4.5 or 8.5 bits a value), so what counts is instructions per value: at 6.5 TB/s an SM
// sees about 40 four-bit values a clock.  Both products run on mma.sync m16n8k16 (fp16 in, fp32 sums) with the cache as
// the 16-row operand, straight from global memory: the codes' bits ARE the operand.  A code c masked out of its word
// is the fp16 denormal c 2^-24 (16 c 2^-24 for the upper nibble of a byte), which the tensor cores multiply exactly, so a
// 4-bit pair costs one AND and no conversion; the factor 2^24 and the queries' 1 / 16 are folded into constants.
// (tcgen05 would need the unpacked values written to shared memory first, more bytes a clock than an SM writes.)  The codes'
// offset (8 or 128) comes out as its own term: in the scores it is the accumulator's start, -off sum_i q[i] per block,
// in the output one more product with a constant row a block.  Scales stay out of the products: d_k multiplies a block's
// 16 x 8 scores in fp32, d_v goes into p before it is rounded to fp16.
//
// Queries are fp16 after a power of two per row (exact for bf16 and fp16); fp32 queries are two fp16 parts (HL), and so
// is p d_v then, which keeps fp32's accuracy.  The softmax reference only moves when a score passes it by 2^4 or a d_v
// its limit (checked with one vote a tile): p d_v 2^E stays below 2^15.  Sums and statistics are fp32.
//
// Work: units of 64 keys (16 a warp) of segments (sequence, key head, tile of 8 NT rows); the list of all units is cut into
// equal runs, one a CTA, so unequal lengths do not unbalance it.  A segment cut over several CTAs leaves its parts in the
// workspace and attn_join_kernel adds them in order.
#pragma once
#include <algorithm>
#include <type_traits>

#include "qmv_kv.cuh"

namespace qmv {

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
    int row_tiles;                        // tiles of query rows (token-major over the heads of a key head)
    int split;                            // segments may be cut: parts, desc, attn_join_kernel follows
    int by_segment;                       // desc has an entry a segment (else a CTA)
    float* parts;                         // [2 a CTA][8 NT rows][dim + 2]: sums, then reference and weight
    int4* desc;                           // first part, parts, (sequence, key head x row tiles + row tile)
    int* status;
};

constexpr int kAttnWarps = 4;
constexpr int kAttnUnit = 64;             // keys a unit
constexpr int kAttnMinUnits = 4;          // units a CTA takes at least before segments are cut
constexpr float kAttnNone = -1e30f;       // reference of a row that has seen no key

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t movm(uint32_t x) {            // 8 x 8 transpose of fp16 over the warp
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// N words from p to the lane's places in shared memory (16-byte pieces of a warp side by side), asynchronously; p is
// aligned to N words' largest power of two up to 16 bytes
template <int N> constexpr int kPiece = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;     // words of a copy
template <int N>
__device__ __forceinline__ void stage_words(uint32_t dst, const void* p, int lane) {
    constexpr int W = kPiece<N>;
#pragma unroll
    for (int i = 0; i < N; i += W) {
        const uint32_t d = dst + (32 * i + W * lane) * 4;
        if constexpr (W == 4)
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(d), "l"(static_cast<const uint8_t*>(p) + 4 * i) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" :: "r"(d), "l"(static_cast<const uint8_t*>(p) + 4 * i), "n"(4 * W) : "memory");
    }
}
template <int N>
__device__ __forceinline__ void staged_words(uint32_t (&w)[N], uint32_t src, int lane) {
    constexpr int W = kPiece<N>;
#pragma unroll
    for (int i = 0; i < N; i += W) {
        const uint32_t a = src + (32 * i + W * lane) * 4;
        if constexpr (W == 4)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(a));
        else if constexpr (W == 2)
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(a));
        else
            asm volatile("ld.shared.u32 %0, [%1];" : "=r"(w[i]) : "r"(a));
    }
}

// The 16 keys of a warp's tile as a lane (g = lane / 4, t = lane % 4) uses them: run t of the K rows of keys g and g + 8,
// run g of the V pairs t and t + 4, the scales of keys g and g + 8.  Each lane copies its own words to shared memory
// some tiles ahead (cp.async), so nothing but its own copies has to be waited for and no register holds them.
template <int J, int KB, int VB>
struct AttnTile {
    static constexpr int kK = J * KB / 4, kV = J * VB / 4, kWords = 2 * (kK + kV + J);     // words a lane
    static constexpr int kBytes = 32 * 4 * kWords;
    static __device__ __forceinline__ void issue(uint32_t buf, const KvView& c, long long page, int head, int at, int lane) {
        const int g = lane >> 2, t = lane & 3;
        const long long row = ((page * c.n_kv + head) << c.page_shift) + at;
        const uint8_t* k = c.k + (row + g) * (4 * J * KB) + t * J * KB;
        const uint8_t* v = c.v + ((row >> 1) + t) * (8 * J * VB) + g * J * VB;
        const __half* sc = c.sc + (row + g) * (2 * J);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            stage_words<kK>(buf + 128 * h * kK, k + 8 * h * (4 * J * KB), lane);
            stage_words<J>(buf + 128 * (2 * kK + h * J), sc + 8 * h * (2 * J), lane);
            stage_words<kV>(buf + 128 * (2 * kK + 2 * J + h * kV), v + 4 * h * (8 * J * VB), lane);
        }
    }
    static __device__ __forceinline__ void keys(uint32_t (&k)[2][kK], uint32_t (&sc)[2][J], uint32_t buf, int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            staged_words<kK>(k[h], buf + 128 * h * kK, lane);
            staged_words<J>(sc[h], buf + 128 * (2 * kK + h * J), lane);
        }
    }
    static __device__ __forceinline__ void vals(uint32_t (&v)[2][kV], uint32_t buf, int lane) {
#pragma unroll
        for (int h = 0; h < 2; ++h) staged_words<kV>(v[h], buf + 128 * (2 * kK + 2 * J + h * kV), lane);
    }
};
// half i of a key's scales (K's J, then V's J)
template <int J>
__device__ __forceinline__ float scale_of(const uint32_t (&sc)[J], int i) {
    return h2f(i & 1 ? sc[i >> 1] >> 16 : sc[i >> 1] & 0xFFFFu);
}

// CTAs an SM is to hold, and the tiles a warp has in shared memory, within 227 KB an SM
template <int DT, int J, int NT> constexpr int kAttnCtas = J == 8 || NT == 2 ? 2 : DT == QMV_OUT_F32 ? 3 : 4;
template <int DT, int J, int KB, int VB, int NT>
__host__ __device__ constexpr int attn_stages() {
    const int room = (226 * 1024) / kAttnCtas<DT, J, NT> - 1024 - (DT == QMV_OUT_F32 ? 2 : 1) * NT * J * 512 - 256;
    const int n = room / (kAttnWarps * AttnTile<J, KB, VB>::kBytes);
    return n > 4 ? 4 : n;
}

template <int J, int NT>
__host__ __device__ constexpr int attn_part_floats() { return 8 * NT * (32 * J + 2); }

// where a unit lies: sequence, segment within it, unit within that; found once a CTA, then stepped
struct AttnSeq {
    int row0, n, len, first_unit, units;  // query rows, tokens in the cache, units of a segment
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& P, int b, bool report) {
    AttnSeq s;
    int row1;
    if (P.starts) {
        s.row0 = min(max(__ldg(P.starts + b), 0), P.n_rows);
        row1 = min(max(__ldg(P.starts + b + 1), s.row0), P.n_rows);
    } else {
        s.row0 = b, row1 = b + 1;
    }
    const int len = __ldg(P.lens + b), cap = P.width << P.c.page_shift;
    s.n = row1 - s.row0;
    s.len = min(max(len, 0), cap);
    if (report && P.status && (len < 0 || len > cap || s.n > P.max_new)) atomicOr(P.status, DEV_BAD_ADDRESS);
    const int first = s.n == 0 ? 0 : max(0, min(P.window > 0 ? s.len - s.n - P.window + 1 : 0, s.len));
    s.first_unit = first / kAttnUnit;
    s.units = s.n == 0 ? 1 : max(1, (s.len + kAttnUnit - 1) / kAttnUnit - s.first_unit);
    return s;
}

// one thread's share of a row's output or part: sums over `count` parts `stride` floats apart, weighted to one reference
template <int D>
__device__ __forceinline__ float4 attn_join(const float* parts, long long stride, int count, int row, int rows, int i0, float& ref,
                                            float& sum) {
    ref = kAttnNone;
    for (int k = 0; k < count; ++k) ref = fmaxf(ref, parts[k * stride + rows * D + row]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    sum = 0.f;
    for (int k = 0; k < count; ++k) {
        const float* p = parts + k * stride;
        const float f = ex2(p[rows * D + row] - ref);
        const float4 x = *reinterpret_cast<const float4*>(p + row * D + i0);
        sum = fmaf(f, p[rows * D + rows + row], sum);
        o.x = fmaf(f, x.x, o.x), o.y = fmaf(f, x.y, o.y), o.z = fmaf(f, x.z, o.z), o.w = fmaf(f, x.w, o.w);
    }
    return o;
}
template <class T>
__device__ __forceinline__ void attn_store(const AttnParams& P, int row0, int r, int group, int hk, int i0, float4 o, float sum) {
    const float inv = sum > 0.f ? __fdividef(1.f, sum) : 0.f;     // no key: zeros
    T* out = static_cast<T*>(P.out) + ((long long)(row0 + r / group) * P.n_heads + hk * group + r % group) * P.c.dim + i0;
    store4(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

template <int DT, int J, int KB, int VB, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, (kAttnCtas<DT, J, NT>)) attn_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    constexpr bool HL = DT == QMV_OUT_F32;
    constexpr int D = 32 * J, R = 8 * NT, kParts = HL ? 2 : 1;
    constexpr float kOffK = KB == 4 ? 8.f : 128.f;
    constexpr uint32_t kOffV = VB == 4 ? 0x00080008u : 0x00800080u;
    constexpr int S_ = attn_stages<DT, J, KB, VB, NT>();
    using Tile = AttnTile<J, KB, VB>;
    extern __shared__ __align__(16) float s_part[];              // the warps' tiles [warps][S_]; then [warps][R (D + 2)]
    __shared__ uint2 s_q[kParts][NT][J][2][32];                  // query fragments
    __shared__ long long s_scan[kAttnWarps + 1];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const int group = P.n_heads / P.c.n_kv, segs = P.c.n_kv * P.row_tiles;

    // ---- this CTA's run of units: all units, then the sequence that holds the first one
    long long total = 0, u0 = 0, u1 = 0;
    int ctas = gridDim.x;
    if (P.split) {
        for (int b = tid; b < P.n_seq; b += 32 * kAttnWarps) total += attn_seq(P, b, blockIdx.x == 0).units;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
        if (lane == 0) s_scan[warp] = total;
        __syncthreads();
        total = 0;
#pragma unroll
        for (int w = 0; w < kAttnWarps; ++w) total += s_scan[w];
        total *= segs;
        const long long most = max((total + kAttnMinUnits - 1) / kAttnMinUnits, (long long)P.n_seq * segs);
        if (most < ctas) ctas = int(most);
        if (blockIdx.x >= ctas) {
            if (tid == 0 && !P.by_segment) P.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
            asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
            return;
        }
        u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
    } else {
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
    int b = 0, seg = 0, unit = 0;                                 // the next unit
    AttnSeq S;
    if (P.split) {
        long long before = 0;                                     // units of earlier sequences
        for (int b0 = 0; b0 < P.n_seq; b0 += 32 * kAttnWarps) {
            const int mine = b0 + tid;
            const long long x = mine < P.n_seq ? (long long)attn_seq(P, mine, false).units * segs : 0;
            long long inc = x;
#pragma unroll
            for (int o = 1; o < 32; o *= 2) {
                const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                if (lane >= o) inc += y;
            }
            __syncthreads();
            if (lane == 31) s_scan[warp] = inc;
            __syncthreads();
            long long base = before;
            for (int w = 0; w < warp; ++w) base += s_scan[w];
            long long all = before;
            for (int w = 0; w < kAttnWarps; ++w) all += s_scan[w];
            if (u0 < all) {                                       // the same for every thread
                const bool hit = base + inc - x <= u0 && u0 < base + inc;
                __syncthreads();
                if (hit) s_scan[0] = mine, s_scan[1] = base + inc - x;
                __syncthreads();
                b = int(s_scan[0]);
                before = s_scan[1];
                break;
            }
            before = all;
        }
        S = attn_seq(P, b, false);
        const long long in = u0 - before;
        seg = int(in / S.units), unit = int(in - (long long)seg * S.units);
    } else {                                                      // one CTA a segment
        b = blockIdx.x / segs, seg = blockIdx.x - b * segs;
        S = attn_seq(P, b, seg == 0 && tid == 0);
        u1 = S.units;
    }
    bool owns = false;                                            // desc of this CTA written

    while (u0 < u1) {
        const int todo = int(min((long long)(S.units - unit), u1 - u0));
        const int hk = seg / P.row_tiles, rt = seg - hk * P.row_tiles;
        const int rows = min(max(min(S.n, P.max_new) * group - rt * R, 0), R);     // live query rows of this tile
        const int pos0 = S.len - S.n;                             // position of the sequence's first new token
        const int tok0 = rt * R / group, tok1 = (rt * R + max(rows, 1) - 1) / group;
        const int last = min(pos0 + tok1, S.len - 1);             // keys of interest: first .. last
        const int first = P.window > 0 ? max(0, pos0 + tok0 - P.window + 1) : 0;
        // every row sees keys full0 .. full1
        const int full0 = P.window > 0 ? max(0, pos0 + tok1 - P.window + 1) : 0, full1 = pos0 + tok0;

        float start[NT][J][2], cs[NT][2], M[NT][2], sum[NT][2], o[NT][J][2][4], off[NT][4];
        int pos[NT][2];
        float E = 0.f;
        uint32_t lim = 0;
        if (rows > 0) {
            // queries: lane (g, t) holds row g's values 8 t .. 8 t + 7 of each block, scaled to fp16 by a power of two
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const int r = 8 * nt + g, rr = rt * R + r;
                const bool live = r < rows;
                const T* src = static_cast<const T*>(P.q) + (live ? (S.row0 + rr / group) * P.q_stride + (hk * group + rr % group) * D : 0);
                float4 x[J][2];
                float top = 0.f;
#pragma unroll
                for (int j = 0; j < J; ++j)
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        x[j][m] = live ? load4(src + 32 * j + 8 * t + 4 * m) : make_float4(0.f, 0.f, 0.f, 0.f);
                        top = fmaxf(top, fmaxf(fmaxf(fabsf(x[j][m].x), fabsf(x[j][m].y)), fmaxf(fabsf(x[j][m].z), fabsf(x[j][m].w))));
                    }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // 2^14 <= top 2^-e < 2^15; a row of zeros or with an infinity keeps its size
                const int ex = int((__float_as_uint(top) >> 23) & 255u);
                const int e = ex == 0 || ex == 255 ? 0 : ex - 127 - 14;
                const float down = __uint_as_float(uint32_t(127 - max(-120, min(120, e))) << 23);
                const float up = P.scale * 1.4426950408889634f * 16777216.f * __uint_as_float(uint32_t(127 + max(-120, min(120, e))) << 23);
                cs[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);
                cs[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    float part = 0.f;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        constexpr float kHigh = KB == 4 ? 1.f / 16.f : 1.f;     // the upper nibbles arrive 16 times too large
                        const float a = x[j][m].x * down, b2 = x[j][m].y * down, c = x[j][m].z * down * kHigh, d = x[j][m].w * down * kHigh;
                        const uint32_t lo = pack_h2(a, b2), hi = pack_h2(c, d);
                        const float2 fl = unpack_h2(lo), fh = unpack_h2(hi);
                        part += (fl.x + fl.y) + (fh.x + fh.y) * (1.f / kHigh);
                        if (warp == 0) s_q[0][nt][j][m][lane] = make_uint2(lo, hi);
                        if constexpr (HL) {
                            const uint32_t lo2 = pack_h2(a - fl.x, b2 - fl.y), hi2 = pack_h2(c - fh.x, d - fh.y);
                            const float2 gl = unpack_h2(lo2), gh = unpack_h2(hi2);
                            part += (gl.x + gl.y) + (gh.x + gh.y) * (1.f / kHigh);
                            if (warp == 0) s_q[kParts - 1][nt][j][m][lane] = make_uint2(lo2, hi2);
                        }
                    }
                    part += __shfl_xor_sync(0xffffffffu, part, 1);
                    part += __shfl_xor_sync(0xffffffffu, part, 2);
                    part *= -kOffK * 5.9604644775390625e-8f;
                    start[nt][j][0] = __shfl_sync(0xffffffffu, part, 8 * t);
                    start[nt][j][1] = __shfl_sync(0xffffffffu, part, 8 * t + 4);
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[nt][j][m][i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    M[nt][i] = kAttnNone, sum[nt][i] = 0.f;
                    pos[nt][i] = pos0 + (rt * R + min(8 * nt + 2 * t + i, rows - 1)) / group;
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) off[nt][i] = 0.f;
            }
            __syncthreads();
            // ---- this warp's tiles: one a unit
            const int* table = P.tables + (long long)b * P.width;
            const int key0 = (S.first_unit + unit) * kAttnUnit + 16 * warp;
            auto page_of = [&](int key) -> long long {            // -1: nothing to see here
                if (key > last || key + 15 < first) return -1;
                const int p = __ldg(table + (key >> P.c.page_shift));
                if (p >= 0 && p < P.c.n_pages) return p;
                if (lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
                return -1;
            };
            const uint32_t buf0 = smem_u32(s_part) + warp * S_ * Tile::kBytes;
            uint32_t held = 0;                                    // bit i: slot i of the ring holds a tile
            auto ask = [&](int u) {                               // starts the copies of unit u's tile
                const int key = key0 + u * kAttnUnit, slot = u % S_;
                const long long page = u < todo ? page_of(key) : -1;
                held = (held & ~(1u << slot)) | (page >= 0 ? 1u << slot : 0u);
                if (page >= 0) Tile::issue(buf0 + slot * Tile::kBytes, P.c, page, hk, key & (P.c.page() - 1), lane);
                asm volatile("cp.async.commit_group;" ::: "memory");
            };
#pragma unroll
            for (int u = 0; u < S_ - 1; ++u) ask(u);
            for (int u = 0; u < todo; ++u) {
                const int key = key0 + u * kAttnUnit;
                ask(u + S_ - 1);
                asm volatile("cp.async.wait_group %0;" :: "n"(S_ - 1) : "memory");
                const uint32_t buf = buf0 + (u % S_) * Tile::kBytes;
                if (held >> (u % S_) & 1u) {
                    uint32_t kw[2][Tile::kK], sc[2][J];
                    Tile::keys(kw, sc, buf, lane);
                    // keys nobody sees hold anything (NaN scales too): scale 0, and their scores are masked
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = 0; i < J; ++i)
                            if (uint32_t(key + g + 8 * h - first) > uint32_t(last - first)) sc[h][i] = 0u;
                    // scores: C row g / g + 8 = keys, columns 2 t, 2 t + 1 = query rows
                    float s[NT][4];
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][i] = 0.f;
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float d0 = scale_of(sc[0], j), d1 = scale_of(sc[1], j);
                        uint32_t a[2][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if constexpr (KB == 4) {
                                const uint32_t w = kw[h][j], w8 = w >> 8;
                                a[0][h] = w & 0x000F000Fu, a[0][2 + h] = w & 0x00F000F0u;
                                a[1][h] = w8 & 0x000F000Fu, a[1][2 + h] = w8 & 0x00F000F0u;
                            } else {
                                const uint32_t w = kw[h][2 * j], x = kw[h][2 * j + 1];
                                a[0][h] = w & 0x00FF00FFu, a[0][2 + h] = (w >> 8) & 0x00FF00FFu;
                                a[1][h] = x & 0x00FF00FFu, a[1][2 + h] = (x >> 8) & 0x00FF00FFu;
                            }
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            float c[4] = {start[nt][j][0], start[nt][j][1], start[nt][j][0], start[nt][j][1]};
#pragma unroll
                            for (int p = 0; p < kParts; ++p)
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    const uint2 w = s_q[p][nt][j][m][lane];
                                    mma16816(c, a[m][0], a[m][1], a[m][2], a[m][3], w.x, w.y);
                                }
                            s[nt][0] = fmaf(d0, c[0], s[nt][0]), s[nt][1] = fmaf(d0, c[1], s[nt][1]);
                            s[nt][2] = fmaf(d1, c[2], s[nt][2]), s[nt][3] = fmaf(d1, c[3], s[nt][3]);
                        }
                    }
                    // log2 scores; a tile that some row does not see whole is masked key by key
                    const bool whole = key >= full0 && key + 15 <= full1;
                    float top = kAttnNone;
                    const float limit = 4.f + E;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            s[nt][i] *= cs[nt][i & 1];
                            if (!whole) {
                                const int k = key + g + 8 * (i >> 1), p = pos[nt][i & 1];
                                if (k > p || k > last || (P.window > 0 && p - k >= P.window)) s[nt][i] = -INFINITY;
                            }
                            top = fmaxf(top, s[nt][i] - (M[nt][i & 1] - E));
                        }
                    uint32_t dv = 0;                              // the largest |d_v| of the lane's keys, as fp16 bits
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int i = J / 2; i < J; ++i) dv = __vmaxu2(dv, sc[h][i] & (J % 2 && i == J / 2 ? 0x7FFF0000u : 0x7FFF7FFFu));
                    dv = max(dv >> 16, dv & 0xFFFFu);
                    if (__any_sync(0xffffffffu, top > limit || dv > lim)) {
                        float old[NT][2];
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 2; ++i) {
                                old[nt][i] = M[nt][i] - E;
                                float m = fmaxf(s[nt][i], s[nt][i + 2]);
#pragma unroll
                                for (int w = 4; w < 32; w *= 2) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, w));
                                M[nt][i] = fmaxf(M[nt][i], m);
                            }
                        dv = __reduce_max_sync(0xffffffffu, dv);
                        if (dv > lim) {                           // up to 2^(ev - 11) with a factor of 8 to 16 to spare
                            const uint32_t ev = max(1u, dv >> 10);
                            lim = min((ev + 4) << 10, 0x7BFFu);
                            E = float(22 - int(ev));
                        }
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float f0 = ex2(old[nt][0] - (M[nt][0] - E)), f1 = ex2(old[nt][1] - (M[nt][1] - E));
                            sum[nt][0] *= f0, sum[nt][1] *= f1;
                            off[nt][0] *= f0, off[nt][1] *= f1;
#pragma unroll
                            for (int j = 0; j < J; ++j)
#pragma unroll
                                for (int m = 0; m < 2; ++m) {
                                    o[nt][j][m][0] *= f0, o[nt][j][m][1] *= f1;
                                    o[nt][j][m][2] *= f0, o[nt][j][m][3] *= f1;
                                }
                        }
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[nt][i] = ex2(s[nt][i] - (M[nt][i & 1] - E));
                        sum[nt][0] += s[nt][0] + s[nt][2], sum[nt][1] += s[nt][1] + s[nt][3];
                    }
                    uint32_t vw[2][Tile::kV];
                    Tile::vals(vw, buf, lane);
                    // output: rows = values g / g + 8 of two tiles a block, k = keys, columns = query rows
#pragma unroll
                    for (int j = 0; j < J; ++j) {
                        const float d0 = scale_of(sc[0], J + j), d1 = scale_of(sc[1], J + j);
                        uint32_t a[2][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {             // pair t (k 2 t, 2 t + 1), pair t + 4 (k 8 + 2 t, 9 + 2 t)
                            if constexpr (VB == 4) {
                                const uint32_t w = vw[h][j], w8 = w >> 8;
                                a[0][2 * h] = w & 0x000F000Fu, a[0][2 * h + 1] = w & 0x00F000F0u;
                                a[1][2 * h] = w8 & 0x000F000Fu, a[1][2 * h + 1] = w8 & 0x00F000F0u;
                            } else {
                                const uint32_t w = vw[h][2 * j], x = vw[h][2 * j + 1];
                                a[0][2 * h] = w & 0x00FF00FFu, a[0][2 * h + 1] = (w >> 8) & 0x00FF00FFu;
                                a[1][2 * h] = x & 0x00FF00FFu, a[1][2 * h + 1] = (x >> 8) & 0x00FF00FFu;
                            }
                        }
                        const uint32_t one = g == j ? kOffV : 0u; // row j of the offset's product
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            const float p0 = s[nt][0] * d0, p1 = s[nt][1] * d0, p2 = s[nt][2] * d1, p3 = s[nt][3] * d1;
                            const uint32_t h0 = pack_h2(p0, p1), h1 = pack_h2(p2, p3);
#pragma unroll
                            for (int p = 0; p < kParts; ++p) {
                                uint32_t x0 = h0, x1 = h1;
                                if (p == 1) {
                                    const float2 f0 = unpack_h2(h0), f1 = unpack_h2(h1);
                                    x0 = pack_h2(p0 - f0.x, p1 - f0.y), x1 = pack_h2(p2 - f1.x, p3 - f1.y);
                                }
                                const uint32_t b0 = movm(x0), b1 = movm(x1);
                                mma16816(o[nt][j][0], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
                                mma16816(o[nt][j][1], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
                                mma16816(off[nt], one, 0u, one, 0u, b0, b1);
                            }
                        }
                    }
                }
            }
            asm volatile("cp.async.wait_group 0;" ::: "memory");
            __syncthreads();                                      // every warp is done with its tiles
            // ---- the warps' sums side by side in shared memory
            float* mine = s_part + warp * attn_part_floats<J, NT>();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    constexpr float kUp = 16777216.f, kHigh = VB == 4 ? kUp / 16.f : kUp;
                    const float z0 = __shfl_sync(0xffffffffu, off[nt][0], 4 * j + t) * kUp, z1 = __shfl_sync(0xffffffffu, off[nt][1], 4 * j + t) * kUp;
                    const float(&x)[2][4] = o[nt][j];
                    float* p = mine + (8 * nt + 2 * t) * D + 32 * j + 4 * g;
                    *reinterpret_cast<float4*>(p) = make_float4(fmaf(x[0][0], kUp, -z0), fmaf(x[0][2], kHigh, -z0), fmaf(x[1][0], kUp, -z0), fmaf(x[1][2], kHigh, -z0));
                    *reinterpret_cast<float4*>(p + D) = make_float4(fmaf(x[0][1], kUp, -z1), fmaf(x[0][3], kHigh, -z1), fmaf(x[1][1], kUp, -z1), fmaf(x[1][3], kHigh, -z1));
                }
#pragma unroll
                for (int i = 0; i < 2; ++i) {
#pragma unroll
                    for (int w = 4; w < 32; w *= 2) sum[nt][i] += __shfl_xor_sync(0xffffffffu, sum[nt][i], w);
                    if (g == 0) {
                        mine[R * D + 8 * nt + 2 * t + i] = M[nt][i] - E;
                        mine[R * D + R + 8 * nt + 2 * t + i] = sum[nt][i];
                    }
                }
            }
        }
        // ---- and joined: the output, or this CTA's part of a cut segment
        const bool whole = todo == S.units, head_part = unit > 0;
        if (P.split && tid == 0 && !head_part) {                  // the segment starts here
            const long long end = u0 + S.units;                   // how many later CTAs work on it
            const int more = whole ? 0 : int(((end * ctas + total - 1) / total) - 1 - blockIdx.x);
            const int4 d = make_int4(int(blockIdx.x), whole || rows == 0 ? 0 : more + 1, b, seg);
            if (P.by_segment) P.desc[b * segs + seg] = d;
            else if (!whole) P.desc[blockIdx.x] = d, owns = true;
        }
        if (rows > 0) {
            __syncthreads();
            float* slot = P.parts + (2LL * blockIdx.x + (head_part ? 0 : 1)) * attn_part_floats<J, NT>();
            for (int i = tid; i < rows * (D / 4); i += 32 * kAttnWarps) {
                const int r = i / (D / 4), i0 = 4 * (i % (D / 4));
                float ref, weight;
                const float4 x = attn_join<D>(s_part, attn_part_floats<J, NT>(), kAttnWarps, r, R, i0, ref, weight);
                if (whole) {
                    attn_store<T>(P, S.row0, rt * R + r, group, hk, i0, x, weight);
                } else {
                    *reinterpret_cast<float4*>(slot + r * D + i0) = x;
                    if (i0 == 0) slot[R * D + r] = ref, slot[R * D + R + r] = weight;
                }
            }
            __syncthreads();
        }
        u0 += todo;
        unit = 0;
        if (u0 < u1 && ++seg == segs) {
            seg = 0;
            S = attn_seq(P, ++b, false);
        }
    }
    if (P.split) {
        if (!P.by_segment && tid == 0 && !owns) P.desc[blockIdx.x] = make_int4(0, 0, 0, 0);
        asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    }
}

// Joins the parts of cut segments: block (entry, row), four warps share the parts, a lane 4 values (8 for wide heads).
template <int DT, int J, int NT>
__global__ void __launch_bounds__(128) attn_join_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    constexpr int D = 32 * J, R = 8 * NT, F = attn_part_floats<J, NT>();
    __shared__ float4 s_o[4][D / 4];
    __shared__ float s_sum[4];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 d = P.desc[blockIdx.x];
    if (d.y == 0) return;
    const int group = P.n_heads / P.c.n_kv, hk = d.w / P.row_tiles, rt = d.w - hk * P.row_tiles;
    const AttnSeq S = attn_seq(P, d.z, false);
    const int r = blockIdx.y;
    if (rt * R + r >= min(S.n, P.max_new) * group) return;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // part k: the second slot of the segment's first CTA, then the first slots of the following ones
    auto part = [&](int k) { return P.parts + (2LL * (d.x + k) + (k == 0)) * F; };
    float ref = kAttnNone;
    for (int k = lane; k < d.y; k += 32) ref = fmaxf(ref, part(k)[R * D + r]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ref = fmaxf(ref, __shfl_xor_sync(0xffffffffu, ref, o));
    constexpr int V = (D + 127) / 128;
    float4 x[V];
    float sum = 0.f;
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = warp; k < d.y; k += 4) {
        const float* p = part(k);
        const float f = ex2(p[R * D + r] - ref);
        sum = fmaf(f, p[R * D + R + r], sum);
#pragma unroll
        for (int v = 0; v < V; ++v) {
            const int i = 128 * v + 4 * lane;
            if (i < D) {
                const float4 y = *reinterpret_cast<const float4*>(p + r * D + i);
                x[v].x = fmaf(f, y.x, x[v].x), x[v].y = fmaf(f, y.y, x[v].y), x[v].z = fmaf(f, y.z, x[v].z), x[v].w = fmaf(f, y.w, x[v].w);
            }
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (128 * v + 4 * lane < D) s_o[warp][32 * v + lane] = x[v];
    if (lane == 0) s_sum[warp] = sum;
    __syncthreads();
    for (int i = threadIdx.x; i < D / 4; i += 128) {
        float4 y = s_o[0][i];
        float w = s_sum[0];
#pragma unroll
        for (int k = 1; k < 4; ++k) {
            const float4 z = s_o[k][i];
            y = make_float4(y.x + z.x, y.y + z.y, y.z + z.z, y.w + z.w);
            w += s_sum[k];
        }
        attn_store<T>(P, S.row0, rt * R + r, group, hk, 4 * i, y, w);
    }
}

// ---- host -------------------------------------------------------------------------------------------

// Geometry of a call, the same for its workspace size and its launch.
struct AttnPlan {
    int nt, row_tiles, split, by_segment, grid, entries;
    long long part_bytes, bytes;          // workspace: parts, then desc
};
inline AttnPlan attn_plan(const KvView& c, int dtype, int n_heads, int n_seq, int max_new, int width, int window) {
    AttnPlan p{};
    const bool hl = dtype == QMV_OUT_F32, wide = c.J == 8;
    const long long rows = (long long)max_new * (n_heads / c.n_kv);
    p.nt = rows > 8 && !hl && !wide ? 2 : 1;
    p.row_tiles = int((rows + 8 * p.nt - 1) / (8 * p.nt));
    const long long segs = (long long)n_seq * c.n_kv * p.row_tiles;
    long long keys = (long long)width << c.page_shift;
    if (window > 0 && keys > (long long)window + max_new) keys = (long long)window + max_new + kAttnUnit;
    const long long units = (keys + kAttnUnit - 1) / kAttnUnit;   // of a segment, at most
    p.split = units > kAttnMinUnits;
    const long long most = p.split ? std::max((segs * units + kAttnMinUnits - 1) / kAttnMinUnits, segs) : segs;
    const int resident = sm_count() * (wide || p.nt == 2 ? 2 : hl ? 3 : 4);     // kAttnCtas
    p.grid = p.split ? int(std::min<long long>(most, resident)) : segs <= 0x7FFFFFFF ? int(segs) : 0;
    if (segs > 0x7FFFFFFF) p.grid = 0;                            // refused
    p.by_segment = p.split && segs <= p.grid;
    p.entries = p.by_segment ? int(segs) : p.grid;
    p.part_bytes = p.split ? 2LL * p.grid * (8LL * p.nt * (c.dim + 2)) * 4 : 0;
    p.part_bytes = (p.part_bytes + 255) / 256 * 256;
    p.bytes = p.part_bytes + (p.split ? 16LL * p.entries : 0) + 256;
    return p;
}

template <int DT, int J, int KB, int VB, int NT>
int attn_launch(const AttnParams& P, const AttnPlan& pl, cudaStream_t st) {
    const size_t smem = std::max(size_t(kAttnWarps) * attn_part_floats<J, NT>() * 4,
                                 size_t(kAttnWarps) * attn_stages<DT, J, KB, VB, NT>() * AttnTile<J, KB, VB>::kBytes);
    static SmemGrant grant;
    if (const int e = grant(attn_kernel<DT, J, KB, VB, NT>, smem)) return e;
    const int rc = launch_pdl_smem(attn_kernel<DT, J, KB, VB, NT>, dim3(pl.grid), dim3(32 * kAttnWarps), smem, st, P);
    if (rc || !pl.split) return rc;
    cudaLaunchConfig_t cfg = {};                                  // may start while the last parts are written
    cfg.gridDim = dim3(pl.entries, std::min<long long>(8 * NT, (long long)P.max_new * (P.n_heads / P.c.n_kv)));
    cfg.blockDim = dim3(128);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, attn_join_kernel<DT, J, NT>, P);
    return launched();
}

// every kernel of one head size (one translation unit each)
template <int J>
int attn_dispatch(const AttnParams& P, int dtype, const AttnPlan& pl, cudaStream_t st) {
    return by_elem(dtype, [&](auto c) {
        constexpr int DT = decltype(c)::value;
        auto pick = [&](auto kb, auto vb) {
            constexpr int KB = decltype(kb)::value, VB = decltype(vb)::value;
            if constexpr (J < 8 && DT != QMV_OUT_F32)
                if (pl.nt == 2) return attn_launch<DT, J, KB, VB, 2>(P, pl, st);
            return attn_launch<DT, J, KB, VB, 1>(P, pl, st);
        };
        using I4 = std::integral_constant<int, 4>;
        using I8 = std::integral_constant<int, 8>;
        if (P.c.kb == 4) return P.c.vb == 4 ? pick(I4{}, I4{}) : pick(I4{}, I8{});
        return P.c.vb == 4 ? pick(I8{}, I4{}) : pick(I8{}, I8{});
    });
}
extern template int attn_dispatch<2>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
extern template int attn_dispatch<3>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
extern template int attn_dispatch<4>(const AttnParams&, int, const AttnPlan&, cudaStream_t);
extern template int attn_dispatch<8>(const AttnParams&, int, const AttnPlan&, cudaStream_t);

}  // namespace qmv
