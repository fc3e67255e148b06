// Attention of few query rows over the quantised cache (layout: qmv_kv.cuh): decode steps, drafted tokens, and every call
// with fp32 queries.
//
//   s[r][key] = scale * sum_j d_k[key][j] * sum_{i in block j} q[r][i] code_k[key][i]
//   o[r][i]   = sum_key p[r][key] d_v[key][j(i)] code_v[key][i] / sum_key p[r][key],   p = 2^(s log2 e - ref)
//
// Bound by reading the cache once (4.5 or 8.5 bits a value), so what counts is instructions per value: at 6.5 TB/s an SM
// sees about 40 four-bit values a clock.  Both products run on mma.sync m16n8k16 (fp16 in, fp32 sums) with the cache as
// the 16-row operand, as it lies: the codes' bits ARE the operand.  A code c masked out of its word
// is the fp16 denormal c 2^-24 (16 c 2^-24 for the upper nibble of a byte, c 2^-18 for V's nibbles), which the tensor cores
// multiply exactly, so a 4-bit pair costs one AND (V's a shift too) and no conversion; these factors and the queries' 1 / 16 are folded
// into constants.
// (tcgen05 would need the unpacked values written to shared memory first, more bytes a clock than an SM writes.)  The codes'
// offset (8 or 128) comes out as its own term: in the scores it is the accumulator's start, -off sum_i q[i] per block,
// in the output one more product with a constant row a block.  (fp32 queries take it off the codes first: the term is many
// times the sum's size, and its rounding showed as 1e-5 of the result.)  Scales stay out of the products: d_k multiplies a block's
// 16 x 8 scores in fp32, d_v goes into p before it is rounded to fp16.
//
// Queries are fp16 after a power of two per row, which puts the largest at 2^14: bf16 values are exact down to 2^-31 of it, fp16's
// down to 2^-28, smaller ones are off by up to 2^-39 of it (those that meet the upper nibbles of 4-bit keys go in 1 / 16 as large:
// 2^-27, 2^-24, 2^-35); fp32 queries are two fp16 parts (HL), and so is p d_v then: 22 bits, down to 2^-35 of a row's largest
// product. (Second parts 2^11 times as large against codes 2^-11 times as large would go down to 2^-46; they take 44 us for one
// sequence of 65519 tokens where this takes 40.) The softmax reference only moves when a score passes it by 2^4 or a d_v the next
// power of two (checked with one vote a tile). p d_v is rounded to fp16 once: it stays below 2^15 and is 2^10 at least for the
// reference and the largest d_v, whatever V's size, so 2^-24 of that is still a normal number. (p as fp16 times d_v as fp16 took 3 %
// less for 64 sequences of bf16 queries, but holds no p large enough for a small d_v.) Sums and statistics are
// fp32.
//
// Work: units of 64 or 128 keys (one or two tiles of 16 a warp) of segments (sequence, key head, tile of 8 NT rows); the list of all units is cut into
// equal runs, one a CTA, so unequal lengths do not unbalance it.  A segment cut over several CTAs leaves its parts in the
// workspace and attn_join_kernel adds them in order.
#pragma once
#include <algorithm>
#include <climits>
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
    int split;                            // segments may be cut: parts, desc, attn_join_kernel follows (attn_tc_kernel: parts of a tile's keys)
    int by_segment;                       // desc has an entry a segment (else a CTA)
    float* parts;                         // [2 a CTA][8 NT rows][dim + 2]: sums, then reference and weight (attn_tc_kernel: its kPart a CTA)
    int4* desc;                           // two an entry: first part's CTA, parts (0: nothing to join), sequence's first row, key head;
                                          // first of the tile's rows, rows
    int* status;
};

constexpr int kAttnWarps = 4;
constexpr int kAttnMinKeys = 256;         // keys a CTA takes at least before segments are cut (128 and 512 took the same time)
constexpr float kAttnNone = -1e30f;       // reference of a row that has seen no key

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// d = a b + c with c somewhere else (no copy of it), and in place
__device__ __forceinline__ void mma16816(float (&d)[4], uint4 a, uint32_t b0, uint32_t b1, const float4& c) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%10, %11, %12, %13};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3]) : "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b0), "r"(b1), "f"(c.x), "f"(c.y), "f"(c.z), "f"(c.w));
}
__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }
__device__ __forceinline__ float2 unpack_h2(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }

// The four fp16 pairs of a code word (8 bits: of two), as the products' operands.  Plain: the codes' bits, denormals c 2^-24 (the
// upper nibbles 16 times that).  CENTRED: c - offset, exactly: an OR of fp16's 1024 gives 1024 + c, or 1024 + 16 c, and one
// operation takes the rest off.
template <int BYTES, bool CENTRED>
__device__ __forceinline__ void code_pairs(const uint32_t* w, uint32_t (&o)[4]) {
    if constexpr (BYTES == 4) {
        const uint32_t a = w[0], b = w[0] >> 8;
        if constexpr (CENTRED) {
            const __half2 low = __float2half2_rn(-1032.f), high = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
            o[0] = h2_bits(__hadd2(bits_h2((a & 0x000F000Fu) | 0x64006400u), low));
            o[1] = h2_bits(__hfma2(bits_h2((a & 0x00F000F0u) | 0x64006400u), sixteenth, high));
            o[2] = h2_bits(__hadd2(bits_h2((b & 0x000F000Fu) | 0x64006400u), low));
            o[3] = h2_bits(__hfma2(bits_h2((b & 0x00F000F0u) | 0x64006400u), sixteenth, high));
        } else {
            o[0] = a & 0x000F000Fu, o[1] = a & 0x00F000F0u, o[2] = b & 0x000F000Fu, o[3] = b & 0x00F000F0u;
        }
    } else {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const uint32_t a = w[i] & 0x00FF00FFu, b = (w[i] >> 8) & 0x00FF00FFu;
            if constexpr (CENTRED) {
                const __half2 low = __float2half2_rn(-1152.f);
                o[2 * i] = h2_bits(__hadd2(bits_h2(a | 0x64006400u), low)), o[2 * i + 1] = h2_bits(__hadd2(bits_h2(b | 0x64006400u), low));
            } else {
                o[2 * i] = a, o[2 * i + 1] = b;
            }
        }
    }
}

// V's four nibbles a half for the second product, each at bits 6 to 9: c 2^-18.  The tensor cores align a step's products at the largest
// exponent before they cut them off, and a denormal counts there as 2^-14, whatever its bits.  At c 2^-24 a step of 16 keys lost up to
// 2^-11 of a block's largest value (2^-16 on random data, all one way in the upper nibbles), at c 2^-18 2^-17; the
// shifts cost 3 % for 64 sequences.  K's codes stay as they are: the queries' signs keep what is cut off from adding up.
__device__ __forceinline__ void v_pairs(uint32_t w, uint32_t (&o)[4]) {
    o[0] = (w << 6) & 0x03C003C0u, o[1] = (w << 2) & 0x03C003C0u, o[2] = (w >> 2) & 0x03C003C0u, o[3] = (w >> 6) & 0x03C003C0u;
}

// f(std::integral_constant<int, 0>) .. of N
template <int N, int I = 0, class Fn>
__device__ __forceinline__ void each(Fn&& f) {
    if constexpr (I < N) {
        f(std::integral_constant<int, I>{});
        each<N, I + 1>(f);
    }
}

// N words of shared memory at a + O (aligned to N words' largest power of two up to 16 bytes; the constant part of an address
// stays out of the register), from pieces S bytes apart (16: side by side)
template <int N> constexpr int kPiece = N % 4 == 0 ? 4 : N % 2 == 0 ? 2 : 1;     // words of a load
template <int N, int O, int S = 0>
__device__ __forceinline__ void lds_words(uint32_t (&w)[N], uint32_t a) {
    constexpr int W = kPiece<N>;
    constexpr int step = S ? S : 4 * W;
    auto piece = [&](auto at) {
        constexpr int i = decltype(at)::value * W, o = O + decltype(at)::value * step;
        if constexpr (W == 4)
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4 + %5];" : "=r"(w[i]), "=r"(w[i + 1]), "=r"(w[i + 2]), "=r"(w[i + 3]) : "r"(a), "n"(o));
        else if constexpr (W == 2)
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2 + %3];" : "=r"(w[i]), "=r"(w[i + 1]) : "r"(a), "n"(o));
        else
            asm volatile("ld.shared.u32 %0, [%1 + %2];" : "=r"(w[i]) : "r"(a), "n"(o));
    };
    each<N / W>(piece);
}
// N words from global p + O to shared a + Q, in pieces 32 lanes' pieces apart, asynchronously
template <int N, int O, int Q>
__device__ __forceinline__ void copy_words(uint32_t a, const uint8_t* p) {
    constexpr int W = kPiece<N>;
    auto piece = [&](auto at) {
        constexpr int i = decltype(at)::value;
        if constexpr (W == 4)
            asm volatile("cp.async.cg.shared.global [%0 + %1], [%2 + %3], 16;" :: "r"(a), "n"(Q + 128 * W * i), "l"(p), "n"(O + 4 * W * i) : "memory");
        else
            asm volatile("cp.async.ca.shared.global [%0 + %1], [%2 + %3], %4;" :: "r"(a), "n"(Q + 128 * W * i), "l"(p), "n"(O + 4 * W * i), "n"(4 * W) : "memory");
    };
    each<N / W>(piece);
}
__device__ __forceinline__ void copy_bulk(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 :: "r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// A slot of the CTA's ring in shared memory: a unit's 4 KT tiles of 16 keys, KT a warp.  A lane (g = lane / 4, t = lane % 4)
// uses run t of the K rows of keys g and g + 8, run g of the V pairs t and t + 4, and the scales of keys 2 t, 2 t + 1, 2 t + 8
// and 2 t + 9.  The warps take turns in asking for a unit.  K and scales come as they lie, page by page in bulk copies; V's runs
// would meet on the same banks that way (four pairs, 128 bytes apart), so each lane copies the runs of its place, side by
// side with the other lanes'.  (Every warp asking for its own tiles took 72 of a tile's 313 instructions; V pair by pair in
// bulk, padded, 136: a bulk copy is one lane's.)
template <int J, int KB, int VB, int KT>
struct AttnSlot {
    static constexpr int kK = J * KB / 4, kV = J * VB / 4, kS = (J + 1) / 2;       // words of a lane's runs, of a key's K or V scales
    static constexpr int kRowK = 4 * J * KB, kRowV = 8 * J * VB, kRowS = 4 * J;    // bytes of a key, a pair, a key's scales
    static constexpr int kTiles = kAttnWarps * KT, kTileV = 256 * kV;
    static constexpr int kOffK = kTiles * kTileV, kOffS = kOffK + kTiles * 16 * kRowK, kBytes = kOffS + kTiles * 16 * kRowS;
    template <int X>
    static __device__ __forceinline__ void keys(uint32_t (&k)[2][kK], uint32_t at) {           // at: slot + lane_k
        lds_words<kK, kOffK + 16 * X * kRowK>(k[0], at);
        lds_words<kK, kOffK + (16 * X + 8) * kRowK>(k[1], at);
    }
    static __device__ __forceinline__ uint32_t lane_k(int warp, int g, int t) { return (16 * KT * warp + g) * kRowK + t * J * KB; }
    template <int X>
    static __device__ __forceinline__ void vals(uint32_t (&v)[2][kV], uint32_t at) {           // at: slot + KT warp tiles + lane_v
        lds_words<kV, kTileV * X, 128 * kPiece<kV>>(v[0], at);
        lds_words<kV, kTileV * X + 128 * kV, 128 * kPiece<kV>>(v[1], at);
    }
    static __device__ __forceinline__ uint32_t lane_v(int lane) { return 4 * kPiece<kV> * lane; }
    static __device__ __forceinline__ void copy_vals(uint32_t at, const uint8_t* from) {       // from: the tile's pair t, run g
        copy_words<kV, 0, 0>(at, from);
        copy_words<kV, 4 * kRowV, 128 * kV>(at, from);
    }
    // K's (V: V's) scale words of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 (J 3: the first of V's is half K's); at: slot + the warp's and 2 t rows
    template <int X, bool V>
    static __device__ __forceinline__ void scales(uint32_t (&sc)[4][kS], uint32_t at) {
        constexpr int o = kOffS + 16 * X * kRowS + (V ? 4 * (J - kS) : 0);
        if constexpr (J == 3) {                                   // rows of 12 bytes: word by word
            lds_words<1, o>(*reinterpret_cast<uint32_t(*)[1]>(sc[0]), at), lds_words<1, o + 4>(*reinterpret_cast<uint32_t(*)[1]>(sc[0] + 1), at);
            lds_words<1, o + 12>(*reinterpret_cast<uint32_t(*)[1]>(sc[1]), at), lds_words<1, o + 16>(*reinterpret_cast<uint32_t(*)[1]>(sc[1] + 1), at);
            lds_words<1, o + 96>(*reinterpret_cast<uint32_t(*)[1]>(sc[2]), at), lds_words<1, o + 100>(*reinterpret_cast<uint32_t(*)[1]>(sc[2] + 1), at);
            lds_words<1, o + 108>(*reinterpret_cast<uint32_t(*)[1]>(sc[3]), at), lds_words<1, o + 112>(*reinterpret_cast<uint32_t(*)[1]>(sc[3] + 1), at);
        } else {
            lds_words<kS, o>(sc[0], at), lds_words<kS, o + kRowS>(sc[1], at);
            lds_words<kS, o + 8 * kRowS>(sc[2], at), lds_words<kS, o + 9 * kRowS>(sc[3], at);
        }
    }
    // scale j of those words
    static __device__ __forceinline__ float scale(const uint32_t (&sc)[kS], int j, bool v) {
        const int i = j + (v ? J % 2 : 0);
        const __half2 h = bits_h2(sc[i >> 1]);
        return i & 1 ? __high2float(h) : __low2float(h);
    }
};
// Tiles of 16 keys a warp works on at once (two: each instruction has another that does not wait for it, and the loop's and
// the softmax's bookkeeping counts half; 64 sequences of 8191 keys, 8 heads of 128: 174 us, with one 220), keys a unit, CTAs
// an SM is to hold (heads of 64 or 96 values: three, 64 sequences of 8192 keys 112 and 142 us against 131 and 157 with two; of 128:
// two, whose registers hold everything, three spill, 101 us against 95 for 32 sequences of 8175 keys), and the units in a
// CTA's ring, within 227 KB an SM.
__host__ __device__ constexpr int attn_tiles(int J, int nt) { return J < 8 && nt == 1 ? 2 : 1; }
__host__ __device__ constexpr int attn_unit(int J, int nt) { return 16 * kAttnWarps * attn_tiles(J, nt); }
__host__ __device__ constexpr int attn_unit_bytes(int J, int kb, int vb, int nt) {
    return kAttnWarps * attn_tiles(J, nt) * 64 * J * (vb + kb + 1);
}
__host__ __device__ constexpr int attn_room(bool hl, int J, int nt, int ctas) {
    return (226 * 1024) / ctas - 1024 - J * 2048 - 256;      // less the fragments
}
__host__ __device__ constexpr int attn_ctas(bool hl, int J, int kb, int vb, int nt) {
    return J < 4 && nt == 1 && attn_room(hl, J, nt, 3) >= 2 * attn_unit_bytes(J, kb, vb, nt) ? 3 : 2;
}
__host__ __device__ constexpr int attn_stages(bool hl, int J, int kb, int vb, int nt) {
    const int n = attn_room(hl, J, nt, attn_ctas(hl, J, kb, vb, nt)) / attn_unit_bytes(J, kb, vb, nt);
    return n > 4 ? 4 : n;
}

template <int J, int NT>
__host__ __device__ constexpr int attn_part_floats() { return 8 * NT * (32 * J + 2); }

// where a unit lies: sequence, segment within it, unit within that; found once a CTA, then stepped
struct AttnSeq {
    int row0, n, len, first_unit, units;  // query rows, tokens in the cache, units of a segment
};
__device__ __forceinline__ AttnSeq attn_seq(const AttnParams& P, int b, bool report, int unit_keys) {
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
    s.first_unit = first / unit_keys;
    s.units = s.n == 0 ? 1 : max(1, (s.len + unit_keys - 1) / unit_keys - s.first_unit);
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
    store4_held(out, make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv));
}

template <int DT, int J, int KB, int VB, int NT>
__global__ void __launch_bounds__(32 * kAttnWarps, (attn_ctas(DT == QMV_OUT_F32, J, KB, VB, NT))) attn_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    constexpr bool HL = DT == QMV_OUT_F32;                       // queries and weights as two fp16 parts
    constexpr int D = 32 * J, R = 8 * NT, kParts = HL ? 2 : 1;
    constexpr float kOffK = KB == 4 ? 8.f : 128.f;
    constexpr uint32_t kOffV = VB == 4 ? 0x02000200u : 0x00800080u;
    constexpr int S_ = attn_stages(HL, J, KB, VB, NT), KT = attn_tiles(J, NT), kUnit = attn_unit(J, NT);
    using Slot = AttnSlot<J, KB, VB, KT>;
    static_assert(Slot::kBytes == attn_unit_bytes(J, KB, VB, NT), "the launch's shared memory");
    extern __shared__ __align__(16) float s_part[];              // the warps' tiles [warps][S_]; then [warps][R (D + 2)]
    constexpr bool two = HL || NT == 2;                          // the scores' rows g + 8 are used
    // per block and lane, whole operands (put together in registers they cost a move a word): the queries of the two k steps, the
    // scores' start, and the row of the offset's product
    __shared__ uint4 s_q[J][2][32], s_one[J][32];
    __shared__ float4 s_start[J][32];
    __shared__ long long s_scan[kAttnWarps + 1];
    __shared__ uint64_t s_bar[2][4];
    __shared__ uint32_t s_held[4];                               // the unit's runs of keys in one page that were copied, a bit each
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    const uint32_t full0 = smem_u32(s_bar[0]), empty0 = smem_u32(s_bar[1]), ring = smem_u32(s_part);
    if (tid == 0) {
        for (int i = 0; i < S_; ++i) mbar_init(full0 + 8 * i, 33), mbar_init(empty0 + 8 * i, kAttnWarps);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    // slots of the next unit to work on and to ask for, and the phase of its full (its empty, the one before) barrier
    constexpr int kAhead = S_ > 2 ? S_ - 2 : 1;                  // units asked for ahead: S_ - 2 leaves the other warps a unit's time
    int slot = 0, slot_in = 0;
    uint32_t phase = 0, phase_in = 1;
    bool dead = false;                                            // a copy did not come in time: this warp takes no more units
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");      // the join finds room as CTAs leave, and waits for the last
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int group = P.n_heads / P.c.n_kv, segs = P.c.n_kv * P.row_tiles;

    // ---- this CTA's run of units: the list's length, and the sequence that holds the run's first one
    long long total = 0, u0 = 0, u1 = 0;
    int ctas = gridDim.x, b = 0, seg = 0, unit = 0;               // sequence, segment, unit: the next one
    AttnSeq S;
    if (P.split) {
        long long before = 0;                                     // units of earlier sequences
        if (P.n_seq == 1) {
            S = attn_seq(P, 0, blockIdx.x == 0 && tid == 0, kUnit);
            total = (long long)S.units * segs;
        } else {
            // sequences 128 at a time, a thread each; one round of them is looked at once
            long long x = 0, inc = 0;
            for (int b0 = 0; b0 < P.n_seq; b0 += 32 * kAttnWarps) {
                x = b0 + tid < P.n_seq ? (long long)attn_seq(P, b0 + tid, blockIdx.x == 0, kUnit).units * segs : 0;
                inc = x;
#pragma unroll
                for (int o = 1; o < 32; o *= 2) {
                    const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                    if (lane >= o) inc += y;
                }
                if (b0) __syncthreads();
                if (lane == 31) s_scan[warp] = inc;
                __syncthreads();
#pragma unroll
                for (int w = 0; w < kAttnWarps; ++w) {
                    if (w < warp) inc += s_scan[w];
                    total += s_scan[w];
                }
            }
            const long long most = max((total + kAttnMinKeys / kUnit - 1) / (kAttnMinKeys / kUnit), (long long)P.n_seq * segs);
            if (most < ctas) ctas = int(most);
            const long long first_u = total * blockIdx.x / ctas;
            __syncthreads();
            if (P.n_seq <= 32 * kAttnWarps) {
                if (inc - x <= first_u && first_u < inc) s_scan[0] = tid, s_scan[1] = inc - x;
                __syncthreads();
            } else if (blockIdx.x < ctas) {
                long long base = 0;
                for (int b0 = 0; b0 < P.n_seq; b0 += 32 * kAttnWarps) {
                    x = b0 + tid < P.n_seq ? (long long)attn_seq(P, b0 + tid, false, kUnit).units * segs : 0;
                    inc = x;
#pragma unroll
                    for (int o = 1; o < 32; o *= 2) {
                        const long long y = __shfl_up_sync(0xffffffffu, inc, o);
                        if (lane >= o) inc += y;
                    }
                    if (lane == 31) s_scan[warp] = inc;
                    __syncthreads();
                    long long all = base;
                    inc += base;
#pragma unroll
                    for (int w = 0; w < kAttnWarps; ++w) {
                        if (w < warp) inc += s_scan[w];
                        all += s_scan[w];
                    }
                    __syncthreads();
                    if (first_u < all) {                          // the same for every thread
                        if (inc - x <= first_u && first_u < inc) s_scan[0] = b0 + tid, s_scan[1] = inc - x;
                        __syncthreads();
                        break;
                    }
                    base = all;
                }
            }
            b = int(s_scan[0]);
            before = s_scan[1];
        }
        const long long most = max((total + kAttnMinKeys / kUnit - 1) / (kAttnMinKeys / kUnit), (long long)P.n_seq * segs);
        if (most < ctas) ctas = int(most);
        if (blockIdx.x >= ctas) {
            if (tid == 0 && !P.by_segment) P.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
            return;
        }
        u0 = total * blockIdx.x / ctas, u1 = total * (blockIdx.x + 1) / ctas;
        if (P.n_seq > 1) S = attn_seq(P, b, false, kUnit);
        const long long in = u0 - before;
        seg = int(in / S.units), unit = int(in - (long long)seg * S.units);
    } else {                                                      // one CTA a segment
        b = blockIdx.x / segs, seg = blockIdx.x - b * segs;
        S = attn_seq(P, b, seg == 0 && tid == 0, kUnit);
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
        // every row sees keys seen0 .. seen1
        const int seen0 = P.window > 0 ? max(0, pos0 + tok1 - P.window + 1) : 0, seen1 = pos0 + tok0;

        float cs[NT], M[NT], rn[NT], sum[NT], o[NT][J][2][4], off[NT][4];        // of rows g, g + 8; o, off: columns 2 t, 2 t + 1
        int pos[NT];
        float top_p = 0.f;                                        // log2 of the largest p allowed
        uint32_t lim = 0u;                                        // ... while every |d_v| is at most this (two fp16)
        if (rows > 0) {
            // ---- the units' copies; the first ones start before the queries are looked at
            const int turns = dead ? 0 : todo;
            const int* table = P.tables + (long long)b * P.width;
            const int key0 = (S.first_unit + unit) * kUnit;
            const uint32_t lane_k = Slot::lane_k(warp, g, t), lane_v = KT * warp * Slot::kTileV + Slot::lane_v(lane),
                           lane_s = (16 * KT * warp + 2 * t) * Slot::kRowS;
            const int shift = P.c.page_shift, in_page = (1 << shift) - 1;
            constexpr int kUnitShift = kUnit == 64 ? 6 : 7;
            const int run = min(shift, kUnitShift), runs = 1 << (kUnitShift - run);         // log2 of a run's keys, runs a unit
            // this key head's rows of page 0, this lane's V run of it, and the bytes between pages
            const uint8_t* head_k = P.c.k + ((long long)hk << shift) * Slot::kRowK;
            const uint8_t* head_v = P.c.v + ((long long)hk << (shift - 1)) * Slot::kRowV + t * Slot::kRowV + g * J * VB;
            const uint8_t* head_s = reinterpret_cast<const uint8_t*>(P.c.sc) + ((long long)hk << shift) * Slot::kRowS;
            const uint32_t page_k = uint32_t(P.c.n_kv * Slot::kRowK) << shift, page_v = uint32_t(P.c.n_kv * Slot::kRowV) << (shift - 1),
                           page_s = uint32_t(P.c.n_kv * Slot::kRowS) << shift;
            constexpr int kNoKey = INT_MIN;                       // nothing to see there
            auto look = [&](int u) {                              // lane c: the page of unit u's run c
                const int key = key0 + u * kUnit + (lane << run);
                return u < turns && lane < runs && key <= last && key + (1 << run) > first ? __ldg(table + (key >> shift)) : kNoKey;
            };
            auto ask = [&](int u, int entry) {                    // one warp: starts the copies of unit u into slot_in
                const bool there = entry >= 0 && entry < P.c.n_pages;
                if (!there && entry != kNoKey && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
                const uint32_t mask = __ballot_sync(0xffffffffu, there), full = full0 + 8 * slot_in;
                if (!__all_sync(0xffffffffu, mbar_wait(empty0 + 8 * slot_in, phase_in))) {
                    if (lane == 0 && P.status) atomicOr(P.status, DEV_TIMEOUT);
                    return;                                       // the unit never gets full: every warp gives up there
                }
                const uint32_t to = ring + slot_in * Slot::kBytes;
                if (lane == 0) {
                    s_held[slot_in] = mask;
                    mbar_arrive_tx(full, __popc(mask) * ((Slot::kRowK + Slot::kRowS) << run));
                }
                const int at = (key0 + u * kUnit) & in_page;      // within a page that holds the whole unit (else 0)
                for (int c = 0; c < runs; ++c) {
                    if (!(mask >> c & 1u)) continue;
                    const uint32_t page = __shfl_sync(0xffffffffu, entry, c);
                    const int first_key = c << run;
                    if (lane == 0) {
                        copy_bulk(to + Slot::kOffK + first_key * Slot::kRowK, head_k + (unsigned long long)page * page_k + at * Slot::kRowK, Slot::kRowK << run, full);
                        copy_bulk(to + Slot::kOffS + first_key * Slot::kRowS, head_s + (unsigned long long)page * page_s + at * Slot::kRowS, Slot::kRowS << run, full);
                    }
                    const uint8_t* from = head_v + (unsigned long long)page * page_v + (at >> 1) * Slot::kRowV;
                    uint32_t dst = to + (first_key >> 4) * Slot::kTileV + Slot::lane_v(lane);
#pragma unroll 4
                    for (int x = 0; x < 1 << (run - 4); ++x, from += 8 * Slot::kRowV, dst += Slot::kTileV) Slot::copy_vals(dst, from);
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(full) : "memory");
            };
            auto next_in = [&]() {
                if (++slot_in == S_) slot_in = 0, phase_in ^= 1u;
            };
            int entry = look(warp);                               // of the next unit this warp asks for: warp, warp + 4, ...
#pragma unroll
            for (int u = 0; u < kAhead; ++u)
                if (u < turns) {
                    if ((u & (kAttnWarps - 1)) == warp) {
                        ask(u, entry);
                        entry = look(u + kAttnWarps);
                    }
                    next_in();
                }
            // Queries, scaled to fp16 by a power of two per row: lane (g, t) holds values 8 t .. 8 t + 7 of each block of row g
            // as the product's rows g, and as rows g + 8 the second parts (HL) or row g + 8 (NT 2)
            uint32_t part[2][J][2][2];                            // [rows g / g + 8][block][k step][half]
            float start[NT][J];
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
                const int e = ex == 0 || ex == 255 ? 0 : max(-120, ex - 127 - 14);
                // the scale's sign goes into the queries: cs is positive, and masked scores stay -inf
                const float down = __uint_as_float((uint32_t(127 - e) << 23) | (P.scale < 0.f ? 0x80000000u : 0u));
                // (2^e first, in halves: a scale near fp32's end times 2^24 would pass it though its queries are as small)
                const float up = __uint_as_float(uint32_t(127 + e / 2) << 23);
                cs[nt] = fmaxf(fabsf(P.scale) * 1.4426950408889634f * up * (HL ? 1.f : 16777216.f) * __uint_as_float(uint32_t(127 + e - e / 2) << 23), 1e-30f);
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    float all = 0.f;
#pragma unroll
                    for (int m = 0; m < 2; ++m) {
                        constexpr float kHigh = KB == 4 && !HL ? 1.f / 16.f : 1.f;      // the upper nibbles arrive 16 times too large
                        const float a = x[j][m].x * down, b2 = x[j][m].y * down, c = x[j][m].z * down * kHigh, d = x[j][m].w * down * kHigh;
                        const uint32_t lo = pack_h2(a, b2), hi = pack_h2(c, d);
                        const float2 fl = unpack_h2(lo), fh = unpack_h2(hi);
                        all += (fl.x + fl.y) + (fh.x + fh.y) * (1.f / kHigh);
                        part[nt][j][m][0] = lo, part[nt][j][m][1] = hi;
                        if constexpr (HL) {
                            const uint32_t lo2 = pack_h2(a - fl.x, b2 - fl.y), hi2 = pack_h2(c - fh.x, d - fh.y);
                            const float2 gl = unpack_h2(lo2), gh = unpack_h2(hi2);
                            all += (gl.x + gl.y) + (gh.x + gh.y) * (1.f / kHigh);
                            part[1][j][m][0] = lo2, part[1][j][m][1] = hi2;
                        }
                    }
                    all += __shfl_xor_sync(0xffffffffu, all, 1);
                    all += __shfl_xor_sync(0xffffffffu, all, 2);
                    start[nt][j] = HL ? 0.f : all * (-kOffK * 5.9604644775390625e-8f);
#pragma unroll
                    for (int m = 0; m < 2; ++m)
#pragma unroll
                        for (int i = 0; i < 4; ++i) o[nt][j][m][i] = 0.f;
                }
                M[nt] = kAttnNone, rn[nt] = -kAttnNone, sum[nt] = 0.f;
                pos[nt] = pos0 + (rt * R + min(r, rows - 1)) / group;
#pragma unroll
                for (int i = 0; i < 4; ++i) off[nt][i] = 0.f;
            }
            if (warp == 0) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
#pragma unroll
                    for (int m = 0; m < 2; ++m)
                        s_q[j][m][lane] = make_uint4(part[0][j][m][0], two ? part[1][j][m][0] : 0u, part[0][j][m][1], two ? part[1][j][m][1] : 0u);
                    const float second = NT == 2 ? start[NT - 1][j] : 0.f;
                    s_start[j][lane] = make_float4(start[0][j], start[0][j], second, second);
                    if (!HL) s_one[j][lane] = make_uint4(g == j ? kOffV : 0u, 0u, g == j ? kOffV : 0u, 0u);
                }
            }
            __syncthreads();
            for (int u = 0; u < turns; ++u) {
                const int key = key0 + u * kUnit + 16 * KT * warp;        // this warp's first key
                if (u + kAhead < turns) {
                    if (((u + kAhead) & (kAttnWarps - 1)) == warp) {
                        ask(u + kAhead, entry);
                        entry = look(u + kAhead + kAttnWarps);
                    }
                    next_in();
                }
                const uint32_t buf = ring + slot * Slot::kBytes, empty = empty0 + 8 * slot;
                if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * slot, phase))) {
                    // a copy did not come in time: say so and take no more units (the other warps find the same)
                    dead = true;
                    if (lane == 0 && P.status) atomicOr(P.status, DEV_TIMEOUT);
                    break;
                }
                const uint32_t mask = s_held[slot];
                uint32_t here = 0;                                // bit x: tile x is there and some row sees some of it
#pragma unroll
                for (int x = 0; x < KT; ++x)
                    if (mask >> ((16 * (KT * warp + x)) >> run) & 1u && key + 16 * x <= last && key + 16 * x + 15 >= first) here |= 1u << x;
                if (++slot == S_) slot = 0, phase ^= 1u;
                // A unit that some row does not see whole is masked key by key, in a copy of the code: in one, the masks were
                // predicated instructions that every unit paid for (100 of a tile's 440)
                auto work = [&](auto all_of_it) {
                constexpr bool whole = decltype(all_of_it)::value;
                // scores: C rows g / g + 8 = query rows (or their second parts), columns 2 t, 2 t + 1 = keys, of two 8-key tiles
                float s[KT][NT][4];
                uint32_t dv = 0;                                  // |d_v| as two fp16, every one of the unit's in some lane
                uint32_t kw[KT][2][Slot::kK], sk[KT][4][Slot::kS];         // scales of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9
                each<KT>([&](auto x) {
                    Slot::template keys<decltype(x)::value>(kw[decltype(x)::value], buf + lane_k);
                    Slot::template scales<decltype(x)::value, false>(sk[decltype(x)::value], buf + lane_s);
                });
#pragma unroll
                for (int x = 0; x < KT; ++x) {
                    // the words that hold V's scales: J / 2 a key (J 3: two, the first of them half K's)
                    constexpr int kPer = Slot::kS, kFirst = J - kPer;
#pragma unroll
                    for (int i = 0; i < 16 * kPer; i += 32) {
                        const int w = i + lane, key_w = w / kPer, at = kFirst + w % kPer;
                        if (16 * kPer % 32 == 0 || w < 16 * kPer)
                            if (whole || (here >> x & 1u && uint32_t(key + 16 * x + key_w - first) <= uint32_t(last - first)))
                                dv = __vmaxu2(dv, lds32(buf + Slot::kOffS + ((16 * (KT * warp + x) + key_w) * J + at) * 4) & (J % 2 && at == kFirst ? 0x7FFF0000u : 0x7FFF7FFFu));
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) s[x][nt][i] = 0.f;
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const uint4 q0 = s_q[j][0][lane], q1 = s_q[j][1][lane];
                    const float4 begin = s_start[j][lane];
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int y = 0; y < 2; ++y) {
                            uint32_t k[4];
                            code_pairs<KB, HL>(&kw[x][y][j * KB / 4], k);
                            float c[4];
                            mma16816(c, q0, k[0], k[1], begin);
                            mma16816(c, q1.x, q1.y, q1.z, q1.w, k[2], k[3]);
                            const float d0 = Slot::scale(sk[x][2 * y], j, false), d1 = Slot::scale(sk[x][2 * y + 1], j, false);
                            if (HL) c[0] += c[2], c[1] += c[3];
                            s[x][0][2 * y] = fmaf(d0, c[0], s[x][0][2 * y]), s[x][0][2 * y + 1] = fmaf(d1, c[1], s[x][0][2 * y + 1]);
                            if (NT == 2)
                                s[x][NT - 1][2 * y] = fmaf(d0, c[2], s[x][NT - 1][2 * y]), s[x][NT - 1][2 * y + 1] = fmaf(d1, c[3], s[x][NT - 1][2 * y + 1]);
                        }
                }
                uint32_t gone = 0;                                // bit 4 x + i: key i of tile x is nobody's
                if constexpr (!whole) {
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int k = key + 16 * x + 2 * t + (i & 1) + 8 * (i >> 1);
                            const bool there = here >> x & 1u && uint32_t(k - first) <= uint32_t(last - first);
                            if (!there) gone |= 1u << (4 * x + i);
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                if (!there || k > pos[nt] || (P.window > 0 && pos[nt] - k >= P.window)) s[x][nt][i] = -INFINITY;
                        }
                }
                // p = 2^(s cs + rn); the references move only if some p or d_v would pass its limit
                float p[KT][NT][4], top = kAttnNone;
                auto weigh = [&]() {
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < 4; ++i) p[x][nt][i] = fmaf(s[x][nt][i], cs[nt], rn[nt]);
                };
                weigh();
#pragma unroll
                for (int x = 0; x < KT; ++x)
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) top = fmaxf(top, p[x][nt][i]);
                if (__any_sync(0xffffffffu, top > top_p || __vmaxu2(dv, lim) != lim)) {
                    dv = __reduce_max_sync(0xffffffffu, max(dv >> 16, dv & 0xFFFFu));
                    if (dv > (lim & 0xFFFFu)) {                   // the next power of two, 2^(ev - 14); times 2^top_p it is 2^15
                        const int bits = 31 - __clz(dv), ev = dv < 1024u ? bits - 9 : int(dv >> 10);        // (below 2^-14 denormal)
                        lim = (dv < 1024u ? 2u << bits : min(uint32_t(ev + 1) << 10, 0x7BFFu)) * 0x10001u;
                        top_p = float(29 - ev);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float m = -INFINITY;
#pragma unroll
                        for (int x = 0; x < KT; ++x) m = fmaxf(m, fmaxf(fmaxf(s[x][nt][0], s[x][nt][1]), fmaxf(s[x][nt][2], s[x][nt][3])));
                        m *= cs[nt];
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
                        m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
                        M[nt] = fmaxf(M[nt], m);
                        const float n = top_p - 4.f - M[nt], f = ex2(n - rn[nt]);
                        rn[nt] = n;
                        sum[nt] *= f;
                        const float f0 = __shfl_sync(0xffffffffu, f, 8 * t), f1 = __shfl_sync(0xffffffffu, f, 8 * t + 4);
                        off[nt][0] *= f0, off[nt][1] *= f1;
#pragma unroll
                        for (int j = 0; j < J; ++j)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                o[nt][j][h][0] *= f0, o[nt][j][h][1] *= f1;
                                o[nt][j][h][2] *= f0, o[nt][j][h][3] *= f1;
                            }
                    }
                    weigh();
                }
                uint32_t vw[KT][2][Slot::kV], sv[KT][4][Slot::kS];
#pragma unroll
                for (int x = 0; x < KT; ++x) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) p[x][nt][i] = ex2(p[x][nt][i]);
                        sum[nt] += (p[x][nt][0] + p[x][nt][1]) + (p[x][nt][2] + p[x][nt][3]);
                    }
                }
                each<KT>([&](auto x) {
                    Slot::template vals<decltype(x)::value>(vw[decltype(x)::value], buf + lane_v);
                    Slot::template scales<decltype(x)::value, true>(sv[decltype(x)::value], buf + lane_s);
                });
                if (!whole) {                                     // keys nobody sees hold anything (NaN scales too): 0 times 0
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
#pragma unroll
                            for (int w = 0; w < Slot::kS; ++w) sv[x][i][w] = gone >> (4 * x + i) & 1u ? 0u : sv[x][i][w];
                }
                // output: rows = values g / g + 8 of two tiles a block, k = keys, columns = query rows: the scores' layout is that of
                // the second operand already
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    [[maybe_unused]] const uint4 one = s_one[j][lane];       // row j of the offset's product
#pragma unroll
                    for (int x = 0; x < KT; ++x) {
                        uint32_t a[2][4];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {             // pair t (k 2 t, 2 t + 1), pair t + 4 (k 8 + 2 t, 9 + 2 t)
                            uint32_t v[4];
                            if constexpr (VB == 4 && !HL) v_pairs(vw[x][h][j], v);
                            else code_pairs<VB, HL>(&vw[x][h][j * VB / 4], v);
                            a[0][2 * h] = v[0], a[0][2 * h + 1] = v[1], a[1][2 * h] = v[2], a[1][2 * h + 1] = v[3];
                        }
                        float d[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) d[i] = Slot::scale(sv[x][i], j, true);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            uint32_t bw[2], low[2];
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const float p0 = p[x][nt][2 * y] * d[2 * y], p1 = p[x][nt][2 * y + 1] * d[2 * y + 1];
                                bw[y] = pack_h2(p0, p1);
                                if (HL) {
                                    const float2 f = unpack_h2(bw[y]);
                                    low[y] = pack_h2(p0 - f.x, p1 - f.y);
                                }
                            }
#pragma unroll
                            for (int z = 0; z < kParts; ++z) {
                                const uint32_t b0 = z ? low[0] : bw[0], b1 = z ? low[1] : bw[1];
                                mma16816(o[nt][j][0], a[0][0], a[0][1], a[0][2], a[0][3], b0, b1);
                                mma16816(o[nt][j][1], a[1][0], a[1][1], a[1][2], a[1][3], b0, b1);
                                if constexpr (!HL) mma16816(off[nt], one.x, one.y, one.z, one.w, b0, b1);
                            }
                        }
                    }
                }
                };
                if (here == (1u << KT) - 1u && key >= seen0 && key + 16 * KT - 1 <= seen1) work(std::true_type{});
                else if (here) work(std::false_type{});
                __syncwarp();
                if (lane == 0) mbar_arrive(empty);                // the slot may be filled again
            }
            __syncthreads();                                      // every warp is done with its tiles
            // ---- the warps' sums side by side in shared memory
            float* own = s_part + warp * attn_part_floats<J, NT>();
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    constexpr float kUp = HL ? 1.f : VB == 4 ? 262144.f : 16777216.f;
                    const float z0 = __shfl_sync(0xffffffffu, off[nt][0], 4 * j + t) * kUp, z1 = __shfl_sync(0xffffffffu, off[nt][1], 4 * j + t) * kUp;
                    const float(&x)[2][4] = o[nt][j];
                    float* p = own + (8 * nt + 2 * t) * D + 32 * j + 4 * g;
                    *reinterpret_cast<float4*>(p) = make_float4(fmaf(x[0][0], kUp, -z0), fmaf(x[0][2], kUp, -z0), fmaf(x[1][0], kUp, -z0), fmaf(x[1][2], kUp, -z0));
                    *reinterpret_cast<float4*>(p + D) = make_float4(fmaf(x[0][1], kUp, -z1), fmaf(x[0][3], kUp, -z1), fmaf(x[1][1], kUp, -z1), fmaf(x[1][3], kUp, -z1));
                }
                sum[nt] += __shfl_xor_sync(0xffffffffu, sum[nt], 1);
                sum[nt] += __shfl_xor_sync(0xffffffffu, sum[nt], 2);
                if (t == 0) own[R * D + 8 * nt + g] = -rn[nt], own[R * D + R + 8 * nt + g] = sum[nt];
            }
        }
        // ---- and joined: the output, or this CTA's part of a cut segment
        const bool whole = todo == S.units, head_part = unit > 0;
        if (P.split && tid == 0 && !head_part) {                  // the segment starts here
            const long long end = u0 + S.units;                   // how many later CTAs work on it
            const int more = whole ? 0 : int(((end * ctas + total - 1) / total) - 1 - blockIdx.x);
            const int at = P.by_segment ? b * segs + seg : int(blockIdx.x);
            if (P.by_segment || !whole) {
                P.desc[2 * at] = make_int4(int(blockIdx.x), whole ? 0 : more + 1, S.row0, hk);
                P.desc[2 * at + 1] = make_int4(rt * R, rows, 0, 0);
                owns = true;
            }
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
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // these uses come before the next segment's copies
            __syncthreads();
        }
        u0 += todo;
        unit = 0;
        if (u0 < u1 && ++seg == segs) {
            seg = 0;
            S = attn_seq(P, ++b, false, kUnit);
        }
    }
    if (dead) {                                                   // copies of units asked for ahead may still be on their way here
        for (int i = 0; i <= kAhead; ++i) {
            mbar_wait(full0 + 8 * slot, phase);                   // bounded too
            if (++slot == S_) slot = 0, phase ^= 1u;
        }
        asm volatile("cp.async.wait_all;" ::: "memory");
    }
    if (P.split && !P.by_segment && tid == 0 && !owns) P.desc[2 * blockIdx.x] = make_int4(0, 0, 0, 0);
}

// Joins the parts of cut segments, in their order: block (entry, row), eight warps share the parts, a lane 4 values (8 of
// wide heads).  A chain of three dependent reads: the entry, then references, weights and sums of up to four parts a warp at once.
template <int DT, int J, int NT>
__global__ void __launch_bounds__(256) attn_join_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    constexpr int D = 32 * J, R = 8 * NT, F = attn_part_floats<J, NT>(), W = 8, V = (D + 127) / 128, B = 4;
    __shared__ float4 s_o[W][D / 4];
    __shared__ float s_ref[W], s_sum[W];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int4 d = P.desc[2 * blockIdx.x], e = P.desc[2 * blockIdx.x + 1];
    const int r = blockIdx.y;
    if (d.y == 0 || r >= e.y) return;
    const int group = P.n_heads / P.c.n_kv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    float ref = kAttnNone, sum = 0.f;
    float4 o[V];
#pragma unroll
    for (int v = 0; v < V; ++v) o[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k0 = warp; k0 < d.y; k0 += W * B) {                  // B parts in flight; each warp at its own reference
        float rk[B], wk[B];
        float4 x[B][V];
#pragma unroll
        for (int q = 0; q < B; ++q) {
            const int k = k0 + W * q;
            // part k: the second slot of the segment's first CTA, then the first slots of the following ones
            const float* p = P.parts + (2LL * (d.x + k) + (k == 0)) * F;
            const bool there = k < d.y;
            rk[q] = there ? p[R * D + r] : kAttnNone;
            wk[q] = there ? p[R * D + R + r] : 0.f;
#pragma unroll
            for (int v = 0; v < V; ++v)
                x[q][v] = there && 128 * v + 4 * lane < D ? *reinterpret_cast<const float4*>(p + r * D + 128 * v + 4 * lane) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
        float top = ref;
#pragma unroll
        for (int q = 0; q < B; ++q) top = fmaxf(top, rk[q]);
        const float f = ex2(ref - top);
        ref = top;
        sum *= f;
#pragma unroll
        for (int v = 0; v < V; ++v) o[v] = make_float4(o[v].x * f, o[v].y * f, o[v].z * f, o[v].w * f);
#pragma unroll
        for (int q = 0; q < B; ++q) {
            const float w = ex2(rk[q] - ref);
            sum = fmaf(w, wk[q], sum);
#pragma unroll
            for (int v = 0; v < V; ++v)
                o[v] = make_float4(fmaf(w, x[q][v].x, o[v].x), fmaf(w, x[q][v].y, o[v].y), fmaf(w, x[q][v].z, o[v].z), fmaf(w, x[q][v].w, o[v].w));
        }
    }
#pragma unroll
    for (int v = 0; v < V; ++v)
        if (128 * v + 4 * lane < D) s_o[warp][32 * v + lane] = o[v];
    if (lane == 0) s_ref[warp] = ref, s_sum[warp] = sum;
    __syncthreads();
    for (int i = threadIdx.x; i < D / 4; i += 32 * W) {
        float top = s_ref[0];
#pragma unroll
        for (int k = 1; k < W; ++k) top = fmaxf(top, s_ref[k]);
        float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
        float w = 0.f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            const float f = ex2(s_ref[k] - top);
            const float4 z = s_o[k][i];
            y = make_float4(fmaf(f, z.x, y.x), fmaf(f, z.y, y.y), fmaf(f, z.z, y.z), fmaf(f, z.w, y.w));
            w = fmaf(f, s_sum[k], w);
        }
        attn_store<T>(P, d.z, e.x + r, group, d.w, 4 * i, y, w);
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
    const bool hl = dtype == QMV_OUT_F32;
    const long long rows = (long long)max_new * (n_heads / c.n_kv);
    // Two tiles of 8 rows share a cache tile's unpacked words (8 sequences of 4096 keys, 8 heads of 128: 16 rows 34 us against 36);
    // not where their sums do not fit the registers (heads of 256) or both parts of fp32 queries use the rows.
    p.nt = rows > 8 && !hl && c.J < 8 ? 2 : 1;
    p.row_tiles = int((rows + 8 * p.nt - 1) / (8 * p.nt));
    const long long segs = (long long)n_seq * c.n_kv * p.row_tiles;
    const int unit = attn_unit(c.J, p.nt), least = kAttnMinKeys / unit;
    long long keys = (long long)width << c.page_shift;
    if (window > 0 && keys > (long long)window + max_new) keys = (long long)window + max_new + unit;
    const long long units = (keys + unit - 1) / unit;             // of a segment, at most
    p.split = units > least;
    const long long most = p.split ? std::max((segs * units + least - 1) / least, segs) : segs;
    const int resident = sm_count() * attn_ctas(hl, c.J, c.kb, c.vb, p.nt);
    p.grid = p.split ? int(std::min<long long>(most, resident)) : segs <= 0x7FFFFFFF ? int(segs) : 0;
    if (segs > 0x7FFFFFFF) p.grid = 0;                            // refused
    p.by_segment = p.split && segs <= p.grid;
    p.entries = p.by_segment ? int(segs) : p.grid;
    p.part_bytes = p.split ? 2LL * p.grid * (8LL * p.nt * (c.dim + 2)) * 4 : 0;
    p.part_bytes = (p.part_bytes + 255) / 256 * 256;
    p.bytes = p.part_bytes + (p.split ? 32LL * p.entries : 0) + 256;
    return p;
}

template <int DT, int J, int KB, int VB, int NT>
int attn_launch(const AttnParams& P, const AttnPlan& pl, cudaStream_t st) {
    const size_t smem = std::max(size_t(kAttnWarps) * attn_part_floats<J, NT>() * 4,
                                 size_t(attn_stages(DT == QMV_OUT_F32, J, KB, VB, NT)) * attn_unit_bytes(J, KB, VB, NT));
    static SmemGrant grant;
    if (const int e = grant(attn_kernel<DT, J, KB, VB, NT>, smem)) return e;
    const int rc = launch_pdl_smem(attn_kernel<DT, J, KB, VB, NT>, dim3(pl.grid), dim3(32 * kAttnWarps), smem, st, P);
    if (rc || !pl.split) return rc;
    cudaLaunchConfig_t cfg = {};                                  // may start while the last parts are written
    cfg.gridDim = dim3(pl.entries, std::min<long long>(8 * NT, (long long)P.max_new * (P.n_heads / P.c.n_kv)));
    cfg.blockDim = dim3(256);
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
