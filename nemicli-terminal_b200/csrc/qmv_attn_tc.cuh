// Attention of many query rows (prompts) over the quantised cache, on the 5th-generation tensor cores (layout:
// qmv_kv.cuh; parameters and shared pieces: qmv_attn.cuh).  bf16 and fp16 queries.
//
//   S = Q K^T,  P = 2^(S scale log2 e - ref),  O += P V,  l += sum P   per tile of BN keys, then O / l
//
// A CTA takes NQ tiles of 128 query rows of one sequence and key head (row = token * group + head of the group, so
// the cache is unpacked once for the whole group) over all their keys.  For two tiles, 64 keys and 128 values a step takes
// 1280 clocks of MMA (the scores 768: one of 64 keys from shared memory takes 48 clocks, not 32; the sums 512), 1024 of exp2 (16 a
// clock and SM) and 1280 of shared memory (128 bytes a clock: the scores' operands 768, V 256, the producers' stores 256), all side by
// side; measured about 2200 (8192 tokens, 32 heads: 0.58 to 0.62 ms, 880 to 900 TFLOP/s): no pipe is full, each role waits for another.
// Scores of 128 keys would take their 64 clocks an MMA and half the waits, with one buffer a query tile and the two tiles in turn.  Roles:
//   producers  NP x 4 warps: words of the cache -> d * code in fp16 (one rounding) -> shared memory, in the MMA's K-major core
//              matrices (8 rows x 16 bytes; K: rows = keys, V: rows = values of the head, so a V word, whose halves
//              are two tokens, lands transposed without a shuffle).  Loads one round ahead in registers, page numbers two.
//              Heads of 256 values have one query tile's time for twice the unpacking: two groups take the rounds in turn
//              (6 prompts of up to 1500 tokens on up to 6001, window 1024, 16 heads on 8: 287 -> 262 us), and V's stage is waited
//              for behind K's (-> 240; 236 to 244 now).
//   MMA        one warp: the scores run two steps ahead of the sums, the other tile's softmax runs meanwhile.
//   softmax    NQ x 4 warps, one thread a row: scores from tensor memory, P as fp16 over them, and the row's
//              reference, sum and mask in registers.  P is 2^9 where the reference was set and moves it only past 2^15 (then the
//              warp rescales its rows of O in tensor memory), so weights down to 2^-23 of the row's largest are normal numbers of
//              fp16 (set at 1 and moved past 2^8, the sum kept weights below 2^-14 that P lost).  Set at 2^11, 8192 tokens take 631
//              us, at 2^9 618, at 2^7 617; with 256 values and a window 258, 244 and 242.
// The exponentials are not the bound: a quarter of them as a cubic on the other units gained nothing (595 us without, 610 with it).
// Queries are fp16 after a power of two per row, which puts the largest at 2^14: bf16 values are exact down to 2^-31 of it, fp16's
// down to 2^-28, smaller ones are off by up to 2^-39 of it. Tensor memory: S NQ x 2 x BN columns, O NQ x D columns. Every mbarrier
// wait is bounded; on expiry the CTA sets DEV_TIMEOUT, waits (bounded) for its MMAs, frees its tensor memory and leaves.
#pragma once
#include <climits>

#include "qmv_attn.cuh"

namespace qmv {

template <int J> struct AttnTcShape {
    static constexpr int D = 32 * J;
    static constexpr int NQ = J == 8 ? 1 : 2;                     // tiles of 128 query rows
    static constexpr int BN = 64;                                 // keys a step
    static constexpr int PB = J == 8 ? 64 : 128;                  // keys the producers take at once: one or two steps' stages
    static constexpr int KS = 2 * PB / BN;                        // stages of K and of V
    static constexpr int NP = J == 8 ? 2 : 1;                    // groups of producers (two: each sees every phase of its stage)
    static constexpr int kThreads = (NQ + NP) * 128 + 32;
    static constexpr int kQ = 128 * D * 2, kK = BN * D * 2, kV = D * BN * 2;      // bytes of one tile / stage
    static constexpr int kScaleK = PB * J * 2, kScaleV = J * PB * 2;
    static constexpr int kOffK = NQ * kQ, kOffV = kOffK + KS * kK, kOffSK = kOffV + KS * kV, kOffSV = kOffSK + 2 * kScaleK;
    static constexpr int kOffBar = kOffSV + 4 * kScaleV;          // mbarriers, the tensor-memory address
    static constexpr int kOffBad = kOffBar + 256;                 // [4][4] words: keys whose page is not of the cache
    static constexpr int kOffBig = kOffBad + 64;                  // [4][4] words: bit 0 a large K scale among the warp's keys, bit 1 V
    static constexpr int kSmem = kOffBig + 64;
    static constexpr int kPart = (D + 2) * 128 * NQ;              // floats of a CTA's part: [D / 4][rows][4], references, weights
    static constexpr uint32_t kSboQ = D * 16, kSboK = D * 16, kSboV = BN * 16;    // bytes between 8-row groups
};

// shared-memory matrix descriptor, K-major without swizzle: 128 bytes along K, sbo per 8 rows, version 1
__device__ __forceinline__ uint64_t at_desc(uint32_t saddr, uint32_t sbo) {
    return uint64_t((saddr >> 4) & 0x3FFFu) | (uint64_t(128 >> 4) << 16) | (uint64_t((sbo >> 4) & 0x3FFFu) << 32) | (uint64_t(1) << 46);
}
// kind::f16, fp32 sums, fp16 A and B, both K-major, M = 128
__host__ __device__ constexpr uint32_t at_idesc(int n) { return (1u << 4) | (uint32_t(n >> 3) << 17) | (uint32_t(128 >> 4) << 24); }
__device__ __forceinline__ void at_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }"
                 :: "r"(d), "l"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void at_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
    asm volatile("{ .reg .pred p; setp.ne.b32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p; }"
                 :: "r"(d), "r"(a), "l"(b), "r"(idesc), "r"(acc) : "memory");
}
__device__ __forceinline__ void at_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" :: "r"(bar) : "memory");
}
__device__ __forceinline__ bool at_elect() {                      // true in one lane of the (whole) warp
    uint32_t e;
    asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(e));
    return e != 0;
}
// a word of two bf16 or fp16 as fp32, and back (rounded to nearest)
template <class T> __device__ __forceinline__ float2 raw_f2(uint32_t w);
template <> __device__ __forceinline__ float2 raw_f2<__nv_bfloat16>(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
template <> __device__ __forceinline__ float2 raw_f2<__half>(uint32_t w) { return unpack_h2(w); }
template <class T> __device__ __forceinline__ uint32_t pack_out(float x, float y);
template <> __device__ __forceinline__ uint32_t pack_out<__nv_bfloat16>(float x, float y) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(y), "f"(x));
    return r;
}
template <> __device__ __forceinline__ uint32_t pack_out<__half>(float x, float y) { return pack_held(x, y); }
__device__ __forceinline__ void at_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void at_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void at_fence_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// 32 fp32 columns of the warp's 32 lanes (thread = row); at_wait_ld before use
__device__ __forceinline__ void at_ld32(uint32_t a, uint32_t (&r)[32]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
                   "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
                   "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(a));
}
__device__ __forceinline__ void at_ld16(uint32_t a, uint32_t (&r)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
                   "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(a));
}
// two fp32 at a time, and the larger of three
__device__ __forceinline__ uint64_t pack_f2(float x, float y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ float2 unpack_f2(uint64_t v) {
    float2 r;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
    return r;
}
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ void at_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void at_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void at_st16(uint32_t a, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
                 :: "r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]) : "memory");
}
__device__ __forceinline__ void at_st32(uint32_t a, const uint32_t (&r)[32]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
                 "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
                 :: "r"(a), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
                    "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
                    "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
                    "r"(r[30]), "r"(r[31]) : "memory");
}
__device__ __forceinline__ void at_sts128(uint32_t a, uint32_t x, uint32_t y, uint32_t z, uint32_t w) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" :: "r"(a), "r"(x), "r"(y), "r"(z), "r"(w) : "memory");
}

// words of N bytes-aligned-as-they-come (see load sites) read once from global memory
template <int N>
__device__ __forceinline__ void at_ldg(uint32_t* w, const uint8_t* p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const uint4 x = __ldg(reinterpret_cast<const uint4*>(p + 4 * i));
            w[i] = x.x, w[i + 1] = x.y, w[i + 2] = x.z, w[i + 3] = x.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N; i += 2) {
            const uint2 x = __ldg(reinterpret_cast<const uint2*>(p + 4 * i));
            w[i] = x.x, w[i + 1] = x.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) w[i] = __ldg(reinterpret_cast<const uint32_t*>(p + 4 * i));
    }
}

// d * code stays within fp16: Q8_0's clamped values are 127 times fp16(65504 / 127) = 516, and 65532 rounds to an infinity, which a
// weight of 0 would turn into NaN for the queries that must not see it.  65504 is that value within its rounding, 2^-11.  Only
// rounds of keys with a larger scale than big_scale go over the eight values that a thread has stored at a (unpacking in two
// versions instead: 24.7 us for 517 tokens from a cold start against 22.7, the instructions' fetch)
__device__ __forceinline__ void at_clamp8(uint32_t a) {
    const __half2 most = __float2half2_rn(65504.f), least = __float2half2_rn(-65504.f);
    uint4 w = lds128(a);
    auto in = [&](uint32_t x) { return h2_bits(__hmax2_nan(__hmin2_nan(bits_h2(x), most), least)); };
    at_sts128(a, in(w.x), in(w.y), in(w.z), in(w.w));
}
__host__ __device__ constexpr uint32_t big_scale(int b) { return b == 4 ? 0x6FFFu : 0x5FFFu; }      // 8188, 511.75 (fp16 bits): 8 and 128 times that are 65504

// Eight K values of one word (two for Q8_0) times d: an OR of fp16's 1024 turns a code into 1024 + c (the upper nibbles
// into 1024 + 16 c), the subtraction is exact, and the product with d is the one rounding
template <int KB>
__device__ __forceinline__ void unpack_k8(const uint32_t* w, __half2 d, uint32_t (&o)[4]) {
    if constexpr (KB == 4) {
        const __half2 low = __float2half2_rn(-1032.f), high = __float2half2_rn(-72.f), sixteenth = __float2half2_rn(0.0625f);
        const uint32_t a = w[0], b = w[0] >> 8;
        o[0] = h2_bits(__hmul2(__hadd2(bits_h2((a & 0x000F000Fu) | 0x64006400u), low), d));
        o[1] = h2_bits(__hmul2(__hfma2(bits_h2((a & 0x00F000F0u) | 0x64006400u), sixteenth, high), d));
        o[2] = h2_bits(__hmul2(__hadd2(bits_h2((b & 0x000F000Fu) | 0x64006400u), low), d));
        o[3] = h2_bits(__hmul2(__hfma2(bits_h2((b & 0x00F000F0u) | 0x64006400u), sixteenth, high), d));
    } else {
        const __half2 low = __float2half2_rn(-1152.f);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            o[2 * i] = h2_bits(__hmul2(__hadd2(bits_h2((w[i] & 0x00FF00FFu) | 0x64006400u), low), d));
            o[2 * i + 1] = h2_bits(__hmul2(__hadd2(bits_h2(((w[i] >> 8) & 0x00FF00FFu) | 0x64006400u), low), d));
        }
    }
}
// value i (0..3) of a V word's (two for Q8_0) token pair, times the tokens' scales
template <int VB>
__device__ __forceinline__ uint32_t unpack_v(const uint32_t* w, int i, __half2 d) {
    if constexpr (VB == 4) {
        return h2_bits(__hmul2(__hadd2(bits_h2(((w[0] >> (4 * i)) & 0x000F000Fu) | 0x64006400u), __float2half2_rn(-1032.f)), d));
    } else {
        const uint32_t x = i & 2 ? w[1] : w[0];
        return h2_bits(__hmul2(__hadd2(bits_h2(((x >> (8 * (i & 1))) & 0x00FF00FFu) | 0x64006400u), __float2half2_rn(-1152.f)), d));
    }
}

template <int DT, int J, int KB, int VB>
__global__ void __launch_bounds__(AttnTcShape<J>::kThreads, 1) attn_tc_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    using Sh = AttnTcShape<J>;
    constexpr int D = Sh::D, NQ = Sh::NQ, BN = Sh::BN, KS = Sh::KS, NP = Sh::NP;
    extern __shared__ __align__(128) uint8_t tc_smem_[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = P.n_heads / P.c.n_kv;
    int x = blockIdx.x;
    const int sp = x % P.split;                                   // of the tile's keys
    x /= P.split;
    const int hk = x % P.c.n_kv;
    x /= P.c.n_kv;
    const int qt = P.row_tiles - 1 - x % P.row_tiles, b = x / P.row_tiles;        // the tiles with most keys first
    const AttnSeq S = attn_seq(P, b, tid == 0 && hk == 0 && qt == 0, BN);
    const int rows = min(S.n, P.max_new) * group, base = qt * 128 * NQ;
    if (base >= rows) return;
    const int pos0 = S.len - S.n, tok0 = base / group, tok1 = (min(base + 128 * NQ, rows) - 1) / group;
    const int last = min(pos0 + tok1, S.len - 1);
    const int first = P.window > 0 ? max(0, pos0 + tok0 - P.window + 1) : 0;
    int kt0 = first / BN, n_tiles = last < first ? 0 : last / BN - kt0 + 1;
    if (P.split > 1) {                                            // steps of this CTA
        const int per = (n_tiles + P.split - 1) / P.split;
        kt0 += sp * per, n_tiles = max(0, min(per, n_tiles - sp * per));
    }

    const uint32_t sm = smem_u32(tc_smem_);
    const uint32_t bar = sm + Sh::kOffBar;                        // stages: up to four each; S and P: two buffers a query tile
    const uint32_t k_full = bar, k_free = bar + 32, v_full = bar + 64, v_free = bar + 96, s_full = bar + 128, p_full = bar + 160,
                   o_full = bar + 192, q_full = bar + 224, done = bar + 232;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(tc_smem_ + Sh::kOffBar + 240);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tslot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 4 && lane == 0) {
        for (int i = 0; i < KS; ++i) {
            mbar_init(k_full + 8 * i, 4 * BN / Sh::PB), mbar_init(k_free + 8 * i, 1);
            mbar_init(v_full + 8 * i, 4 * BN / Sh::PB), mbar_init(v_free + 8 * i, 1);
        }
        for (int i = 0; i < 2 * NQ; ++i) mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, 4), mbar_init(o_full + 8 * i, 1);
        mbar_init(done, 1);
        mbar_init(q_full, 4 * NQ);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    at_before();
    __syncthreads();
    at_after();
    constexpr uint32_t tmem = 0;                                  // all 512 columns were asked for: they start at 0
    constexpr uint32_t kO = NQ * 2 * BN;                          // S (and P over it): column (2 a + buffer) BN; O: kO + a D
    const int qa = warp >> 2;                                     // query tile, from NQ on producers, NQ + NP: MMA
    bool ok = true;                                               // no wait ran out so far

    if (qa < NQ) {
        // ---- softmax: one thread a row ----------------------------------------------------------
        const int wr = 32 * (warp & 3), r0 = base + 128 * qa + wr;        // the warp's first row
        const int r = r0 + lane;
        float cs = 0.f;
        const int tok = r / group, head = hk * group + r - tok * group;
        {   // The warp's 32 rows of queries, 8 at a time, to fp16 after a power of two per row.  Read by four neighbouring lanes a
            // row (64 bytes side by side: two tiles in 6200 clocks, with eight rows in neighbouring lanes 7500; one load a piece where
            // rows start on 16 bytes: 5000),
            // stored by eight rows in neighbouring lanes (no two on a bank), exchanged in between.
            constexpr int kCores = D / 32;                        // 16-byte pieces a lane
            const bool wide = !((reinterpret_cast<uintptr_t>(P.q) | uintptr_t(P.q_stride) * sizeof(T)) & 15u);
            const int g = lane >> 2, c = lane & 3, from = 4 * (lane & 7) + (lane >> 3);
            constexpr int kPass = J == 8 ? 2 : 4;
            int mine = 0;                                         // exponent of row `lane`, found by lanes of pass lane / 8
#pragma unroll 1
            for (int q0 = 0; q0 < 4; q0 += kPass) {
                uint32_t h[kPass][kCores][4];
                int e[kPass];
#pragma unroll
                for (int q = 0; q < kPass; ++q) {
                    const int rr = r0 + 8 * (q0 + q) + g;
                    const bool live = rr < rows;
                    const int t = __shfl_sync(0xffffffffu, tok, 8 * (q0 + q) + g), hd = __shfl_sync(0xffffffffu, head, 8 * (q0 + q) + g);
                    const T* src = static_cast<const T*>(P.q) + (live ? (S.row0 + t) * P.q_stride + hd * D : 0);
#pragma unroll
                    for (int i = 0; i < kCores; ++i) {                // raw bits first: every load of the warp in flight
                        uint4 u = make_uint4(0u, 0u, 0u, 0u);
                        if (live && wide) {
                            u = __ldg(reinterpret_cast<const uint4*>(src + 8 * (4 * i + c)));
                        } else if (live) {
                            const uint2* at = reinterpret_cast<const uint2*>(src + 8 * (4 * i + c));
                            const uint2 a = __ldg(at), b2 = __ldg(at + 1);
                            u = make_uint4(a.x, a.y, b2.x, b2.y);
                        }
                        h[q][i][0] = u.x, h[q][i][1] = u.y, h[q][i][2] = u.z, h[q][i][3] = u.w;
                    }
                }
#pragma unroll
                for (int q = 0; q < kPass; ++q) {
                    float top = 0.f;
#pragma unroll
                    for (int i = 0; i < kCores; ++i)
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 x = raw_f2<T>(h[q][i][w]);
                            top = fmaxf(top, fmaxf(fabsf(x.x), fabsf(x.y)));
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const int ex = int((__float_as_uint(top) >> 23) & 255u);
                    e[q] = ex == 0 || ex == 255 ? 0 : max(-120, ex - 127 - 14);       // 2^14 <= top 2^-e < 2^15
                    const float down = __uint_as_float((uint32_t(127 - e[q]) << 23) | (P.scale < 0.f ? 0x80000000u : 0u));
                    const int rl = wr + 8 * (q0 + q) + (lane & 7);
                    const uint32_t dst = sm + qa * Sh::kQ + (rl >> 3) * Sh::kSboQ + (rl & 7) * 16;
#pragma unroll
                    for (int i = 0; i < kCores; ++i) {
                        uint32_t o[4];
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const float2 x = raw_f2<T>(h[q][i][w]);
                            o[w] = __shfl_sync(0xffffffffu, pack_h2(x.x * down, x.y * down), from);
                        }
                        at_sts128(dst + (4 * i + (lane >> 3)) * 128, o[0], o[1], o[2], o[3]);
                    }
                }
#pragma unroll
                for (int q = 0; q < kPass; ++q) {
                    const int x = __shfl_sync(0xffffffffu, e[q], 4 * (lane & 7));
                    if (lane >> 3 == q0 + q) mine = x;
                }
            }
            at_fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_full);
            // positive (the sign went into the queries), so that masked scores stay -inf where the scale is 0
            cs = fmaxf(fabsf(P.scale) * 1.4426950408889634f * __uint_as_float(uint32_t(127 + mine) << 23), 1e-30f);
        }
        const uint32_t quad = tmem + (uint32_t(wr) << 16), o_at = quad + kO + qa * D;
        const int pos = r < rows ? pos0 + tok : -1;
        float ref = kAttnNone, sum = 0.f;
        // keys that every row of this tile of 128 sees
        const int row_a = min(base + 128 * qa, rows - 1), row_b = min(base + 128 * qa + 127, rows - 1);
        const int full1 = pos0 + row_a / group, full0 = P.window > 0 ? pos0 + row_b / group - P.window + 1 : 0;
        const int low = P.window > 0 ? pos - P.window + 1 : 0;
        for (int i = 0; i < n_tiles; ++i) {
            const int buf = i & 1;
            const uint32_t s_at = quad + (2 * qa + buf) * BN;
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * (2 * qa + buf), uint32_t(i >> 1) & 1u));      // the lanes leave together
            if (!ok) break;
            at_after();
            uint32_t v[BN];                                       // the row's scores
#pragma unroll
            for (int c = 0; c < BN; c += 32) at_ld32(s_at + c, *reinterpret_cast<uint32_t(*)[32]>(v + c));
            const int key = (kt0 + i) * BN;
            // keys of pages outside the cache are masked too (the words stay for four rounds)
            uint32_t bad[2];
            asm volatile("ld.shared.v2.u32 {%0, %1}, [%2];" : "=r"(bad[0]), "=r"(bad[1])
                         : "r"(sm + Sh::kOffBad + (Sh::PB == BN ? 16 * (i & 3) : 16 * ((i >> 1) & 3) + 8 * (i & 1))) : "memory");
            const bool whole = key >= full0 && key + BN - 1 <= full1 && !(bad[0] | bad[1]);
            at_wait_ld();
            if (!whole) {                                         // what this row does not see becomes -inf
#pragma unroll
                for (int c = 0; c < BN; c += 32) {
                    const int lo = low - key - c, hi = pos - key - c;
                    const uint32_t from = lo <= 0 ? ~0u : lo > 31 ? 0u : ~0u << lo, to = hi >= 31 ? ~0u : hi < 0 ? 0u : (2u << hi) - 1u;
                    const uint32_t seen = from & to & ~bad[c / 32];
#pragma unroll
                    for (int k = 0; k < 32; ++k)
                        if (!(seen >> k & 1u)) v[c + k] = 0xFF800000u;
                }
            }
            float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int k = 0; k < BN; k += 2) tops[(k >> 1) & 3] = max3(tops[(k >> 1) & 3], __uint_as_float(v[k]), __uint_as_float(v[k + 1]));
            const float top = max3(fmaxf(tops[0], tops[1]), tops[2], tops[3]);
            const float m = top == -INFINITY ? kAttnNone : top * cs;
            const bool move = m > ref + 15.f;
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? ex2(ref - (m - 9.f)) : 1.f;
                if (move) ref = m - 9.f;
                sum *= f;
                if (i > 0) {
                    ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * (2 * qa + (buf ^ 1)), uint32_t((i - 1) >> 1) & 1u));       // O(i - 1) is complete
                    if (!ok) break;
                    at_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 16) {
                        uint32_t y[16];
                        at_ld16(o_at + c, y);
                        at_wait_ld();
#pragma unroll
                        for (int k = 0; k < 16; ++k) y[k] = __float_as_uint(__uint_as_float(y[k]) * f);
                        at_st16(o_at + c, y);
                    }
                }
            }
            uint64_t part[2] = {0ull, 0ull};                      // pairs of fp32 sums
            const uint64_t cs2 = pack_f2(cs, cs), ref2 = pack_f2(-ref, -ref);
#pragma unroll
            for (int c = 0; c < BN; c += 32) {                    // P over the scores
                uint32_t h[16];
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    const float2 x = unpack_f2(fma_f2(pack_f2(__uint_as_float(v[c + k]), __uint_as_float(v[c + k + 1])), cs2, ref2));
                    const float p0 = ex2(x.x), p1 = ex2(x.y);
                    part[(k >> 1) & 1] = add_f2(part[(k >> 1) & 1], pack_f2(p0, p1));
                    h[k >> 1] = pack_h2(p0, p1);
                }
                at_st16(s_at + c / 2, h);
            }
            {
                const float2 x = unpack_f2(add_f2(part[0], part[1]));
                sum += x.x + x.y;
            }
            at_wait_st();
            at_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * (2 * qa + buf));
        }
        if (ok && n_tiles) ok = __all_sync(0xffffffffu, mbar_wait(o_full + 8 * (2 * qa + ((n_tiles - 1) & 1)), uint32_t((n_tiles - 1) >> 1) & 1u));
        at_after();
        // O / sum as the output's type to this warp's part of the query tile (nothing reads it any more), 16-byte pieces in
        // an order that keeps lanes on different banks, and from there whole rows at a time
        const float inv = sum > 0.f ? __fdividef(1.f, sum) : sum == sum ? 0.f : sum;
        const uint32_t stage = sm + qa * Sh::kQ + wr * D * 2;
        if (ok && P.split > 1) {                                  // sums, reference and weight for attn_tc_join_kernel
            float* part = P.parts + (long long)blockIdx.x * Sh::kPart + 128 * qa + wr + lane;
#pragma unroll 1
            for (int c = 0; c < D; c += 16) {
                uint32_t y[16] = {};
                if (n_tiles) {
                    at_ld16(o_at + c, y);
                    at_wait_ld();
                }
                float4* to = reinterpret_cast<float4*>(P.parts + (long long)blockIdx.x * Sh::kPart) + c / 4 * (128 * NQ) + 128 * qa + wr + lane;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (r < rows) to[k * 128 * NQ] = make_float4(__uint_as_float(y[4 * k]), __uint_as_float(y[4 * k + 1]), __uint_as_float(y[4 * k + 2]), __uint_as_float(y[4 * k + 3]));
            }
            part[D * 128 * NQ] = ref, part[(D + 1) * 128 * NQ] = sum;
        } else if (ok) {
#pragma unroll
            for (int c = 0; c < D; c += 32) {
                uint32_t y[32];
                if (n_tiles) {
                    at_ld32(o_at + c, y);
                    at_wait_ld();
                }
#pragma unroll
                for (int k = 0; k < 32; k += 8) {
                    uint32_t o[4];
#pragma unroll
                    for (int w = 0; w < 4; ++w)
                        o[w] = inv != 0.f ? pack_out<T>(__uint_as_float(y[k + 2 * w]) * inv, __uint_as_float(y[k + 2 * w + 1]) * inv) : 0u;
                    const int piece = (c + k) / 8;
                    at_sts128(stage + lane * D * 2 + (D % 64 ? piece : (piece & ~7) | ((piece ^ lane) & 7)) * 16, o[0], o[1], o[2], o[3]);
                }
            }
            __syncwarp();
            constexpr int kPieces = D / 8;                        // of a row
            for (int i = lane; i < 32 * kPieces; i += 32) {
                const int row = i / kPieces, piece = i - row * kPieces;
                const int t = __shfl_sync(0xffffffffu, tok, row), hd = __shfl_sync(0xffffffffu, head, row);
                if (r0 + row >= rows) continue;
                const uint4 y = lds128(stage + row * D * 2 + (D % 64 ? piece : (piece & ~7) | ((piece ^ row) & 7)) * 16);
                T* out = static_cast<T*>(P.out) + ((long long)(S.row0 + t) * P.n_heads + hd) * D;
                reinterpret_cast<uint4*>(out)[piece] = y;
            }
        }
    } else if (qa < NQ + NP) {
        // ---- producers -----------------------------------------------------------------------------
        const int pw = warp & 3, pt = tid & 127, pg = qa - NQ;    // producer warp, thread and group: rounds pg, pg + NP, ..
        constexpr int PB = Sh::PB, kPer = PB / BN;                // keys and stages a round
        constexpr int kRows = PB / 4, kGroups = kRows / 8;        // keys a warp, 8-key groups
        constexpr int kWk = J * KB / 4;                           // words of a lane's K run
        constexpr int JV = PB == 128 ? J : J / 2, kWv = JV * VB / 4;      // V blocks of a lane, words of a pair's run
        uint32_t kw[kGroups][kWk], vw[4][kWv], sw[J], bad = 0;
        const int kk = lane & 7, kt = lane >> 3;                  // K: key within 8, run
        const int vg = lane & 7, vkc = PB == 128 ? lane >> 3 : (lane >> 3) & 1, vj = PB == 128 ? 0 : (lane >> 4) * JV;
        const int* table = P.tables + (long long)b * P.width;
        // The table entries of a tile's 16-key runs that this lane reads: asked for two tiles ahead and first looked at one
        // tile later, so that no load waits for one.  kNoKey: nothing to see there.
        constexpr int kNoKey = INT_MIN;
        auto entry_of = [&](int key) { return key > last || key + 15 < first ? kNoKey : __ldg(table + (key >> P.c.page_shift)); };
        auto valid = [&](int p) { return uint32_t(p) < uint32_t(P.c.n_pages); };
        // this lane's bytes of page 0, and the pages' strides (below 2^31 bytes: a page has at most 2^30 values)
        const uint8_t* const k0 = P.c.k + P.c.k_row(0, hk, kk) + kt * J * KB;
        const uint8_t* const v0 = P.c.v + P.c.v_pair(0, hk, 0) + (vg * J + vj) * VB;
        const uint8_t* const s0 = reinterpret_cast<const uint8_t*>(P.c.sc + P.c.scale_row(0, hk, 0));
        const uint32_t in_page = P.c.page() - 1, rows_page = uint32_t(P.c.n_kv) << P.c.page_shift;
        const uint32_t k_page = rows_page * (4 * J * KB), v_page = rows_page * (4 * J * VB), s_page = rows_page * (4 * J);
        constexpr int kRuns = (kRows + 15) / 16;
        int pk[kRuns], pv, ps;                                    // of K's runs, V's keys, the scale's key
        auto ask = [&](int i) {
            const int key = kt0 * BN + i * PB;
#pragma unroll
            for (int q = 0; q < kRuns; ++q) pk[q] = entry_of(key + kRows * pw + 16 * q);
            pv = entry_of((key + kRows * pw + 8 * vkc) & ~15);
            const int k = key + pt;
            ps = pt < PB && k >= first && k <= last ? entry_of(k & ~15) : kNoKey;
        };
        auto load_k = [&](int i) {
            const int key0 = kt0 * BN + i * PB;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int key = key0 + kRows * pw + 8 * q, page = pk[q >> 1];
                if (valid(page)) {
                    at_ldg<kWk>(kw[q], k0 + ((unsigned long long)page * k_page + (key & in_page) * (4 * J * KB)));
                } else {
#pragma unroll
                    for (int w = 0; w < kWk; ++w) kw[q][w] = 0u;
                }
            }
            // scales of key pt; nobody sees it: 0 (it may hold anything)
            bad = __ballot_sync(0xffffffffu, ps != kNoKey && !valid(ps));
            if (valid(ps)) {
                at_ldg<J>(sw, s0 + ((unsigned long long)ps * s_page + ((key0 + pt) & in_page) * (4 * J)));
            } else {
#pragma unroll
                for (int w = 0; w < J; ++w) sw[w] = 0u;
            }
        };
        auto load_v = [&](int i) {
            const int key = kt0 * BN + i * PB + kRows * pw + 8 * vkc;
            if (valid(pv)) {
                const uint8_t* at = v0 + ((unsigned long long)pv * v_page + (key & in_page) * (4 * J * VB));
#pragma unroll
                for (int p = 0; p < 4; ++p) at_ldg<kWv>(vw[p], at + p * (8 * J * VB));
            } else {
#pragma unroll
                for (int p = 0; p < 4; ++p)
#pragma unroll
                    for (int w = 0; w < kWv; ++w) vw[p][w] = 0u;
            }
        };
        if (n_tiles) {
            ask(pg);
            load_k(pg), load_v(pg);
            ask(pg + NP);
        }
        const int rounds = (n_tiles + kPer - 1) / kPer;
        for (int i = pg; i < rounds; i += NP) {
            const int st = i & 1;                                 // stages kPer st ..
            const uint32_t par = uint32_t(i >> 1) & 1u;
            const uint32_t s_k = sm + Sh::kOffSK + st * Sh::kScaleK, s_v = sm + Sh::kOffSV + (i & 3) * Sh::kScaleV;
            if (i >= 2)
#pragma unroll
                for (int q = 0; q < kPer; ++q)
                    ok = ok && mbar_wait(k_free + 8 * (kPer * st + q), par ^ 1u);
            // scales: K's by key, V's by block (so that eight keys of a block are one word of 16 bytes); four buffers of V's,
            // since a warp may be here while another still reads the ones of this group's last round
            if (pt < PB) {
                __half* dk = reinterpret_cast<__half*>(tc_smem_ + Sh::kOffSK + st * Sh::kScaleK) + pt * J;
                __half* dv = reinterpret_cast<__half*>(tc_smem_ + Sh::kOffSV + (i & 3) * Sh::kScaleV) + pt;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const uint32_t a = sw[j >> 1], c = sw[(J + j) >> 1];
                    dk[j] = __ushort_as_half((unsigned short)(j & 1 ? a >> 16 : a & 0xFFFFu));
                    dv[j * PB] = __ushort_as_half((unsigned short)((J + j) & 1 ? c >> 16 : c & 0xFFFFu));
                }
            }
            uint32_t most[2] = {0u, 0u};                          // |scales| of K and of V, two fp16 each
#pragma unroll
            for (int w = 0; w < J; ++w) {
                const uint32_t of_k = (2 * w < J ? 0x7FFFu : 0u) | (2 * w + 1 < J ? 0x7FFF0000u : 0u);
                if (of_k) most[0] = __vmaxu2(most[0], sw[w] & of_k);
                if (of_k != 0x7FFF7FFFu) most[1] = __vmaxu2(most[1], sw[w] & (of_k ^ 0x7FFF7FFFu));
            }
            const uint32_t big_k = max(most[0] >> 16, most[0] & 0xFFFFu) > big_scale(KB) ? 1u : 0u,
                           big_v = max(most[1] >> 16, most[1] & 0xFFFFu) > big_scale(VB) ? 2u : 0u;
            const uint32_t big = __reduce_or_sync(0xffffffffu, big_k | big_v);
            uint32_t all;                                         // the four warps go on, or leave, together
            if (lane == 0) {
                reinterpret_cast<uint32_t*>(tc_smem_ + Sh::kOffBad)[4 * (i & 3) + pw] = bad;
                reinterpret_cast<uint32_t*>(tc_smem_ + Sh::kOffBig)[4 * (i & 3) + pw] = big;
            }
            if (bad && lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
            asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %1, 0; barrier.cta.red.and.pred q, %2, 128, p; selp.u32 %0, 1, 0, q; }"
                         : "=r"(all) : "r"(uint32_t(ok)), "r"(1 + pg) : "memory");
            ok = all != 0;
            if (!ok) break;
            const uint4 bigs = lds128(sm + Sh::kOffBig + 16 * (i & 3));
            const uint32_t any_big = bigs.x | bigs.y | bigs.z | bigs.w;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int key = kRows * pw + 8 * q + kk;
                const uint32_t dst = sm + Sh::kOffK + kPer * st * Sh::kK + (key >> 3) * Sh::kSboK + (key & 7) * 16;     // stages side by side
                uint32_t d2[(J + 1) / 2];
                if constexpr (J == 3) {                           // three halves: at an odd key not on a word
                    d2[0] = lds16u(s_k + key * 6) | (lds16u(s_k + key * 6 + 2) << 16), d2[1] = lds16u(s_k + key * 6 + 4);
                } else {
#pragma unroll
                    for (int w = 0; w < J / 2; ++w) d2[w] = lds32(s_k + key * 2 * J + 4 * w);
                }
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    uint32_t o[4];
                    const __half2 d = bits_h2(d2[j >> 1]);
                    unpack_k8<KB>(&kw[q][j * KB / 4], j & 1 ? __high2half2(d) : __low2half2(d), o);
                    at_sts128(dst + (4 * j + kt) * 128, o[0], o[1], o[2], o[3]);
                }
            }
            if (any_big & 1u) {
                const int key = kRows * pw + kk;
                const uint32_t dst = sm + Sh::kOffK + kPer * st * Sh::kK + (key >> 3) * Sh::kSboK + (key & 7) * 16 + kt * 128;
#pragma unroll 1
                for (int x = 0; x < kGroups * J; ++x) at_clamp8(dst + x / J * Sh::kSboK + x % J * 512);
            }
            at_fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full + 8 * (kPer * st + kRows * pw / BN));
            if (i + NP < rounds) load_k(i + NP);
            // V's stage is free one step later than K's: waited for here, the scores of this round are not held up by it
            if (i >= 2) {
#pragma unroll
                for (int q = 0; q < kPer; ++q) ok = ok && mbar_wait(v_free + 8 * (kPer * st + q), par ^ 1u);
                ok = __all_sync(0xffffffffu, ok);
            }
            if (ok) {                                             // (if not: all leave at the next round's barrier)
                const int kc = (kRows / 8) * pw + vkc;            // 8-key core of the round
                const uint32_t dst = sm + Sh::kOffV + (kPer * st + kc / (BN / 8)) * Sh::kV + (kc % (BN / 8)) * 128;
#pragma unroll
                for (int j = 0; j < JV; ++j) {
                    uint32_t d[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                                 : "r"(s_v + ((vj + j) * PB + 8 * kc) * 2));
#pragma unroll
                    for (int s = 0; s < 4; ++s) {                 // the value differs by lane: no two of eight lanes share a bank
                        const int e = (s + (vg >> 1)) & 3, n = 32 * (vj + j) + 4 * vg + e;
                        uint32_t o[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) o[p] = unpack_v<VB>(&vw[p][j * VB / 4], e, bits_h2(d[p]));
                        at_sts128(dst + (n >> 3) * Sh::kSboV + (n & 7) * 16, o[0], o[1], o[2], o[3]);
                    }
                }
                if (any_big & 2u) {
#pragma unroll 1
                    for (int x = 0; x < 4 * JV; ++x) {
                        const int n = 32 * (vj + x / 4) + 4 * vg + x % 4;
                        at_clamp8(dst + (n >> 3) * Sh::kSboV + (n & 7) * 16);
                    }
                }
            }
            at_fence_smem();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(v_full + 8 * (kPer * st + kRows * pw / BN));
            if (i + NP < rounds) load_v(i + NP);
            ask(i + 2 * NP);
        }
    } else {
        // ---- MMA -----------------------------------------------------------------------------------
        // The whole warp walks the loop and one elected lane issues: descriptors and addresses stay in uniform registers
        // (issued by `if (lane == 0)` with the tensor-memory address read back, an MMA cost 116 clocks instead of 64).
        // Scores run two steps ahead of the sums, so a tile's softmax finds the next scores ready.
        constexpr uint32_t id_s = at_idesc(BN), id_o = at_idesc(D);
        auto wait = [&](uint32_t b, int phase) {
            ok = ok && __all_sync(0xffffffffu, mbar_wait(b, uint32_t(phase) & 1u));
            at_after();
            return ok;
        };
        auto scores = [&](int a, int i) {
            if (at_elect()) {
                const uint32_t q = sm + a * Sh::kQ, k = sm + Sh::kOffK + (i % KS) * Sh::kK, d = (2 * a + (i & 1)) * BN;
#pragma unroll
                for (int s = 0; s < D / 16; ++s) at_mma_ss(d, at_desc(q + 256 * s, Sh::kSboQ), at_desc(k + 256 * s, Sh::kSboK), id_s, s > 0);
                at_commit(s_full + 8 * (2 * a + (i & 1)));
                if (a == NQ - 1) at_commit(k_free + 8 * (i % KS));
            }
            __syncwarp();
        };
        if (n_tiles) wait(q_full, 0);
        for (int i = 0; i < min(2, n_tiles) && ok; ++i)
            if (wait(k_full + 8 * i, 0))
#pragma unroll
                for (int a = 0; a < NQ; ++a) scores(a, i);
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int st = i % KS;
            const uint32_t v = sm + Sh::kOffV + st * Sh::kV;
#pragma unroll
            for (int a = 0; a < NQ; ++a) {
                if (a == 0 && !wait(v_full + 8 * st, i / KS)) break;
                if (!wait(p_full + 8 * (2 * a + (i & 1)), i >> 1)) break;
                if (at_elect()) {
#pragma unroll
                    for (int s = 0; s < BN / 16; ++s)
                        at_mma_ts(kO + a * D, (2 * a + (i & 1)) * BN + 8 * s, at_desc(v + 256 * s, Sh::kSboV), id_o, i > 0 || s > 0);
                    at_commit(o_full + 8 * (2 * a + (i & 1)));
                    if (a == NQ - 1) at_commit(v_free + 8 * st);
                }
                __syncwarp();
                if (i + 2 < n_tiles) {
                    if (a == 0 && !wait(k_full + 8 * ((i + 2) % KS), (i + 2) / KS)) break;
                    scores(a, i + 2);
                }
            }
        }
        if (n_tiles) {                                            // everything issued is done before the memory is given back
            if (at_elect()) at_commit(done);
            __syncwarp();
            ok = __all_sync(0xffffffffu, mbar_wait(done, 0)) && ok;
        }
    }
    if (!ok && lane == 0 && P.status) atomicOr(P.status, DEV_TIMEOUT);
    __syncwarp();
    at_before();
    __syncthreads();
    at_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
}

// Joins the parts of tiles whose keys were cut: block (32 rows and 32 of their values, key head, sequence), a lane a row, a warp four
// values.
template <int DT, int J>
__global__ void __launch_bounds__(256) attn_tc_join_kernel(const __grid_constant__ AttnParams P) {
    using T = typename Elem<DT>::type;
    using Sh = AttnTcShape<J>;
    constexpr int R = 128 * Sh::NQ, D = Sh::D;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int b = blockIdx.z, hk = blockIdx.y, group = P.n_heads / P.c.n_kv, lane = threadIdx.x & 31;
    const int c = blockIdx.x % J * 8 + (threadIdx.x >> 5);        // values 4 c ..
    const AttnSeq S = attn_seq(P, b, false, Sh::BN);
    const int rows = min(S.n, P.max_new) * group, r = 32 * int(blockIdx.x / J) + lane, qt = r / R, at = r % R;
    if (r >= rows) return;
    const float* part = P.parts + ((long long)(b * P.row_tiles + P.row_tiles - 1 - qt) * P.c.n_kv + hk) * P.split * Sh::kPart;
    float ref = kAttnNone, sum = 0.f;
#pragma unroll 8
    for (int k = 0; k < P.split; ++k) ref = fmaxf(ref, part[(long long)k * Sh::kPart + D * R + at]);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int k = 0; k < P.split; ++k) {
        const float* p = part + (long long)k * Sh::kPart;
        const float w = ex2(p[D * R + at] - ref);
        const float4 y = reinterpret_cast<const float4*>(p)[c * R + at];
        sum = fmaf(w, p[(D + 1) * R + at], sum);
        o = make_float4(fmaf(w, y.x, o.x), fmaf(w, y.y, o.y), fmaf(w, y.z, o.z), fmaf(w, y.w, o.w));
    }
    const float inv = sum > 0.f ? __fdividef(1.f, sum) : sum == sum ? 0.f : sum;
    T* out = static_cast<T*>(P.out) + ((long long)(S.row0 + r / group) * P.n_heads + hk * group + r % group) * D + 4 * c;
    store4_held(out, inv != 0.f ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
}

// ---- host -------------------------------------------------------------------------------------------

// Whether a call takes the tiles (else attn_kernel), and how.  A tile walks its keys at a cost that its rows do not change, one
// CTA an SM: 14.7 ns a key for heads of 64 values, 17.9 for 128, 20.4 for 256.  attn_kernel spreads any work over the GPU, at
// a cost that goes with the rows: 2.6, 3.5 and 11.4 ps a key and row (both measured on 128 tokens and 32768 keys).  So the tiles gain from as many rows a round of CTAs as
// the ratio of the two.  Where the tiles fill at most half the SMs and there are keys enough to pay for a second launch
// (512 a part: 9 us of work, the launch 4 to 5), each one's keys are cut into as many parts as fill the GPU, and
// attn_tc_join_kernel adds them.  Measured in us, cut / uncut / attn_kernel, heads of 128 values, 8 key heads, 4 query heads each:
//   1 sequence of 32768 keys, 16 new tokens: 53 / 585 / 75      64 tokens: 56 / 586 / 248
//   8 sequences of 4096 keys, 16 tokens: 51 / 82 / 81           64 tokens: 57 / 83 / 267
//   1 sequence of 4096 keys, 16 tokens: 21 / 81 / 26 (the last is taken)    64 tokens: 25 / 82 / 50
//   32 sequences of 1024 keys, 24 tokens: - / 55 / 136
// and 64 heads on 4 of 256 values, 8 sequences of 4096 keys, 4 tokens: 37 / 90 / 119
struct AttnTcPlan {
    bool used;
    int row_tiles, split;
    long long grid, bytes;                                        // workspace: the parts
};
inline AttnTcPlan attn_tc_plan(const KvView& c, int dtype, int n_heads, int n_seq, int max_new, int width, int window) {
    AttnTcPlan p{};
    if (dtype == QMV_OUT_F32) return p;                           // fp16 products lack its accuracy
    const int per = c.J == 8 ? 128 : 256;
    const long long rows = (long long)max_new * (n_heads / c.n_kv), heads = (long long)n_seq * c.n_kv, tiles = (rows + per - 1) / per;
    long long keys = (long long)width << c.page_shift;
    if (window > 0) keys = std::min<long long>(keys, (long long)window + max_new);
    p.split = int(std::max<long long>(1, std::min<long long>(sm_count() / std::min<long long>(heads * tiles, sm_count()), keys / 512)));
    const long long rounds = (heads * tiles + sm_count() - 1) / sm_count();
    p.used = heads * rows >= rounds * (c.J == 2 ? 6400 : c.J == 8 ? 1700 : 5400) / p.split;
    p.grid = heads * tiles * p.split;
    if (tiles > INT_MAX) p.grid = LLONG_MAX;                      // refused
    p.row_tiles = int(std::min<long long>(tiles, INT_MAX));
    p.bytes = p.split > 1 ? p.grid * (c.dim + 2) * per * 4 : 0;
    return p;
}

template <int DT, int J, int KB, int VB>
int attn_tc_go(const AttnParams& P, cudaStream_t st) {
    using Sh = AttnTcShape<J>;
    static SmemGrant grant;
    if (const int e = grant(attn_tc_kernel<DT, J, KB, VB>, Sh::kSmem)) return e;
    const int rc = launch_pdl_smem(attn_tc_kernel<DT, J, KB, VB>, dim3(P.row_tiles * P.c.n_kv * P.n_seq * P.split), dim3(Sh::kThreads), Sh::kSmem, st, P);
    if (rc || P.split == 1) return rc;
    cudaLaunchConfig_t cfg = {};                                  // may start while the last parts are written
    cfg.gridDim = dim3(P.row_tiles * Sh::NQ * 4 * J, P.c.n_kv, P.n_seq);
    cfg.blockDim = dim3(256);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, attn_tc_join_kernel<DT, J>, P);
    return launched();
}

template <int J>
int attn_tc_dispatch(const AttnParams& P, int dtype, cudaStream_t st) {
    auto pick = [&](auto dt) {
        constexpr int DT = decltype(dt)::value;
        if (P.c.kb == 4) return P.c.vb == 4 ? attn_tc_go<DT, J, 4, 4>(P, st) : attn_tc_go<DT, J, 4, 8>(P, st);
        return P.c.vb == 4 ? attn_tc_go<DT, J, 8, 4>(P, st) : attn_tc_go<DT, J, 8, 8>(P, st);
    };
    if (dtype == QMV_OUT_BF16) return pick(std::integral_constant<int, QMV_OUT_BF16>{});
    return pick(std::integral_constant<int, QMV_OUT_F16>{});
}
extern template int attn_tc_dispatch<2>(const AttnParams&, int, cudaStream_t);
extern template int attn_tc_dispatch<3>(const AttnParams&, int, cudaStream_t);
extern template int attn_tc_dispatch<4>(const AttnParams&, int, cudaStream_t);
extern template int attn_tc_dispatch<8>(const AttnParams&, int, cudaStream_t);

}  // namespace qmv
