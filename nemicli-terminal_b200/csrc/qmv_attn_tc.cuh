// Attention of many query rows (prompts) over the quantised cache, on the 5th-generation tensor cores (layout:
// qmv_kv.cuh; parameters and shared pieces: qmv_attn.cuh).  bf16 and fp16 queries.
//
//   S = Q K^T,  P = 2^(S scale log2 e - ref),  O += P V,  l += sum P   per tile of BN keys, then O / l
//
// A CTA takes NQ tiles of 128 query rows of one sequence and key head (row = token * group + head of the group, so
// the cache is unpacked once for the whole group) over all their keys.  Bound by the tensor cores and the special
// function units about equally: 128 x 128 scores of 128 values take 1024 clocks of MMA (both products) and
// 1024 of exp2.  Roles:
//   producers  4 warps: words of the cache -> d * code in fp16 (one rounding) -> shared memory, in the MMA's K-major core
//              matrices (8 rows x 16 bytes; K: rows = keys, V: rows = values of the head, so a V word, whose halves
//              are two tokens, lands transposed without a shuffle).  Two stages each, loads one tile ahead in registers.
//   MMA        one thread: S(i + 1) of a tile follows its O(i), the other tile's softmax runs meanwhile.
//   softmax    NQ x 4 warps, one thread a row: scores from tensor memory, P as fp16 over them, and the row's
//              reference, sum and mask in registers.  The reference moves only when the row's maximum passes it by 2^8;
//              then the warp rescales its rows of O in tensor memory.
// Queries are fp16 after a power of two per row (exact but for values 2^-32 below the row's largest).  Tensor memory:
// S NQ x BN columns, O NQ x D columns.  Every mbarrier wait is bounded; on expiry the CTA sets DEV_TIMEOUT, waits
// (bounded) for its MMAs, frees its tensor memory and leaves.
#pragma once
#include "qmv_attn.cuh"

namespace qmv {

template <int J> struct AttnTcShape {
    static constexpr int D = 32 * J;
    static constexpr int NQ = J == 8 ? 1 : 2;                     // tiles of 128 query rows
    static constexpr int BN = J == 8 ? 64 : 128;                  // keys a step
    static constexpr int kThreads = NQ * 128 + 128 + 32;
    static constexpr int kQ = 128 * D * 2, kK = BN * D * 2, kV = D * BN * 2;      // bytes of one tile / stage
    static constexpr int kScaleK = BN * J * 2, kScaleV = J * BN * 2;
    static constexpr int kOffK = NQ * kQ, kOffV = kOffK + 2 * kK, kOffSK = kOffV + 2 * kV, kOffSV = kOffSK + 2 * kScaleK;
    static constexpr int kOffBar = kOffSV + 2 * kScaleV;
    static constexpr int kOffBad = kOffBar + 160;                 // [2][4] words: keys whose page is not of the cache
    static constexpr int kSmem = kOffBar + 256;
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
__device__ __forceinline__ uint32_t h2_bits(__half2 h) { return *reinterpret_cast<uint32_t*>(&h); }
__device__ __forceinline__ __half2 bits_h2(uint32_t w) { return *reinterpret_cast<__half2*>(&w); }

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
    constexpr int D = Sh::D, NQ = Sh::NQ, BN = Sh::BN;
    extern __shared__ __align__(128) uint8_t tc_smem_[];
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = P.n_heads / P.c.n_kv;
    int x = blockIdx.x;
    const int hk = x % P.c.n_kv;
    x /= P.c.n_kv;
    const int qt = P.row_tiles - 1 - x % P.row_tiles, b = x / P.row_tiles;        // the tiles with most keys first
    const AttnSeq S = attn_seq(P, b, tid == 0 && hk == 0 && qt == 0);
    const int rows = min(S.n, P.max_new) * group, base = qt * 128 * NQ;
    if (base >= rows) return;
    const int pos0 = S.len - S.n, tok0 = base / group, tok1 = (min(base + 128 * NQ, rows) - 1) / group;
    const int last = min(pos0 + tok1, S.len - 1);
    const int first = P.window > 0 ? max(0, pos0 + tok0 - P.window + 1) : 0;
    const int kt0 = first / BN, n_tiles = last < first ? 0 : last / BN - kt0 + 1;

    const uint32_t sm = smem_u32(tc_smem_);
    const uint32_t bar = sm + Sh::kOffBar;
    const uint32_t k_full = bar, k_free = bar + 16, v_full = bar + 32, v_free = bar + 48, s_full = bar + 64, p_full = bar + 80, o_full = bar + 96;
    uint32_t* tslot = reinterpret_cast<uint32_t*>(tc_smem_ + Sh::kOffBar + 128);
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" :: "r"(smem_u32(tslot)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(k_full + 8 * i, 4), mbar_init(k_free + 8 * i, 1);
            mbar_init(v_full + 8 * i, 4), mbar_init(v_free + 8 * i, 1);
            mbar_init(s_full + 8 * i, 1), mbar_init(p_full + 8 * i, 4);
        }
        mbar_init(o_full, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }

    // the softmax threads' rows: query values to shared memory
    const int qa = warp >> 2;                                     // which query tile (NQ and above: another role)
    const int r = base + 128 * qa + 32 * (warp & 3) + lane;
    float cs = 0.f;
    int pos = -1;
    if (qa < NQ) {
        const bool live = r < rows;
        const int tok = r / group;
        if (live) pos = pos0 + tok;
        const T* src = static_cast<const T*>(P.q) + (live ? (S.row0 + tok) * P.q_stride + (hk * group + r % group) * D : 0);
        float top = 0.f;
        for (int i = 0; i < D; i += 4) {
            const float4 v = live ? load4(src + i) : make_float4(0.f, 0.f, 0.f, 0.f);
            top = fmaxf(top, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
        }
        const int ex = int((__float_as_uint(top) >> 23) & 255u);
        const int e = ex == 0 || ex == 255 ? 0 : max(-110, min(110, ex - 127 - 8));     // 2^8 <= top 2^-e < 2^9
        const float down = __uint_as_float(uint32_t(127 - e) << 23);
        const float sgn = P.scale < 0.f ? -down : down;           // cs is not negative: the largest score is the largest product
        cs = fabsf(P.scale) * 1.4426950408889634f * __uint_as_float(uint32_t(127 + e) << 23);
        const int rl = 32 * (warp & 3) + lane;
        const uint32_t dst = sm + qa * Sh::kQ + (rl >> 3) * Sh::kSboQ + (rl & 7) * 16;
        for (int i = 0; i < D; i += 8) {
            const float4 u = live ? load4(src + i) : make_float4(0.f, 0.f, 0.f, 0.f), v = live ? load4(src + i + 4) : make_float4(0.f, 0.f, 0.f, 0.f);
            at_sts128(dst + (i >> 3) * 128, pack_h2(u.x * sgn, u.y * sgn), pack_h2(u.z * sgn, u.w * sgn), pack_h2(v.x * sgn, v.y * sgn),
                      pack_h2(v.z * sgn, v.w * sgn));
        }
        at_fence_smem();
    }
    at_before();
    __syncthreads();
    at_after();
    const uint32_t tmem = *tslot;
    bool ok = true;                                               // no wait ran out so far

    if (qa < NQ) {
        // ---- softmax: one thread a row ----------------------------------------------------------
        const uint32_t quad = tmem + (uint32_t(32 * (warp & 3)) << 16);
        const uint32_t s_at = quad + qa * BN, o_at = quad + NQ * BN + qa * D;
        float ref = kAttnNone, sum = 0.f;
        // keys that every row of this tile of 128 sees
        const int row_a = min(base + 128 * qa, rows - 1), row_b = min(base + 128 * qa + 127, rows - 1);
        const int full1 = pos0 + row_a / group, full0 = P.window > 0 ? pos0 + row_b / group - P.window + 1 : 0;
        const int low = P.window > 0 ? pos - P.window + 1 : 0;
        for (int i = 0; i < n_tiles && ok; ++i) {
            ok = __all_sync(0xffffffffu, mbar_wait(s_full + 8 * qa, i & 1));      // the warp's lanes leave together
            if (!ok) break;
            at_after();
            const int key = (kt0 + i) * BN;
            // keys of pages outside the cache are masked too (the words live as long as the tile's V stage)
            uint32_t bad[4];
            asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(bad[0]), "=r"(bad[1]), "=r"(bad[2]), "=r"(bad[3])
                         : "r"(sm + Sh::kOffBad + 16 * (i & 1)) : "memory");
            const bool whole = key >= full0 && key + BN - 1 <= full1 && !(bad[0] | bad[1] | bad[2] | bad[3]);
            float top = -INFINITY;
#pragma unroll
            for (int c = 0; c < BN; c += 32) {
                uint32_t v[32];
                at_ld32(s_at + c, v);
                at_wait_ld();
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 32; ++k) top = fmaxf(top, __uint_as_float(v[k]));
                } else {
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const int at = key + c + k;
                        top = fmaxf(top, at <= pos && at >= low && !(bad[c / 32] >> k & 1u) ? __uint_as_float(v[k]) : -INFINITY);
                    }
                }
            }
            const float m = top == -INFINITY ? kAttnNone : top * cs;
            const bool move = m > ref + 8.f;
            if (__any_sync(0xffffffffu, move)) {
                const float f = move ? ex2(ref - m) : 1.f;
                if (move) ref = m;
                sum *= f;
                if (i > 0) {                                      // O(i - 1) is complete: S(i) was issued after it
#pragma unroll
                    for (int c = 0; c < D; c += 32) {
                        uint32_t v[32];
                        at_ld32(o_at + c, v);
                        at_wait_ld();
#pragma unroll
                        for (int k = 0; k < 32; ++k) v[k] = __float_as_uint(__uint_as_float(v[k]) * f);
                        at_st32(o_at + c, v);
                    }
                }
            }
            float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < BN; c += 32) {                    // P over the scores already read
                uint32_t v[32], h[16];
                at_ld32(s_at + c, v);
                at_wait_ld();
#pragma unroll
                for (int k = 0; k < 32; k += 2) {
                    float p0 = ex2(fmaf(__uint_as_float(v[k]), cs, -ref)), p1 = ex2(fmaf(__uint_as_float(v[k + 1]), cs, -ref));
                    if (!whole) {
                        const int at = key + c + k;
                        if (at > pos || at < low || (bad[c / 32] >> k & 1u)) p0 = 0.f;
                        if (at + 1 > pos || at + 1 < low || (bad[c / 32] >> k & 2u)) p1 = 0.f;
                    }
                    part[(k >> 1) & 1] += p0;
                    part[2 + ((k >> 1) & 1)] += p1;
                    h[k >> 1] = pack_h2(p0, p1);
                }
                at_st16(s_at + c / 2, h);
            }
            sum += (part[0] + part[1]) + (part[2] + part[3]);
            at_wait_st();
            at_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(p_full + 8 * qa);
        }
        if (ok && n_tiles) ok = __all_sync(0xffffffffu, mbar_wait(o_full, 0));
        at_after();
        T* out = static_cast<T*>(P.out) + ((long long)(S.row0 + r / group) * P.n_heads + hk * group + r % group) * D;
        const float inv = sum > 0.f ? __fdividef(1.f, sum) : sum == sum ? 0.f : sum;
#pragma unroll
        for (int c = 0; c < D; c += 32) {
            uint32_t v[32];
            if (n_tiles && ok) {
                at_ld32(o_at + c, v);
                at_wait_ld();
            }
            if (r < rows && ok) {
#pragma unroll
                for (int k = 0; k < 32; k += 4) {
                    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (inv != 0.f)
                        y = make_float4(__uint_as_float(v[k]) * inv, __uint_as_float(v[k + 1]) * inv, __uint_as_float(v[k + 2]) * inv,
                                        __uint_as_float(v[k + 3]) * inv);
                    store4(out + c + k, y);
                }
            }
        }
    } else if (qa == NQ) {
        // ---- producers -----------------------------------------------------------------------------
        const int pw = warp & 3, pt = tid - NQ * 128;             // producer warp and thread
        constexpr int kRows = BN / 4, kGroups = kRows / 8;        // keys a warp, 8-key groups
        constexpr int kWk = J * KB / 4;                           // words of a lane's K run
        constexpr int JV = BN == 128 ? J : J / 2, kWv = JV * VB / 4;      // V blocks of a lane, words of a pair's run
        uint32_t kw[kGroups][kWk], vw[4][kWv], sw[J], bad = 0;
        const int kk = lane & 7, kt = lane >> 3;                  // K: key within 8, run
        const int vg = lane & 7, vkc = BN == 128 ? lane >> 3 : (lane >> 3) & 1, vj = BN == 128 ? 0 : (lane >> 4) * JV;
        const int* table = P.tables + (long long)b * P.width;
        // page of a 16-aligned run of keys, -1: nothing to see there
        auto page_of = [&](int key) -> long long {
            if (key > last || key + 15 < first) return -1;
            const int p = __ldg(table + (key >> P.c.page_shift));
            if (p >= 0 && p < P.c.n_pages) return p;
            if (P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
            return -1;
        };
        auto load_k = [&](int i) {
            const int key0 = (kt0 + i) * BN;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int key = key0 + kRows * pw + 8 * q;
                const long long page = page_of(key & ~15);
                if (page >= 0) {
                    at_ldg<kWk>(kw[q], P.c.k + P.c.k_row(page, hk, (key & (P.c.page() - 1)) + kk) + kt * J * KB);
                } else {
#pragma unroll
                    for (int w = 0; w < kWk; ++w) kw[q][w] = 0u;
                }
            }
            // scales of key pt: nobody sees it: 0 (it may hold anything)
            const int key = key0 + pt;
            const bool seen = pt < BN && key >= first && key <= last;
            const long long page = seen ? page_of(key & ~15) : -1;
            bad = __ballot_sync(0xffffffffu, seen && page < 0);
            if (page >= 0) {
                at_ldg<J>(sw, reinterpret_cast<const uint8_t*>(P.c.sc + P.c.scale_row(page, hk, key & (P.c.page() - 1))));
            } else {
#pragma unroll
                for (int w = 0; w < J; ++w) sw[w] = 0u;
            }
        };
        auto load_v = [&](int i) {
            const int key = (kt0 + i) * BN + kRows * pw + 8 * vkc;
            const long long page = page_of(key & ~15);
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                if (page >= 0) {
                    at_ldg<kWv>(vw[p], P.c.v + P.c.v_pair(page, hk, ((key & (P.c.page() - 1)) >> 1) + p) + (vg * J + vj) * VB);
                } else {
#pragma unroll
                    for (int w = 0; w < kWv; ++w) vw[p][w] = 0u;
                }
            }
        };
        if (n_tiles) load_k(0), load_v(0);
        for (int i = 0; i < n_tiles; ++i) {
            const int st = i & 1;
            const uint32_t par = uint32_t(i >> 1) & 1u;
            const uint32_t s_k = sm + Sh::kOffSK + st * Sh::kScaleK, s_v = sm + Sh::kOffSV + st * Sh::kScaleV;
            if (i >= 2) ok = mbar_wait(k_free + 8 * st, par ^ 1u);
            if (i >= 2 && ok) ok = mbar_wait(v_free + 8 * st, par ^ 1u);
            // scales: K's by key, V's by block (so that eight keys of a block are one word of 16 bytes)
            if (pt < BN) {
                __half* dk = reinterpret_cast<__half*>(tc_smem_ + Sh::kOffSK + st * Sh::kScaleK) + pt * J;
                __half* dv = reinterpret_cast<__half*>(tc_smem_ + Sh::kOffSV + st * Sh::kScaleV) + pt;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    const uint32_t a = sw[j >> 1], c = sw[(J + j) >> 1];
                    dk[j] = __ushort_as_half((unsigned short)(j & 1 ? a >> 16 : a & 0xFFFFu));
                    dv[j * BN] = __ushort_as_half((unsigned short)((J + j) & 1 ? c >> 16 : c & 0xFFFFu));
                }
            }
            uint32_t all;                                         // the four warps go on, or leave, together
            if (lane == 0) reinterpret_cast<uint32_t*>(tc_smem_ + Sh::kOffBad)[4 * st + pw] = bad;
            asm volatile("{ .reg .pred p, q; setp.ne.b32 p, %1, 0; barrier.cta.red.and.pred q, 1, 128, p; selp.u32 %0, 1, 0, q; }"
                         : "=r"(all) : "r"(uint32_t(ok)) : "memory");
            ok = all != 0;
            if (!ok) break;
#pragma unroll
            for (int q = 0; q < kGroups; ++q) {
                const int key = kRows * pw + 8 * q + kk;
                const uint32_t dst = sm + Sh::kOffK + st * Sh::kK + (key >> 3) * Sh::kSboK + (key & 7) * 16;
#pragma unroll
                for (int j = 0; j < J; ++j) {
                    unsigned short d;
                    asm volatile("ld.shared.u16 %0, [%1];" : "=h"(d) : "r"(s_k + (key * J + j) * 2));
                    uint32_t o[4];
                    unpack_k8<KB>(&kw[q][j * KB / 4], __half2half2(__ushort_as_half(d)), o);
                    at_sts128(dst + (4 * j + kt) * 128, o[0], o[1], o[2], o[3]);
                }
            }
            at_fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(k_full + 8 * st);
            if (i + 1 < n_tiles) load_k(i + 1);
            {
                const int kc = (kRows / 8) * pw + vkc;            // 8-key core of the stage
#pragma unroll
                for (int j = 0; j < JV; ++j) {
                    uint32_t d[4];
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(d[0]), "=r"(d[1]), "=r"(d[2]), "=r"(d[3])
                                 : "r"(s_v + ((vj + j) * BN + 8 * kc) * 2));
#pragma unroll
                    for (int s = 0; s < 4; ++s) {                 // the value differs by lane: no two of eight lanes share a bank
                        const int e = (s + (vg >> 1)) & 3, n = 32 * (vj + j) + 4 * vg + e;
                        uint32_t o[4];
#pragma unroll
                        for (int p = 0; p < 4; ++p) o[p] = unpack_v<VB>(&vw[p][j * VB / 4], e, bits_h2(d[p]));
                        at_sts128(sm + Sh::kOffV + st * Sh::kV + (n >> 3) * Sh::kSboV + kc * 128 + (n & 7) * 16, o[0], o[1], o[2], o[3]);
                    }
                }
            }
            at_fence_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(v_full + 8 * st);
            if (i + 1 < n_tiles) load_v(i + 1);
        }
    } else if (lane == 0) {
        // ---- MMA -----------------------------------------------------------------------------------
        constexpr uint32_t id_s = at_idesc(BN), id_o = at_idesc(D);
        auto scores = [&](int a, int i) {
            const uint32_t q = sm + a * Sh::kQ, k = sm + Sh::kOffK + (i & 1) * Sh::kK;
#pragma unroll
            for (int s = 0; s < D / 16; ++s)
                at_mma_ss(tmem + a * BN, at_desc(q + 256 * s, Sh::kSboQ), at_desc(k + 256 * s, Sh::kSboK), id_s, s > 0);
            at_commit(s_full + 8 * a);
        };
        if (n_tiles) {
            ok = mbar_wait(k_full, 0);
            at_after();
            if (ok) {
                for (int a = 0; a < NQ; ++a) scores(a, 0);
                at_commit(k_free);
            }
        }
        for (int i = 0; i < n_tiles && ok; ++i) {
            const int st = i & 1;
            for (int a = 0; a < NQ && ok; ++a) {
                ok = mbar_wait(p_full + 8 * a, i & 1);
                if (a == 0 && ok) ok = mbar_wait(v_full + 8 * st, uint32_t(i >> 1) & 1u);
                if (!ok) break;
                at_after();
                const uint32_t v = sm + Sh::kOffV + st * Sh::kV;
#pragma unroll
                for (int s = 0; s < BN / 16; ++s)
                    at_mma_ts(tmem + NQ * BN + a * D, tmem + a * BN + 8 * s, at_desc(v + 256 * s, Sh::kSboV), id_o, i > 0 || s > 0);
                if (a == NQ - 1) at_commit(v_free + 8 * st);
                if (i + 1 < n_tiles) {
                    if (a == 0) ok = mbar_wait(k_full + 8 * (st ^ 1), uint32_t((i + 1) >> 1) & 1u);
                    if (!ok) break;
                    at_after();
                    scores(a, i + 1);
                    if (a == NQ - 1) at_commit(k_free + 8 * (st ^ 1));
                }
            }
        }
        if (n_tiles) {                                            // everything issued is done before the memory is given back
            at_commit(o_full);
            ok = mbar_wait(o_full, 0) && ok;
        }
    }
    if (!ok && lane == 0 && P.status) atomicOr(P.status, DEV_TIMEOUT);
    __syncwarp();
    at_before();
    __syncthreads();
    at_after();
    if (warp == 0) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" :: "r"(tmem), "r"(512) : "memory");
}

// ---- host -------------------------------------------------------------------------------------------


// Rows of a sequence (new tokens x heads of a key head) from which the tiles are used.
constexpr int kAttnTcRows = 65;

inline bool attn_tc_used(const KvView& c, int dtype, int n_heads, int max_new) {
    return dtype != QMV_OUT_F32 && (long long)max_new * (n_heads / c.n_kv) >= kAttnTcRows;
}
inline int attn_tc_tiles(const KvView& c, int n_heads, int max_new) {
    const long long rows = (long long)max_new * (n_heads / c.n_kv);
    const int per = c.J == 8 ? 128 : 256;
    return int((rows + per - 1) / per);
}

template <int DT, int J, int KB, int VB>
int attn_tc_go(const AttnParams& P, cudaStream_t st) {
    using Sh = AttnTcShape<J>;
    static SmemGrant grant;
    if (const int e = grant(attn_tc_kernel<DT, J, KB, VB>, Sh::kSmem)) return e;
    return launch_pdl_smem(attn_tc_kernel<DT, J, KB, VB>, dim3(P.row_tiles * P.c.n_kv * P.n_seq), dim3(Sh::kThreads), Sh::kSmem, st, P);
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
