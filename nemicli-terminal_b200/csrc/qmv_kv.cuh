// The quantised key / value cache: where its bytes lie, and what the kernels of qmv_kv.cu (write, read)
// and qmv_attn.cu (attention) share.
//
// The cache is paged.  A slot is page * P + place for pages of P tokens.  K and V are each held as Q4_0 or
// Q8_0: blocks of 32 values along the head dimension, one fp16 scale d a block, value = d * code.  The bytes
// of a token are ordered for the tensor-core fragments of the attention kernels, so that one 4 (Q4_0) or 8
// (Q8_0) byte word unpacks into fp16 pairs without a shuffle (J = dim / 32 blocks, b = 4 or 8):
//   k       [page][head][P][4 t][J][b]       values 8 t .. 8 t + 7 of block j: lane t of a quad holds every
//                                            block's 8 values in one run of J * b bytes
//   v       [page][head][P / 2][8 g][J][b]   values 4 g .. 4 g + 3 of block j of tokens 2 i and 2 i + 1: the
//                                            16-bit halves of each word are one token each, so a word
//                                            unpacks into (even token, odd token) pairs of one value
//   scales  [page][head][P][2][J] fp16       K's, then V's
// Codes are offset by 8 or 128.  In a Q4_0 K word value n sits at bit 16 (n & 1) + 4 (n >> 1); in a V word at
// bit 16 (token & 1) + 4 n.  In the two Q8_0 K words value n sits in word n >> 2 at byte 2 (n & 1) + ((n & 3) >> 1);
// in the V words in word n >> 1 at byte 2 (token & 1) + (n & 1).
#pragma once
#include <atomic>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "qmv_host.cuh"
#include "../../include/nemicli_qmv.h"

namespace qmv {

constexpr float kKvMax = 65504.0f;        // values are clamped to fp16's range before they are quantised

struct KvView {
    uint8_t* k;
    uint8_t* v;
    __half* sc;
    long long n_pages;
    int n_kv, page_shift;                 // key heads, log2 of the tokens a page
    int dim, J;                           // values a head, blocks a head
    int kb, vb;                           // bytes of 8 K values and of 4 + 4 V values: 4 (Q4_0) or 8 (Q8_0)
    __host__ __device__ int page() const { return 1 << page_shift; }
    // byte offsets of the rows (64 bits: a long cache passes 2^31)
    __device__ __forceinline__ long long k_row(long long page, int head, int at) const {
        return (((page * n_kv + head) << page_shift) + at) * (long long)(4 * J * kb);
    }
    __device__ __forceinline__ long long v_pair(long long page, int head, int pair) const {
        return (((page * n_kv + head) << (page_shift - 1)) + pair) * (long long)(8 * J * vb);
    }
    __device__ __forceinline__ long long scale_row(long long page, int head, int at) const {      // in halves
        return (((page * n_kv + head) << page_shift) + at) * (long long)(2 * J);
    }
};

// the host's description (include/nemicli_qmv.h) checked and turned into a view; a QMV_* status
inline int kv_view(const qmv_kv_cache* c, KvView& view) {
    if (!c || !c->k || !c->v || !c->scales) return ST_NULL;
    if ((c->k_type != F_Q4_0 && c->k_type != F_Q8_0) || (c->v_type != F_Q4_0 && c->v_type != F_Q8_0)) return ST_BAD_FORMAT;
    if (c->dim != 64 && c->dim != 96 && c->dim != 128 && c->dim != 256) return ST_BAD_SHAPE;
    int shift = 4;
    while (shift < 10 && (1 << shift) != c->page) ++shift;
    if ((1 << shift) != c->page || c->n_pages <= 0 || c->n_kv <= 0 || c->n_kv > 65535) return ST_BAD_SHAPE;
    if (c->n_pages > (1LL << 40) / c->page) return ST_BAD_SHAPE;
    if ((long long)c->n_kv * c->dim * c->page > (1LL << 30)) return ST_BAD_SHAPE;      // a page's bytes fit 31 bits
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->scales, 16)) return ST_BAD_ALIGN;
    view.k = static_cast<uint8_t*>(c->k);
    view.v = static_cast<uint8_t*>(c->v);
    view.sc = static_cast<__half*>(c->scales);
    view.n_pages = c->n_pages;
    view.n_kv = c->n_kv;
    view.page_shift = shift;
    view.dim = c->dim;
    view.J = c->dim / 32;
    view.kb = c->k_type == F_Q4_0 ? 4 : 8;
    view.vb = c->v_type == F_Q4_0 ? 4 : 8;
    return ST_OK;
}

// the right to more than 48 KB of shared memory (a kernel's fixed part, under 16 KB, counts too), asked for once a kernel and device
struct SmemGrant {
    std::atomic<uint64_t> done{0};
    template <class Kernel>
    int operator()(Kernel* kernel, size_t bytes) {
        int dev = 0;
        cudaGetDevice(&dev);
        if (bytes <= 32 * 1024 || (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1))) return ST_OK;
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(bytes));
        if (e != cudaSuccess) {
            set_last_cuda_error(int(e));
            return ST_LAUNCH;
        }
        if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
        return ST_OK;
    }
};

// element types of dense inputs and outputs (QMV_OUT_*): four consecutive values at a time
template <int DT> struct Elem;
template <> struct Elem<QMV_OUT_F32> { using type = float; };
template <> struct Elem<QMV_OUT_BF16> { using type = __nv_bfloat16; };
template <> struct Elem<QMV_OUT_F16> { using type = __half; };
__host__ __device__ constexpr int elem_bytes(int dt) { return dt == QMV_OUT_F32 ? 4 : 2; }

__device__ __forceinline__ float4 load4(const float* p) { return __ldg(reinterpret_cast<const float4*>(p)); }
__device__ __forceinline__ float4 load4(const __nv_bfloat16* p) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                       __uint_as_float(w.y & 0xFFFF0000u));
}
__device__ __forceinline__ float4 load4(const __half* p) {
    const uint2 w = __ldg(reinterpret_cast<const uint2*>(p));
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x));
    const float2 b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(float* p, float4 v) { *reinterpret_cast<float4*>(p) = v; }
__device__ __forceinline__ void store4(__nv_bfloat16* p, float4 v) {
    __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}
__device__ __forceinline__ void store4(__half* p, float4 v) {
    __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<uint32_t*>(&a), *reinterpret_cast<uint32_t*>(&b));
}
// Four values that a cache holds, or a mean of such: fp16 ends at 65504 (a Q8_0 block of clamped values holds 65532, which would
// round to an infinity)
__device__ __forceinline__ uint32_t pack_held(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
template <class T>
__device__ __forceinline__ void store4_held(T* p, float4 v) {
    if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<uint2*>(p) = make_uint2(pack_held(v.x, v.y), pack_held(v.z, v.w));
    else store4(p, v);
}
__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
__device__ __forceinline__ void from_float(float& o, float v) { o = v; }
__device__ __forceinline__ void from_float(__nv_bfloat16& o, float v) { o = __float2bfloat16_rn(v); }
__device__ __forceinline__ void from_float(__half& o, float v) { o = __float2half_rn(v); }

// Calls f(std::integral_constant<int, DT>) for a QMV_OUT_* type; ST_BAD_SHAPE for an unknown one.
template <class Fn>
int by_elem(int dt, Fn&& f) {
    switch (dt) {
    case QMV_OUT_F32: return f(std::integral_constant<int, QMV_OUT_F32>{});
    case QMV_OUT_BF16: return f(std::integral_constant<int, QMV_OUT_BF16>{});
    case QMV_OUT_F16: return f(std::integral_constant<int, QMV_OUT_F16>{});
    }
    return ST_BAD_SHAPE;
}

}  // namespace qmv
