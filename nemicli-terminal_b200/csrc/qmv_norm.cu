// The norms before and after a block, fused with its gate and residual (C-ABI declaration: include/nemicli_qmv.h).
#include <type_traits>

#include "qmv_kv.cuh"

using namespace qmv;

namespace {

struct NormBlockParams {
    const void* y;
    const void* h;
    const void* gate;                     // null, or rows gate_stride values apart (0: one row for all)
    const float* w_post;                  // null: no norm after the block
    const float* w_pre;                   // null: no norm before the next one (xn unused)
    long long y_stride, h_stride, gate_stride;
    void* h_out;                          // dense rows of n
    void* xn;
    int8_t* xq;                           // activation input of xn (all four or none)
    int8_t* xq2;
    float* xd;
    float* xs;
    float eps, rs;
    int n;
};

__device__ __forceinline__ float block_sum(float v, float* red) {
    v = warp_sum(v);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    const int warps = blockDim.x >> 5, lane = threadIdx.x & 31;
    return warp_sum(lane < warps ? red[lane] : 0.f);
}

// One CTA a row: z = y rsqrt(mean y^2 + eps) w_post, h' = h + rs gate z, xn = h' rsqrt(mean h'^2 + eps) w_pre, the sums
// and h' in fp32 (shared memory), each output rounded once from them.
template <int DT>
__global__ void __launch_bounds__(256) norm_block_kernel(const __grid_constant__ NormBlockParams P) {
    using T = typename Elem<DT>::type;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    extern __shared__ float v[];          // y, then h'
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* y = static_cast<const T*>(P.y) + row * P.y_stride;
    const T* h = static_cast<const T*>(P.h) + row * P.h_stride;
    const T* gate = P.gate ? static_cast<const T*>(P.gate) + row * P.gate_stride : nullptr;
    float ss = 0.f;
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
        const float a = to_float(y[i]);
        v[i] = a;
        ss += a * a;
    }
    float inv = 1.f;
    if (P.w_post) inv = rsqrtf(block_sum(ss, red[0]) / float(P.n) + P.eps);
    ss = 0.f;
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
        float z = P.w_post ? v[i] * inv * P.w_post[i] : v[i];
        if (gate) z *= to_float(gate[i]);
        const float a = to_float(h[i]) + P.rs * z;
        v[i] = a;
        ss += a * a;
        from_float(static_cast<T*>(P.h_out)[row * P.n + i], a);
    }
    if (!P.w_pre) return;
    inv = rsqrtf(block_sum(ss, red[1]) / float(P.n) + P.eps);
    for (int i = threadIdx.x; i < P.n; i += blockDim.x) {
        const float x = v[i] * inv * P.w_pre[i];
        from_float(static_cast<T*>(P.xn)[row * P.n + i], x);
        if (P.xq) quantize_group(x, row * P.n + i, P.xq, P.xq2, P.xd, P.xs);     // n % 32 == 0: whole warps
    }
}

}  // namespace

extern "C" int qmv_norm_block(const void* y, long long y_stride, const void* h, long long h_stride, const void* gate,
                              long long gate_stride, const float* w_post, const float* w_pre, int dtype, float eps,
                              float rs, long long rows, int n, void* h_out, void* xn, int8_t* xq, int8_t* xq2, float* xd,
                              float* xs, void* stream) {
    if (!y || !h || !h_out || (w_pre && !xn) || (xq && (!w_pre || !xq2 || !xd || !xs))) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (n <= 0 || n > QMV_NORM_BLOCK_MAX || (xq && n % 32) || y_stride < n || h_stride < n ||
        (gate && gate_stride != 0 && gate_stride < n))
        return ST_BAD_SHAPE;
    if (rows < 0 || rows > 0x7FFFFFFFLL) return ST_BAD_TOKENS;
    const uintptr_t one = elem_bytes(dtype);
    if (!aligned(y, one) || !aligned(h, one) || !aligned(gate, one) || !aligned(h_out, one) || !aligned(xn, one) ||
        !aligned(w_post, 4) || !aligned(w_pre, 4) || !aligned(xq, 16) || !aligned(xq2, 16) || !aligned(xd, 4) || !aligned(xs, 4))
        return ST_BAD_ALIGN;
    if (rows == 0) return ST_OK;
    NormBlockParams P{y, h, gate, w_post, w_pre, y_stride, h_stride, gate_stride, h_out, xn, xq, xq2, xd, xs, eps, rs, n};
    return by_elem(dtype, [&](auto c) {
        constexpr int DT = decltype(c)::value;
        const size_t smem = size_t(n) * 4;
        static SmemGrant grant;
        if (smem > 32 * 1024)
            if (const int e = grant(norm_block_kernel<DT>, size_t(QMV_NORM_BLOCK_MAX) * 4)) return e;
        return launch_pdl_smem(norm_block_kernel<DT>, dim3(unsigned(rows)), dim3(256), smem, static_cast<cudaStream_t>(stream), P);
    });
}
