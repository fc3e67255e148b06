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

// the activation input of a thread's V consecutive values (32 / V lanes a group): the arithmetic of quantize_group
template <int V>
__device__ __forceinline__ void quantise_run(const float (&x)[V], long long i, bool live, const NormBlockParams& P) {
    float a = 0.f, sum = 0.f;
#pragma unroll
    for (int k = 0; k < V; ++k) a = fmaxf(a, fabsf(x[k])), sum += x[k];
#pragma unroll
    for (int o = 1; o < 32 / V; o *= 2) {
        a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, o));
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    const float d = __fdiv_rn(a, 127.0f), d2 = __fdiv_rn(d, 254.0f);
    uint32_t q1[V / 4], q2[V / 4];
#pragma unroll
    for (int k = 0; k < V; ++k) {
        int q = 0, r2 = 0;
        if (d > 0.f) {
            q = __float2int_rn(__fdiv_rn(x[k], d));
            r2 = max(-127, min(127, __float2int_rn(__fdiv_rn(__fmaf_rn(-float(q), d, x[k]), d2))));
        }
        if (k % 4 == 0) q1[k / 4] = q2[k / 4] = 0u;
        q1[k / 4] |= (uint32_t(q) & 255u) << (8 * (k % 4)), q2[k / 4] |= (uint32_t(r2) & 255u) << (8 * (k % 4));
    }
    if (!live) return;
#pragma unroll
    for (int k = 0; k < V / 4; ++k) {
        reinterpret_cast<uint32_t*>(P.xq + i)[k] = q1[k];
        reinterpret_cast<uint32_t*>(P.xq2 + i)[k] = q2[k];
    }
    if (i % 32 == 0) P.xd[i / 32] = d, P.xs[i / 32] = sum;
}

// 16 bytes of values as fp32 and back
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[4], float) {
    x[0] = __uint_as_float(w.x), x[1] = __uint_as_float(w.y), x[2] = __uint_as_float(w.z), x[3] = __uint_as_float(w.w);
}
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[8], __nv_bfloat16) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) x[2 * i] = __uint_as_float(v[i] << 16), x[2 * i + 1] = __uint_as_float(v[i] & 0xFFFF0000u);
}
__device__ __forceinline__ void unpack16(uint4 w, float (&x)[8], __half) {
    const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&v[i]));
        x[2 * i] = f.x, x[2 * i + 1] = f.y;
    }
}
template <class T, int V>
__device__ __forceinline__ void store_run(T* p, const float (&x)[V]) {
    if constexpr (V == 4) {
        store4(p, make_float4(x[0], x[1], x[2], x[3]));
    } else {
        uint4 w;
        T* t = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < 8; ++i) from_float(t[i], x[i]);
        *reinterpret_cast<uint4*>(p) = w;
    }
}

// One CTA a row of whole 16-byte pieces, C of them a thread: z = y rsqrt(mean y^2 + eps) w_post, h' = h + rs gate z,
// xn = h' rsqrt(mean h'^2 + eps) w_pre.  Everything a thread reads of the row is asked for at once and stays in registers
// between the two sums, so the row crosses memory once each way; sums in fp32, each output rounded once.  Bound by memory for
// many rows (C chosen so that a CTA has about 256 threads), by two barriers behind one trip to memory for few (C least).
template <int DT, int C, int TH>
__global__ void __launch_bounds__(TH) norm_rows_kernel(const __grid_constant__ NormBlockParams P) {
    using T = typename Elem<DT>::type;
    constexpr int V = 16 / elem_bytes(DT);
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* y = static_cast<const T*>(P.y) + row * P.y_stride;
    const T* h = static_cast<const T*>(P.h) + row * P.h_stride;
    const T* gate = P.gate ? static_cast<const T*>(P.gate) + row * P.gate_stride : nullptr;
    uint4 ry[C], rh[C], rg[C];
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        ry[c] = rh[c] = rg[c] = make_uint4(0u, 0u, 0u, 0u);
        if (i < P.n) {
            ry[c] = __ldg(reinterpret_cast<const uint4*>(y + i));
            rh[c] = *reinterpret_cast<const uint4*>(h + i);       // may be h_out itself
            if (gate) rg[c] = __ldg(reinterpret_cast<const uint4*>(gate + i));
        }
    }
    float inv = 1.f;
    if (P.w_post) {
        float ss = 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            float x[V];
            unpack16(ry[c], x, T{});
#pragma unroll
            for (int k = 0; k < V; ++k) ss = fmaf(x[k], x[k], ss);
        }
        inv = rsqrtf(block_sum(ss, red[0]) / float(P.n) + P.eps);
    }
    float v[C][V], ss = 0.f;
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        float z[V], a[V], g[V], w[V];
        unpack16(ry[c], z, T{});
        unpack16(rh[c], a, T{});
        unpack16(rg[c], g, T{});
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const float4 f = P.w_post && i < P.n ? load4(P.w_post + i + k) : make_float4(1.f, 1.f, 1.f, 1.f);
            w[k] = f.x, w[k + 1] = f.y, w[k + 2] = f.z, w[k + 3] = f.w;
        }
#pragma unroll
        for (int k = 0; k < V; ++k) {
            float t = P.w_post ? z[k] * inv * w[k] : z[k];
            if (gate) t *= g[k];
            v[c][k] = i < P.n ? a[k] + P.rs * t : 0.f;
            ss = fmaf(v[c][k], v[c][k], ss);
        }
        if (i < P.n) store_run(static_cast<T*>(P.h_out) + row * P.n + i, v[c]);
    }
    if (!P.w_pre) return;
    inv = rsqrtf(block_sum(ss, red[1]) / float(P.n) + P.eps);
#pragma unroll
    for (int c = 0; c < C; ++c) {
        const int i = (c * int(blockDim.x) + int(threadIdx.x)) * V;
        float x[V];
#pragma unroll
        for (int k = 0; k < V; k += 4) {
            const float4 f = i < P.n ? load4(P.w_pre + i + k) : make_float4(0.f, 0.f, 0.f, 0.f);
            x[k] = v[c][k] * inv * f.x, x[k + 1] = v[c][k + 1] * inv * f.y, x[k + 2] = v[c][k + 2] * inv * f.z, x[k + 3] = v[c][k + 3] * inv * f.w;
        }
        if (i < P.n) store_run(static_cast<T*>(P.xn) + row * P.n + i, x);
        if (P.xq) quantise_run<V>(x, row * P.n + i, i < P.n, P);  // n % 32 == 0: whole groups
    }
}

// Rows of any length and alignment, value by value through shared memory (y, then h'), four values of a thread in flight (4000
// rows of 4099 bf16 values: one at a time 78 us, four 44).
template <int DT, int TH>
__global__ void __launch_bounds__(TH) norm_any_kernel(const __grid_constant__ NormBlockParams P) {
    using T = typename Elem<DT>::type;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    extern __shared__ float v[];          // y, then h'
    __shared__ float red[2][32];
    const long long row = blockIdx.x;
    const T* y = static_cast<const T*>(P.y) + row * P.y_stride;
    const T* h = static_cast<const T*>(P.h) + row * P.h_stride;
    const T* gate = P.gate ? static_cast<const T*>(P.gate) + row * P.gate_stride : nullptr;
    constexpr int U = 4;                  // values a thread asks for before it uses one
    float ss = 0.f;
    for (int i0 = threadIdx.x; i0 < P.n; i0 += U * TH) {
        T ry[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) ry[u] = y[i0 + TH * u];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) {
                const float a = to_float(ry[u]);
                v[i0 + TH * u] = a;
                ss += a * a;
            }
    }
    float inv = 1.f;
    if (P.w_post) inv = rsqrtf(block_sum(ss, red[0]) / float(P.n) + P.eps);
    ss = 0.f;
    for (int i0 = threadIdx.x; i0 < P.n; i0 += U * TH) {
        T rh[U], rg[U];
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) {
                const int i = i0 + TH * u;
                rh[u] = h[i];             // may be h_out itself
                w[u] = P.w_post ? P.w_post[i] : 1.f;
                if (gate) rg[u] = gate[i];
            }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) {
                const int i = i0 + TH * u;
                float z = P.w_post ? v[i] * inv * w[u] : v[i];
                if (gate) z *= to_float(rg[u]);
                const float a = to_float(rh[u]) + P.rs * z;
                v[i] = a;
                ss += a * a;
                from_float(static_cast<T*>(P.h_out)[row * P.n + i], a);
            }
    }
    if (!P.w_pre) return;
    inv = rsqrtf(block_sum(ss, red[1]) / float(P.n) + P.eps);
    for (int i0 = threadIdx.x; i0 < P.n; i0 += U * TH) {
        float w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) w[u] = P.w_pre[i0 + TH * u];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (i0 + TH * u < P.n) {
                const int i = i0 + TH * u;
                const float x = v[i] * inv * w[u];
                from_float(static_cast<T*>(P.xn)[row * P.n + i], x);
                if (P.xq) quantize_group(x, row * P.n + i, P.xq, P.xq2, P.xd, P.xs);     // n % 32 == 0: whole warps
            }
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
    const bool whole = n % (16 / int(one)) == 0 && aligned(y, 16) && aligned(h, 16) && aligned(gate, 16) && aligned(h_out, 16) && aligned(xn, 16) &&
                       aligned(w_post, 16) && aligned(w_pre, 16) && y_stride * one % 16 == 0 && h_stride * one % 16 == 0 && gate_stride * one % 16 == 0;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return by_elem(dtype, [&](auto c) {
        constexpr int DT = decltype(c)::value;
        if (whole) {
            // Pieces a thread: for rows that fill the GPU CTAs of about 256 threads (8192 rows of 4096 values: bf16 52 us, fp32 83;
            // of up to 1024 threads 74 and 104), else the fewest (one row, 200 calls in a graph: fp32 2.6 us a call, with 256 threads 3.4).  C 4 with up
            // to 512 threads has the registers for it.  Rows of more than 4096 pieces are left to the other kernel
            const int pieces = n * int(one) / 16, most = rows >= 2LL * sm_count() ? 256 : 1024;
            const int C = pieces <= most ? 1 : pieces <= 2 * most ? 2 : 4;
            const dim3 block(((pieces + C - 1) / C + 31) / 32 * 32), grid(static_cast<unsigned>(rows));
            if (C == 1) return launch_pdl(norm_rows_kernel<DT, 1, 1024>, grid, block, st, P);
            if (C == 2) return launch_pdl(norm_rows_kernel<DT, 2, 1024>, grid, block, st, P);
            if (block.x <= 512) return launch_pdl(norm_rows_kernel<DT, 4, 512>, grid, block, st, P);
            if (block.x <= 1024) return launch_pdl(norm_rows_kernel<DT, 4, 1024>, grid, block, st, P);
        }
        // fewer threads for short rows (20000 of 131 bf16 values: 64 threads 22 us, 256 43), more where a row's shared memory leaves
        // few CTAs an SM (1000 of 16381 in fp32: 512 threads 68 us, 256 98)
        auto any = [&](auto th) {
            constexpr int TH = decltype(th)::value;
            const size_t smem = size_t(n) * 4;
            static SmemGrant grant;
            if (smem > 32 * 1024)
                if (const int e = grant(norm_any_kernel<DT, TH>, size_t(QMV_NORM_BLOCK_MAX) * 4)) return e;
            return launch_pdl_smem(norm_any_kernel<DT, TH>, dim3(unsigned(rows)), dim3(TH), smem, st, P);
        };
        if (n <= 256) return any(std::integral_constant<int, 64>{});
        if (n <= 8192) return any(std::integral_constant<int, 256>{});
        return any(std::integral_constant<int, 512>{});
    });
}
