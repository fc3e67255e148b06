// Writing a quantised key / value cache and reading it back (layout: qmv_kv.cuh; C-ABI declarations:
// include/nemicli_qmv.h).
#include <type_traits>

#include "qmv_kv.cuh"

using namespace qmv;

namespace {

struct KvWriteParams {
    KvView c;
    const void* k;
    const void* v;
    const void* q;                        // queries to rotate (or null)
    void* q_out;
    long long k_stride, v_stride, q_stride;   // values between rows
    const long long* slots;
    const float* cos_t;                   // [n_pos][rot / 2] (or null: no rotation)
    const float* sin_t;
    const long long* pos;
    long long n_pos;
    int rot, paired, n_q;
    int rows;
    int* status;
};

// The four values 4 m .. 4 m + 3 of block j of one head, rotated: value i < rot pairs with i + rot / 2 (or,
// paired, 2 i with 2 i + 1), angle i of the row's position.  y1 = x1 c - x2 s, y2 = x2 c + x1 s; every product and
// sum is rounded on its own (no fused multiply-add), so the codes follow from the inputs bit for bit.
template <class T>
__device__ __forceinline__ float4 rotated(const T* row, int i0, const KvWriteParams& P, const float* c, const float* s) {
    float4 x = load4(row + i0);
    if (!c || i0 >= P.rot) return x;
    if (P.paired) {
        const float2 cc = __ldg(reinterpret_cast<const float2*>(c + i0 / 2)), ss = __ldg(reinterpret_cast<const float2*>(s + i0 / 2));
        return make_float4(__fsub_rn(__fmul_rn(x.x, cc.x), __fmul_rn(x.y, ss.x)), __fadd_rn(__fmul_rn(x.y, cc.x), __fmul_rn(x.x, ss.x)),
                           __fsub_rn(__fmul_rn(x.z, cc.y), __fmul_rn(x.w, ss.y)), __fadd_rn(__fmul_rn(x.w, cc.y), __fmul_rn(x.z, ss.y)));
    }
    const int half = P.rot / 2;
    const bool first = i0 < half;
    const int a = first ? i0 : i0 - half;
    const float4 o = load4(row + (first ? i0 + half : a)), cc = load4(c + a), ss = load4(s + a);
    if (first)
        return make_float4(__fsub_rn(__fmul_rn(x.x, cc.x), __fmul_rn(o.x, ss.x)), __fsub_rn(__fmul_rn(x.y, cc.y), __fmul_rn(o.y, ss.y)),
                           __fsub_rn(__fmul_rn(x.z, cc.z), __fmul_rn(o.z, ss.z)), __fsub_rn(__fmul_rn(x.w, cc.w), __fmul_rn(o.w, ss.w)));
    return make_float4(__fadd_rn(__fmul_rn(x.x, cc.x), __fmul_rn(o.x, ss.x)), __fadd_rn(__fmul_rn(x.y, cc.y), __fmul_rn(o.y, ss.y)),
                       __fadd_rn(__fmul_rn(x.z, cc.z), __fmul_rn(o.z, ss.z)), __fadd_rn(__fmul_rn(x.w, cc.w), __fmul_rn(o.w, ss.w)));
}

__device__ __forceinline__ float cleaned(float x) {          // NaN counts as 0, the rest is clamped to +-65504
    return x != x ? 0.f : fminf(fmaxf(x, -kKvMax), kKvMax);
}

// Eight lanes (m = 0..7) hold four values each of one 32-value block; the block's scale, and each lane's codes with their
// offset.  Q4_0: d = fp16(x / -8) of the value of largest magnitude (the first of equal ones), codes
// clamp(rint(x / d), -8, 7); Q8_0: d = fp16(max |x| / 127), codes clamp(rint(x / d), -127, 127).  Divisions are
// IEEE, by the rounded d, the one the reader multiplies with.
__device__ __forceinline__ uint4 quantise4(float4 x, bool q4, __half& d) {
    x = make_float4(cleaned(x.x), cleaned(x.y), cleaned(x.z), cleaned(x.w));
    float m = x.x;
    if (fabsf(x.y) > fabsf(m)) m = x.y;
    if (fabsf(x.z) > fabsf(m)) m = x.z;
    if (fabsf(x.w) > fabsf(m)) m = x.w;
    const int lane = threadIdx.x & 7;
#pragma unroll
    for (int o = 1; o < 8; o *= 2) {
        const float other = __shfl_xor_sync(0xffffffffu, m, o);
        const bool lower = (lane & o) != 0;                   // the other lane's values come first
        if (fabsf(other) > fabsf(m) || (lower && fabsf(other) == fabsf(m))) m = other;
    }
    d = __float2half_rn(q4 ? __fmul_rn(m, -0.125f) : __fdiv_rn(fabsf(m), 127.0f));
    const float df = __half2float(d);
    const float lo = q4 ? -8.f : -127.f, hi = q4 ? 7.f : 127.f, off = q4 ? 8.f : 128.f;
    float c[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = (df == 0.f ? 0.f : fminf(fmaxf(rintf(__fdiv_rn(c[i], df)), lo), hi)) + off;
    return make_uint4(uint32_t(c[0]), uint32_t(c[1]), uint32_t(c[2]), uint32_t(c[3]));
}

// One 32-value block of one head of one row on eight lanes; rows x (K heads, V heads, rotated query heads) x J blocks.
// Bound by memory for long prompts, by its launch for a decode step.
template <int DT>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvWriteParams P) {
    using T = typename Elem<DT>::type;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int J = P.c.J, kv = P.c.n_kv;
    const int per_row = (2 * kv + P.n_q) * J;
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    const bool live = item < (long long)P.rows * per_row;     // idle groups still take part in the shuffles
    const int m = threadIdx.x & 7;
    const int row = live ? int(item / per_row) : 0, rem = live ? int(item - (long long)row * per_row) : 0;
    int head = rem / J;
    const int j = rem - head * J, i0 = 32 * j + 4 * m;
    const int kind = head < kv ? 0 : head < 2 * kv ? 1 : 2;   // K, V, Q
    head -= kind * kv;
    const float* c = nullptr;
    const float* s = nullptr;
    bool bad = false;
    if (P.cos_t) {
        const long long p = __ldg(P.pos + row);
        bad = p < 0 || p >= P.n_pos;
        if (kind != 1) {
            c = P.cos_t + (bad ? 0 : p) * (P.rot / 2);
            s = P.sin_t + (bad ? 0 : p) * (P.rot / 2);
        }
    }
    if (kind == 2) {
        float4 x = rotated(static_cast<const T*>(P.q) + row * P.q_stride + head * P.c.dim, i0, P, c, s);
        if (bad) x = make_float4(0.f, 0.f, 0.f, 0.f);
        if (live) store4(static_cast<T*>(P.q_out) + ((long long)row * P.n_q + head) * P.c.dim + i0, x);
    }
    const T* src = kind == 1 ? static_cast<const T*>(P.v) + row * P.v_stride : static_cast<const T*>(P.k) + row * P.k_stride;
    const bool q4 = (kind == 1 ? P.c.vb : P.c.kb) == 4;
    __half d;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (kind != 2) x = rotated(src + head * P.c.dim, i0, P, c, s);
    const uint4 n = quantise4(x, q4, d);
    // K: lanes 2 t and 2 t + 1 share the 8 values of t
    uint32_t word = q4 ? n.x | (n.y << 16) | (n.z << 4) | (n.w << 20) : n.x | (n.y << 16) | (n.z << 8) | (n.w << 24);
    if (q4 && (m & 1)) word <<= 8;
    const uint32_t both = word | __shfl_xor_sync(0xffffffffu, word, 1);
    if (!live || kind == 2) {
        if (live && bad && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
        return;
    }
    const long long slot = __ldg(P.slots + row);
    if (slot < 0) return;                                     // a padding row
    const long long page = slot >> P.c.page_shift;
    if (bad || page >= P.c.n_pages) {
        if (P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
        return;
    }
    const int at = int(slot & (P.c.page() - 1));
    if (m == 0) P.c.sc[P.c.scale_row(page, head, at) + kind * J + j] = d;
    if (kind == 0) {
        uint8_t* dst = P.c.k + P.c.k_row(page, head, at) + ((m >> 1) * J + j) * P.c.kb;
        if (!q4) *reinterpret_cast<uint32_t*>(dst + 4 * (m & 1)) = word;
        else if (!(m & 1)) *reinterpret_cast<uint32_t*>(dst) = both;
    } else {
        uint8_t* dst = P.c.v + P.c.v_pair(page, head, at >> 1) + (m * J + j) * P.c.vb + 2 * (at & 1);
        if (q4) {
            *reinterpret_cast<uint16_t*>(dst) = uint16_t(n.x | (n.y << 4) | (n.z << 8) | (n.w << 12));
        } else {
            *reinterpret_cast<uint16_t*>(dst) = uint16_t(n.x | (n.y << 8));
            *reinterpret_cast<uint16_t*>(dst + 4) = uint16_t(n.z | (n.w << 8));
        }
    }
}

struct KvReadParams {
    KvView c;
    const long long* slots;
    void* k;
    void* v;
    int rows;
    int* status;
};

// four values of a block (the inverse of kv_write_kernel's stores): d * code, one rounded product each
template <int DT>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadParams P) {
    using T = typename Elem<DT>::type;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int J = P.c.J, kv = P.c.n_kv, per_row = 2 * kv * J;
    const long long item = ((long long)blockIdx.x * blockDim.x + threadIdx.x) >> 3;
    if (item >= (long long)P.rows * per_row) return;
    const int m = threadIdx.x & 7;
    const int row = int(item / per_row), rem = int(item - (long long)row * per_row);
    int head = rem / J;
    const int j = rem - head * J, kind = head < kv ? 0 : 1;
    head -= kind * kv;
    const long long slot = __ldg(P.slots + row), page = slot >> P.c.page_shift;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    if (slot >= 0 && page < P.c.n_pages) {
        const int at = int(slot & (P.c.page() - 1));
        const float d = __half2float(P.c.sc[P.c.scale_row(page, head, at) + kind * J + j]);
        uint32_t n[4];
        if (kind == 0) {
            const uint8_t* src = P.c.k + P.c.k_row(page, head, at) + ((m >> 1) * J + j) * P.c.kb;
            if (P.c.kb == 4) {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(src) >> (8 * (m & 1));
                n[0] = w & 15u, n[1] = (w >> 16) & 15u, n[2] = (w >> 4) & 15u, n[3] = (w >> 20) & 15u;
            } else {
                const uint32_t w = *reinterpret_cast<const uint32_t*>(src + 4 * (m & 1));
                n[0] = w & 255u, n[1] = (w >> 16) & 255u, n[2] = (w >> 8) & 255u, n[3] = w >> 24;
            }
        } else {
            const uint8_t* src = P.c.v + P.c.v_pair(page, head, at >> 1) + (m * J + j) * P.c.vb + 2 * (at & 1);
            const uint32_t w = *reinterpret_cast<const uint16_t*>(src);
            if (P.c.vb == 4) {
                n[0] = w & 15u, n[1] = (w >> 4) & 15u, n[2] = (w >> 8) & 15u, n[3] = w >> 12;
            } else {
                const uint32_t u = *reinterpret_cast<const uint16_t*>(src + 4);
                n[0] = w & 255u, n[1] = w >> 8, n[2] = u & 255u, n[3] = u >> 8;
            }
        }
        const int off = (kind == 0 ? P.c.kb : P.c.vb) == 4 ? 8 : 128;
        o = make_float4(__fmul_rn(d, float(int(n[0]) - off)), __fmul_rn(d, float(int(n[1]) - off)),
                        __fmul_rn(d, float(int(n[2]) - off)), __fmul_rn(d, float(int(n[3]) - off)));
    } else if (slot >= 0 && P.status) {
        atomicOr(P.status, DEV_BAD_ADDRESS);
    }
    T* out = static_cast<T*>(kind == 0 ? P.k : P.v) + ((long long)row * kv + head) * P.c.dim + 32 * j + 4 * m;
    store4(out, o);
}

// blocks of 256 threads for rows x per_row groups of eight lanes; 0 if that passes a launch's grid
unsigned blocks_of(long long rows, long long per_row) {
    const long long b = (rows * per_row + 31) / 32;
    return b <= 0x7FFFFFFFLL ? unsigned(b) : 0u;
}

}  // namespace

extern "C" {

int qmv_kv_write(const qmv_kv_cache* cache, const void* k, const void* v, int dtype, long long k_stride,
                 long long v_stride, const long long* slots, long long rows, const float* cos_table,
                 const float* sin_table, const long long* positions, long long n_positions, int rot_dim, int paired,
                 const void* q, long long q_stride, int n_q, void* q_out, void* stream) {
    KvWriteParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!k || !v || !slots || (cos_table && (!sin_table || !positions)) || (q && !q_out)) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (rows < 0 || rows > 0x7FFFFFFFLL || (q && (n_q <= 0 || n_q > 65535))) return ST_BAD_TOKENS;
    const long long row = (long long)P.c.n_kv * P.c.dim;
    if (k_stride < row || v_stride < row || (q && q_stride < (long long)n_q * P.c.dim)) return ST_BAD_SHAPE;
    if (cos_table && (rot_dim < 8 || rot_dim > P.c.dim || rot_dim % 8 || n_positions <= 0)) return ST_BAD_SHAPE;
    const uintptr_t four = 4 * elem_bytes(dtype);             // rows are read four values at a time
    if (!aligned(k, four) || !aligned(v, four) || k_stride % 4 || v_stride % 4 || !aligned(slots, 8)) return ST_BAD_ALIGN;
    if (q && (!aligned(q, four) || !aligned(q_out, four) || q_stride % 4)) return ST_BAD_ALIGN;
    if (cos_table && (!aligned(cos_table, 16) || !aligned(sin_table, 16) || !aligned(positions, 8))) return ST_BAD_ALIGN;
    if (rows == 0) return ST_OK;
    P.k = k, P.v = v, P.q = q, P.q_out = q_out;
    P.k_stride = k_stride, P.v_stride = v_stride, P.q_stride = q_stride;
    P.slots = slots;
    P.cos_t = cos_table, P.sin_t = sin_table, P.pos = positions, P.n_pos = n_positions;
    P.rot = rot_dim, P.paired = paired, P.n_q = q ? n_q : 0;
    P.rows = int(rows);
    P.status = device_status_ptr();
    const unsigned blocks = blocks_of(rows, (long long)(2 * P.c.n_kv + P.n_q) * P.c.J);
    if (!blocks) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return launch_pdl(kv_write_kernel<decltype(c)::value>, dim3(blocks), dim3(256), static_cast<cudaStream_t>(stream), P);
    });
}

int qmv_kv_read(const qmv_kv_cache* cache, const long long* slots, long long rows, void* k, void* v, int dtype,
                void* stream) {
    KvReadParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!slots || !k || !v) return ST_NULL;
    if (dtype != QMV_OUT_F32 && dtype != QMV_OUT_BF16 && dtype != QMV_OUT_F16) return ST_BAD_SHAPE;
    if (rows < 0 || rows > 0x7FFFFFFFLL) return ST_BAD_TOKENS;
    if (!aligned(k, 16) || !aligned(v, 16) || !aligned(slots, 8)) return ST_BAD_ALIGN;
    if (rows == 0) return ST_OK;
    P.slots = slots, P.k = k, P.v = v;
    P.rows = int(rows);
    P.status = device_status_ptr();
    const unsigned blocks = blocks_of(rows, 2LL * P.c.n_kv * P.c.J);
    if (!blocks) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return launch_pdl(kv_read_kernel<decltype(c)::value>, dim3(blocks), dim3(256), static_cast<cudaStream_t>(stream), P);
    });
}

}  // extern "C"
