// Writing a quantised key / value cache and reading it back (layout: qmv_kv.cuh; C-ABI declarations:
// include/nemicli_qmv.h).
#include <algorithm>
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
    int rows, parts, per_part;            // warps a row, blocks a warp (a multiple of 4)
    int* status;
};

// Four consecutive values x of a head, rotated: value i < rot pairs with i + rot / 2 (o: the partners, cos and sin of the
// angles), or, paired, 2 i with 2 i + 1 (cos.x, cos.y: of the two pairs).  y1 = x1 c - x2 s, y2 = x2 c + x1 s; every product
// and sum is rounded on its own (no fused multiply-add), so the codes follow from the inputs bit for bit.
__device__ __forceinline__ float4 rotated(float4 x, float4 o, float4 c, float4 s, bool paired, bool first) {
    if (paired)
        return make_float4(__fsub_rn(__fmul_rn(x.x, c.x), __fmul_rn(x.y, s.x)), __fadd_rn(__fmul_rn(x.y, c.x), __fmul_rn(x.x, s.x)),
                           __fsub_rn(__fmul_rn(x.z, c.y), __fmul_rn(x.w, s.y)), __fadd_rn(__fmul_rn(x.w, c.y), __fmul_rn(x.z, s.y)));
    if (first) s = make_float4(-s.x, -s.y, -s.z, -s.w);           // a - b s = a + b (-s), exactly
    return make_float4(__fadd_rn(__fmul_rn(x.x, c.x), __fmul_rn(o.x, s.x)), __fadd_rn(__fmul_rn(x.y, c.y), __fmul_rn(o.y, s.y)),
                       __fadd_rn(__fmul_rn(x.z, c.z), __fmul_rn(o.z, s.z)), __fadd_rn(__fmul_rn(x.w, c.w), __fmul_rn(o.w, s.w)));
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

// A warp takes some of one row's 32-value blocks (K heads, then V heads, then the queries to rotate), four at a time on eight
// lanes each, and kAhead such passes' loads go out together.  Rows' angles are the same for all of a lane's passes where
// a head has 2 or 4 blocks.  Bound by memory for long prompts (divisions and reductions are about as many clocks), by its
// launch for a decode step.
template <int DT, int J>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvWriteParams P) {
    using T = typename Elem<DT>::type;
    constexpr int kAhead = 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int kv = P.c.n_kv, blocks = (2 * kv + P.n_q) * J;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = int(id / P.parts), part = int(id - (long long)row * P.parts);
    if (row >= P.rows) return;                                    // whole warps
    const int lane = threadIdx.x & 31, m = lane & 7;
    const int b1 = min(blocks, (part + 1) * P.per_part);
    const long long slot = __ldg(P.slots + row), page = slot >> P.c.page_shift;
    const int at = int(slot & (P.c.page() - 1));
    bool bad = slot >= 0 && page >= P.c.n_pages, lost = false;    // not to be written; queries without a position
    const float* ct = nullptr;
    const float* st = nullptr;
    const int half = P.rot / 2;
    if (P.cos_t) {
        const long long p = __ldg(P.pos + row);
        lost = p < 0 || p >= P.n_pos;
        bad |= lost;
        ct = P.cos_t + (lost ? 0 : p) * half;
        st = P.sin_t + (lost ? 0 : p) * half;
    }
    if (bad && lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    const bool write = slot >= 0 && !bad;
    auto angles = [&](int i0, float4& c, float4& s) {
        if (P.paired) {
            const float2 cc = __ldg(reinterpret_cast<const float2*>(ct + i0 / 2)), ss = __ldg(reinterpret_cast<const float2*>(st + i0 / 2));
            c = make_float4(cc.x, cc.y, 0.f, 0.f), s = make_float4(ss.x, ss.y, 0.f, 0.f);
        } else {
            const int a = i0 < half ? i0 : i0 - half;
            c = load4(ct + a), s = load4(st + a);
        }
    };
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), s = c;
    const int own = 32 * ((lane >> 3) % J) + 4 * m;               // 4 % J == 0: this lane's values of every head
    if (4 % J == 0 && ct && own < P.rot) angles(own, c, s);
    for (int b0 = part * P.per_part; b0 < b1; b0 += 4 * kAhead) {
        float4 x[kAhead], o[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int blk = b0 + 4 * q + (lane >> 3), h = blk / J, i0 = 32 * (blk - h * J) + 4 * m;
            x[q] = o[q] = make_float4(0.f, 0.f, 0.f, 0.f);
            if (blk < b1) {
                const T* src = h < kv ? static_cast<const T*>(P.k) + row * P.k_stride + h * (32 * J)
                             : h < 2 * kv ? static_cast<const T*>(P.v) + row * P.v_stride + (h - kv) * (32 * J)
                                          : static_cast<const T*>(P.q) + row * P.q_stride + (h - 2 * kv) * (32 * J);
                x[q] = load4(src + i0);
                if (ct && !P.paired && i0 < P.rot && (h < kv || h >= 2 * kv)) o[q] = load4(src + (i0 < half ? i0 + half : i0 - half));
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int blk = b0 + 4 * q + (lane >> 3), h = blk / J, j = blk - h * J, i0 = 32 * j + 4 * m;
            if (b0 + 4 * q >= b1) break;                          // whole warps
            const int kind = h < kv ? 0 : h < 2 * kv ? 1 : 2, head = h - kind * kv;
            if (ct && kind != 1 && i0 < P.rot) {
                if (4 % J != 0) angles(i0, c, s);
                x[q] = rotated(x[q], o[q], c, s, P.paired, i0 < half);
            }
            const bool live = blk < b1;
            if (kind == 2 && live)
                store4(static_cast<T*>(P.q_out) + ((long long)row * P.n_q + head) * (32 * J) + i0, lost ? make_float4(0.f, 0.f, 0.f, 0.f) : x[q]);
            if (!__any_sync(0xffffffffu, kind != 2 && live)) continue;
            const bool q4 = (kind == 1 ? P.c.vb : P.c.kb) == 4;
            __half d;
            const uint4 n = quantise4(x[q], q4, d);
            // K: lanes 2 t and 2 t + 1 share the 8 values of t
            uint32_t word = q4 ? n.x | (n.y << 16) | (n.z << 4) | (n.w << 20) : n.x | (n.y << 16) | (n.z << 8) | (n.w << 24);
            if (q4 && (m & 1)) word <<= 8;
            const uint32_t both = word | __shfl_xor_sync(0xffffffffu, word, 1);
            if (kind == 2 || !live || !write) continue;
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
    }
}

struct KvReadParams {
    KvView c;
    const long long* slots;
    void* k;
    void* v;
    int rows, parts, per_part;
    int* status;
};

// The inverse of kv_write_kernel's stores, a warp some of one row's blocks: d * code, one rounded product each.
template <int DT, int J>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadParams P) {
    using T = typename Elem<DT>::type;
    constexpr int kAhead = 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int kv = P.c.n_kv, blocks = 2 * kv * J;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = int(id / P.parts), part = int(id - (long long)row * P.parts);
    if (row >= P.rows) return;
    const int lane = threadIdx.x & 31, m = lane & 7, b1 = min(blocks, (part + 1) * P.per_part);
    const long long slot = __ldg(P.slots + row), page = slot >> P.c.page_shift;
    const int at = int(slot & (P.c.page() - 1));
    const bool there = slot >= 0 && page < P.c.n_pages;
    if (slot >= 0 && !there && lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    for (int b0 = part * P.per_part; b0 < b1; b0 += 4 * kAhead) {
        uint32_t w[kAhead], u[kAhead];
        float d[kAhead];
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int blk = b0 + 4 * q + (lane >> 3), h = blk / J, j = blk - h * J, kind = h < kv ? 0 : 1, head = h - kind * kv;
            w[q] = u[q] = 0u, d[q] = 0.f;
            if (!there || blk >= b1) continue;
            d[q] = __half2float(P.c.sc[P.c.scale_row(page, head, at) + kind * J + j]);
            if (kind == 0) {
                const uint8_t* src = P.c.k + P.c.k_row(page, head, at) + ((m >> 1) * J + j) * P.c.kb;
                w[q] = P.c.kb == 4 ? *reinterpret_cast<const uint32_t*>(src) >> (8 * (m & 1)) : *reinterpret_cast<const uint32_t*>(src + 4 * (m & 1));
            } else {
                const uint8_t* src = P.c.v + P.c.v_pair(page, head, at >> 1) + (m * J + j) * P.c.vb + 2 * (at & 1);
                w[q] = *reinterpret_cast<const uint16_t*>(src);
                if (P.c.vb == 8) u[q] = *reinterpret_cast<const uint16_t*>(src + 4);
            }
        }
#pragma unroll
        for (int q = 0; q < kAhead; ++q) {
            const int blk = b0 + 4 * q + (lane >> 3), h = blk / J, j = blk - h * J, kind = h < kv ? 0 : 1, head = h - kind * kv;
            if (blk >= b1) continue;
            uint32_t n[4];
            const bool q4 = (kind == 0 ? P.c.kb : P.c.vb) == 4;
            if (kind == 0) {
                const int a = q4 ? 4 : 8, mask = q4 ? 15 : 255;
                n[0] = w[q] & mask, n[1] = (w[q] >> 16) & mask, n[2] = (w[q] >> a) & mask, n[3] = (w[q] >> (16 + a)) & mask;
            } else if (q4) {
                n[0] = w[q] & 15u, n[1] = (w[q] >> 4) & 15u, n[2] = (w[q] >> 8) & 15u, n[3] = w[q] >> 12;
            } else {
                n[0] = w[q] & 255u, n[1] = w[q] >> 8, n[2] = u[q] & 255u, n[3] = u[q] >> 8;
            }
            const int off = q4 ? 8 : 128;
            const float4 y = !there ? make_float4(0.f, 0.f, 0.f, 0.f)
                                    : make_float4(__fmul_rn(d[q], float(int(n[0]) - off)), __fmul_rn(d[q], float(int(n[1]) - off)),
                                                  __fmul_rn(d[q], float(int(n[2]) - off)), __fmul_rn(d[q], float(int(n[3]) - off)));
            store4(static_cast<T*>(kind == 0 ? P.k : P.v) + ((long long)row * kv + head) * (32 * J) + 32 * j + 4 * m, y);
        }
    }
}

// Warps a row and blocks a warp: rows on their own where they fill the GPU (16 warps an SM), else cut so that there are as
// many, at least one pass of 4 blocks each; the launch's CTAs, 0 if they pass a grid.
unsigned cut_rows(long long rows, int blocks, int& parts, int& per_part) {
    const long long want = 16LL * sm_count();
    const int passes = (blocks + 3) / 4;
    parts = int(std::min<long long>(passes, std::max<long long>(1, want / rows)));
    per_part = 4 * ((passes + parts - 1) / parts);
    parts = (blocks + per_part - 1) / per_part;
    const long long ctas = (rows * parts + 7) / 8;
    return ctas <= 0x7FFFFFFFLL ? unsigned(ctas) : 0u;
}
// f(std::integral_constant<int, dim / 32>)
template <class Fn>
int by_blocks(int J, Fn&& f) {
    switch (J) {
    case 2: return f(std::integral_constant<int, 2>{});
    case 3: return f(std::integral_constant<int, 3>{});
    case 4: return f(std::integral_constant<int, 4>{});
    case 8: return f(std::integral_constant<int, 8>{});
    }
    return ST_BAD_SHAPE;
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
    const unsigned ctas = cut_rows(rows, (2 * P.c.n_kv + P.n_q) * P.c.J, P.parts, P.per_part);
    if (!ctas) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return by_blocks(P.c.J, [&](auto j) {
            return launch_pdl(kv_write_kernel<decltype(c)::value, decltype(j)::value>, dim3(ctas), dim3(256), static_cast<cudaStream_t>(stream), P);
        });
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
    const unsigned ctas = cut_rows(rows, 2 * P.c.n_kv * P.c.J, P.parts, P.per_part);
    if (!ctas) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return by_blocks(P.c.J, [&](auto j) {
            return launch_pdl(kv_read_kernel<decltype(c)::value, decltype(j)::value>, dim3(ctas), dim3(256), static_cast<cudaStream_t>(stream), P);
        });
    });
}

}  // extern "C"
