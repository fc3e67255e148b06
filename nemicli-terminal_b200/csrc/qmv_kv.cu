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
    const long long* pos;                 // [axes][rows]
    long long n_pos;
    int rot, paired, n_q;
    int n_axes;
    uint64_t axis_of[4];                  // the axis of each frequency, two bits
    int rows, parts, per_part;            // warps a row, passes a warp
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

// Eight lanes (m = 0..7) hold four values each of one 32-value block; the block's scale, and each lane's codes without
// offset, a byte each.  Q4_0: d = fp16(x / -8) of the value of largest magnitude (the first of equal ones), codes
// clamp(rint(x / d), -8, 7); Q8_0: d = fp16(max |x| / 127), codes clamp(rint(x / d), -127, 127).  The quotient is the IEEE one by
// the rounded d, the one the reader multiplies with.  It is formed as x (1 / d) first: that is within 2^-15 of it
// (|x / d| <= 128, the reciprocal's error and a rounding), so only where that lies within 2^-11 of a border between codes is the division made.
template <bool Q4>
__device__ __forceinline__ uint32_t quantise4(float4 x, __half& d) {
    float v[4] = {x.x, x.y, x.z, x.w};
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) odd |= !(fabsf(v[i]) <= kKvMax);
    if (__any_sync(0xffffffffu, odd)) {                           // NaN counts as 0
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = v[i] != v[i] ? 0.f : fminf(fmaxf(v[i], -kKvMax), kKvMax);
    }
    float top = fmaxf(fmaxf(fabsf(v[0]), fabsf(v[1])), fmaxf(fabsf(v[2]), fabsf(v[3])));
#pragma unroll
    for (int o = 1; o < 8; o *= 2) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if constexpr (Q4) {
        // the sign of the first value of that magnitude, from the first lane of the eight that has one
        const float first = fabsf(v[0]) == top ? v[0] : fabsf(v[1]) == top ? v[1] : fabsf(v[2]) == top ? v[2] : v[3];
        const int group = threadIdx.x & 24;
        const uint32_t has = __ballot_sync(0xffffffffu, fabsf(first) == top) >> group & 255u;
        const uint32_t minus = __ballot_sync(0xffffffffu, first < 0.f) >> group;
        const float m = minus >> (__ffs(has) - 1) & 1u ? -top : top;
        d = __float2half_rn(__fmul_rn(m, -0.125f));
    } else {
        d = __float2half_rn(__fdiv_rn(top, 127.0f));
    }
    const float df = __half2float(d);
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(df));
    if (df == 0.f) r = 0.f;
    constexpr float kRound = 12582912.f;                          // 1.5 2^23: added, the sum's low bits are rint(t)
    float t[4];
    bool near = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float p = v[i] * r;
        t[i] = __fadd_rn(p, kRound);
        near |= fabsf(__fsub_rn(p, __fsub_rn(t[i], kRound))) > 0.5f - 0.00048828125f;
    }
    if (__any_sync(0xffffffffu, near)) {
#pragma unroll
        for (int i = 0; i < 4; ++i) t[i] = __fadd_rn(df == 0.f ? 0.f : __fdiv_rn(v[i], df), kRound);
    }
    const float lo = kRound - (Q4 ? 8.f : 127.f), hi = kRound + (Q4 ? 7.f : 127.f);
    uint32_t n[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) n[i] = __float_as_uint(fminf(fmaxf(t[i], lo), hi));
    return __byte_perm(__byte_perm(n[0], n[1], 0x0040), __byte_perm(n[2], n[3], 0x0040), 0x5410);
}

// four values of a row as they lie in memory
template <int DT> struct Raw4 { using type = uint2; };
template <> struct Raw4<QMV_OUT_F32> { using type = uint4; };
__device__ __forceinline__ float4 raw4(uint4 w, float) { return make_float4(__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)); }
__device__ __forceinline__ float4 raw4(uint2 w, __nv_bfloat16) {
    return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xFFFF0000u));
}
__device__ __forceinline__ float4 raw4(uint2 w, __half) {
    const float2 a = __half22float2(*reinterpret_cast<const __half2*>(&w.x)), b = __half22float2(*reinterpret_cast<const __half2*>(&w.y));
    return make_float4(a.x, a.y, b.x, b.y);
}

// A warp takes some of one row's passes of 128 consecutive values (four blocks, eight lanes each): K's, V's, then those of the
// queries to rotate; kAhead passes' loads go out together.  Angles are the same for all of a lane's passes where a head
// has 2 or 4 blocks.  The formats are template choices (tested value by value they cost 12 of 58 us).  16381 bf16 tokens of 8
// key heads of 128 values: 46 us (50 in Q4_0), bound by the 142 instructions for four values a lane; with 32 query heads rotated
// along 88, where the queries' part moves at 6.4 TB/s.  Five or six CTAs an SM (fewer registers) instead of four: 88 and 94.
// A decode step is bound by its launch (64 tokens written 3.2 us, read 1.9, both 5.3, calls in a graph).
// AXES: a row has a position on each of up to four axes and every frequency its axis, so a frequency's angle lies in the axis's row of the
// tables, loaded value by value, once a row where a lane keeps its place in every head: 16381 rows with queries 90.9 us against 89.6.
template <int DT, int J, bool AXES>
__global__ void __launch_bounds__(256) kv_write_kernel(const __grid_constant__ KvWriteParams P) {
    using T = typename Elem<DT>::type;
    using W = typename Raw4<DT>::type;
    constexpr int D = 32 * J, kAhead = 4;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, m = lane & 7;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = int(id / P.parts), part = int(id - (long long)row * P.parts);
    if (row >= P.rows) return;                                    // whole warps
    const int kv = P.c.n_kv, n_kv = kv * D, n_q = P.n_q * D;      // values of a section
    const int pk = (n_kv + 127) / 128, pq = (n_q + 127) / 128;
    const int p1 = min(2 * pk + pq, (part + 1) * P.per_part);
    const long long slot = __ldg(P.slots + row), page = slot >> P.c.page_shift;
    const int at = int(slot & (P.c.page() - 1));
    bool bad = slot >= 0 && page >= P.c.n_pages, lost = false;    // not to be written; queries without a position
    const float* ct = nullptr;
    const float* st = nullptr;
    const int half = P.rot / 2;
    long long from[4] = {0, 0, 0, 0};                             // of each axis, its row of the tables
    if constexpr (AXES) {
        ct = P.cos_t, st = P.sin_t;
#pragma unroll
        for (int a = 0; a < 4; ++a) {
            if (a >= P.n_axes) continue;
            const long long p = __ldg(P.pos + (long long)a * P.rows + row);
            lost |= p < 0 || p >= P.n_pos;
            from[a] = p * half;
        }
        bad |= lost;
        if (lost) from[0] = from[1] = from[2] = from[3] = 0;
    } else if (P.cos_t) {
        const long long p = __ldg(P.pos + row);
        lost = p < 0 || p >= P.n_pos;
        bad |= lost;
        ct = P.cos_t + (lost ? 0 : p) * half;
        st = P.sin_t + (lost ? 0 : p) * half;
    }
    if (bad && lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    const bool write = slot >= 0 && !bad;
    auto place = [&](int f) {                                     // of frequency f, in the tables
        const int a = int(P.axis_of[f >> 5] >> (2 * (f & 31)) & 3);
        return (a == 0 ? from[0] : a == 1 ? from[1] : a == 2 ? from[2] : from[3]) + f;
    };
    auto angles = [&](int i0, float4& c, float4& s) {
        if constexpr (AXES) {
            const int f = P.paired ? i0 / 2 : i0 < half ? i0 : i0 - half;
            const long long f0 = place(f), f1 = place(f + 1);
            c.x = __ldg(ct + f0), s.x = __ldg(st + f0), c.y = __ldg(ct + f1), s.y = __ldg(st + f1);
            if (!P.paired) {
                const long long f2 = place(f + 2), f3 = place(f + 3);
                c.z = __ldg(ct + f2), s.z = __ldg(st + f2), c.w = __ldg(ct + f3), s.w = __ldg(st + f3);
            }
        } else if (P.paired) {
            const float2 cc = __ldg(reinterpret_cast<const float2*>(ct + i0 / 2)), ss = __ldg(reinterpret_cast<const float2*>(st + i0 / 2));
            c = make_float4(cc.x, cc.y, 0.f, 0.f), s = make_float4(ss.x, ss.y, 0.f, 0.f);
        } else {
            const int a = i0 < half ? i0 : i0 - half;
            c = load4(ct + a), s = load4(st + a);
        }
    };
    float4 c = make_float4(0.f, 0.f, 0.f, 0.f), s = c;
    constexpr bool kSame = 4 % J == 0;                            // this lane's place in every head
    const int own = (4 * lane) % D;
    if (kSame && ct && own < P.rot) angles(own, c, s);
    // bytes between heads of a page (a page's bytes fit 31 bits), and this row's places in head 0
    const uint32_t head_k = uint32_t(4 * J * P.c.kb) << P.c.page_shift, head_v = uint32_t(8 * J * P.c.vb) << (P.c.page_shift - 1),
                   head_s = uint32_t(2 * J) << P.c.page_shift;
    uint8_t* k_to = P.c.k + P.c.k_row(page, 0, at) + (m >> 1) * J * P.c.kb;
    uint8_t* v_to = P.c.v + P.c.v_pair(page, 0, at >> 1) + 2 * (at & 1) + m * J * P.c.vb;
    __half* s_to = P.c.sc + P.c.scale_row(page, 0, at);

    // passes first .. last of a section of n values at src; KIND 0: K, 1: V, 2: queries
    auto section = [&](auto kind_c, auto q4_c, const T* src, int n, int first, int last) {
        constexpr int KIND = decltype(kind_c)::value;
        constexpr bool q4 = decltype(q4_c)::value;
        const bool turn = KIND != 1 && ct != nullptr;
        auto batch = [&](int p0, auto count, bool check) {
            constexpr int A = decltype(count)::value;
            const T* at0 = src + 128 * p0 + 4 * lane;
            W w[A], o[A];
#pragma unroll
            for (int a = 0; a < A; ++a) {
                const int off = 128 * (p0 + a) + 4 * lane;
                w[a] = o[a] = W{};
                if (check && off >= n) continue;
                w[a] = __ldg(reinterpret_cast<const W*>(at0 + 128 * a));
                if (turn && !P.paired) {
                    const int i0 = kSame ? own : off % D;
                    if (i0 < P.rot) o[a] = __ldg(reinterpret_cast<const W*>(at0 + 128 * a + (i0 < half ? half : -half)));
                }
            }
#pragma unroll
            for (int a = 0; a < A; ++a) {
                const int off = 128 * (p0 + a) + 4 * lane, i0 = kSame ? own : off % D;
                const bool live = !check || off < n;
                float4 x = raw4(w[a], T{});
                if (turn && i0 < P.rot) {
                    if (!kSame) angles(i0, c, s);
                    x = rotated(x, raw4(o[a], T{}), c, s, P.paired, i0 < half);
                }
                if constexpr (KIND == 2) {
                    if (live) store4(static_cast<T*>(P.q_out) + (long long)row * n + off, lost ? make_float4(0.f, 0.f, 0.f, 0.f) : x);
                } else {
                    __half d;
                    uint32_t b = quantise4<q4>(x, d);
                    b = q4 ? (b & 0x0F0F0F0Fu) ^ 0x08080808u : b ^ 0x80808080u;
                    const uint32_t head = uint32_t(off) / D, j = (uint32_t(off) - head * D) / 32;
                    if constexpr (KIND == 0) {
                        // lanes 2 t and 2 t + 1 share the 8 values of t
                        uint32_t word = q4 ? __byte_perm(b, 0u, 0x4140) | __byte_perm(b, 0u, 0x4342) << 4 : __byte_perm(b, 0u, 0x3120);
                        if (q4 && (m & 1)) word <<= 8;
                        const uint32_t both = word | __shfl_xor_sync(0xffffffffu, word, 1);
                        if (!live || !write) continue;
                        uint8_t* dst = k_to + (head * head_k + j * P.c.kb);
                        if (!q4) *reinterpret_cast<uint32_t*>(dst + 4 * (m & 1)) = word;
                        else if (!(m & 1)) *reinterpret_cast<uint32_t*>(dst) = both;
                    } else {
                        if (!live || !write) continue;
                        uint8_t* dst = v_to + (head * head_v + j * P.c.vb);
                        if (q4) {
                            *reinterpret_cast<uint16_t*>(dst) = uint16_t(__byte_perm(b | b >> 4, 0u, 0x4420));
                        } else {
                            *reinterpret_cast<uint16_t*>(dst) = uint16_t(b);
                            *reinterpret_cast<uint16_t*>(dst + 4) = uint16_t(b >> 16);
                        }
                    }
                    if (m == 0) s_to[head * head_s + KIND * J + j] = d;
                }
            }
        };
        int p = first;
        for (; p + kAhead <= last && 128 * (p + kAhead) <= n; p += kAhead) batch(p, std::integral_constant<int, kAhead>{}, false);
        for (; p < last; ++p) batch(p, std::integral_constant<int, 1>{}, true);
    };
    const int q0 = part * P.per_part;
    auto by_format = [&](auto kind_c, int bytes, const T* src, int first, int last) {
        if (bytes == 4) section(kind_c, std::true_type{}, src, n_kv, first, last);
        else section(kind_c, std::false_type{}, src, n_kv, first, last);
    };
    if (q0 < pk) by_format(std::integral_constant<int, 0>{}, P.c.kb, static_cast<const T*>(P.k) + row * P.k_stride, q0, min(p1, pk));
    if (q0 < 2 * pk && p1 > pk)
        by_format(std::integral_constant<int, 1>{}, P.c.vb, static_cast<const T*>(P.v) + row * P.v_stride, max(q0 - pk, 0), min(p1 - pk, pk));
    if (p1 > 2 * pk)
        section(std::integral_constant<int, 2>{}, std::false_type{}, static_cast<const T*>(P.q) + row * P.q_stride, n_q, max(q0 - 2 * pk, 0), p1 - 2 * pk);
}

struct KvReadParams {
    KvView c;
    const long long* slots;
    void* k;
    void* v;
    int rows, parts, per_part;
    int* status;
};

// The inverse of kv_write_kernel's stores, a warp some of one row's passes: d * code, one rounded product each.  16381
// tokens as above to bf16: 21 us (4.4 TB/s of codes read and values written).
template <int DT, int J>
__global__ void __launch_bounds__(256) kv_read_kernel(const __grid_constant__ KvReadParams P) {
    using T = typename Elem<DT>::type;
    constexpr int D = 32 * J, kAhead = 8;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int lane = threadIdx.x & 31, m = lane & 7;
    const long long id = (long long)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int row = int(id / P.parts), part = int(id - (long long)row * P.parts);
    if (row >= P.rows) return;
    const int n_kv = P.c.n_kv * D, pk = (n_kv + 127) / 128, p1 = min(2 * pk, (part + 1) * P.per_part);
    const long long slot = __ldg(P.slots + row), page = slot >> P.c.page_shift;
    const int at = int(slot & (P.c.page() - 1));
    const bool there = slot >= 0 && page < P.c.n_pages;
    if (slot >= 0 && !there && lane == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    const uint32_t head_k = uint32_t(4 * J * P.c.kb) << P.c.page_shift, head_v = uint32_t(8 * J * P.c.vb) << (P.c.page_shift - 1),
                   head_s = uint32_t(2 * J) << P.c.page_shift;
    const uint8_t* k = P.c.k + P.c.k_row(page, 0, at) + (m >> 1) * J * P.c.kb;
    const uint8_t* v = P.c.v + P.c.v_pair(page, 0, at >> 1) + 2 * (at & 1) + m * J * P.c.vb;
    const __half* sc = P.c.sc + P.c.scale_row(page, 0, at);
    auto section = [&](auto kind_c, auto q4_c, int first, int last) {
        constexpr int KIND = decltype(kind_c)::value;
        constexpr bool q4 = decltype(q4_c)::value;
        T* out = static_cast<T*>(KIND == 0 ? P.k : P.v) + (long long)row * n_kv;
        auto batch = [&](int p0, auto count, bool check) {
            constexpr int A = decltype(count)::value;
            uint32_t w[A];
            __half d[A];
#pragma unroll
            for (int a = 0; a < A; ++a) {
                const uint32_t off = 128 * (p0 + a) + 4 * lane, head = off / D, j = (off - head * D) / 32;
                w[a] = 0u, d[a] = __ushort_as_half(0);
                if (!there || (check && int(off) >= n_kv)) continue;
                d[a] = sc[head * head_s + KIND * J + j];
                if constexpr (KIND == 0) {
                    const uint8_t* src = k + (head * head_k + j * P.c.kb);
                    w[a] = q4 ? *reinterpret_cast<const uint32_t*>(src) >> (8 * (m & 1)) : *reinterpret_cast<const uint32_t*>(src + 4 * (m & 1));
                } else {
                    const uint8_t* src = v + (head * head_v + j * P.c.vb);
                    w[a] = *reinterpret_cast<const uint16_t*>(src);
                    if (!q4) w[a] |= uint32_t(*reinterpret_cast<const uint16_t*>(src + 4)) << 16;
                }
            }
#pragma unroll
            for (int a = 0; a < A; ++a) {
                const int off = 128 * (p0 + a) + 4 * lane;
                if (check && off >= n_kv) continue;
                // the four codes as bytes, in order
                uint32_t n = w[a];
                if (q4) n = KIND == 0 ? (n & 0x000F000Fu) | (n & 0x00F000F0u) << 4 : (n & 0x000Fu) | (n & 0x00F0u) << 4 | (n & 0x0F00u) << 8 | (n & 0xF000u) << 12;
                if (KIND == 0) n = __byte_perm(n, 0u, 0x3120);
                const float f = there ? __half2float(d[a]) : 0.f;
                float y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = there ? __fmul_rn(f, float(int(n >> (8 * i) & 255u) - (q4 ? 8 : 128))) : 0.f;
                store4_held(out + off, make_float4(y[0], y[1], y[2], y[3]));
            }
        };
        int p = first;
        for (; p + kAhead <= last && 128 * (p + kAhead) <= n_kv; p += kAhead) batch(p, std::integral_constant<int, kAhead>{}, false);
        for (; p < last; ++p) batch(p, std::integral_constant<int, 1>{}, true);
    };
    const int q0 = part * P.per_part;
    auto by_format = [&](auto kind_c, int bytes, int first, int last) {
        if (bytes == 4) section(kind_c, std::true_type{}, first, last);
        else section(kind_c, std::false_type{}, first, last);
    };
    if (q0 < pk) by_format(std::integral_constant<int, 0>{}, P.c.kb, q0, min(p1, pk));
    if (p1 > pk) by_format(std::integral_constant<int, 1>{}, P.c.vb, max(q0 - pk, 0), p1 - pk);
}

// Warps a row and passes a warp: rows on their own where they fill the GPU (32 warps an SM), else cut so that there are as
// many, one pass each at least (512 bf16 rows of 8 key heads of 128 with 32 query heads, calls in a graph: 7.7 us, uncut 12.4, for 16 warps an SM
// 8.4, for 64 8.1; 64 rows: 3.2, uncut 12.2); the launch's CTAs, 0 if they pass a grid.
unsigned cut_rows(long long rows, int passes, int& parts, int& per_part) {
    const long long want = 32LL * sm_count();
    parts = int(std::min<long long>(passes, std::max<long long>(1, want / rows)));
    per_part = (passes + parts - 1) / parts;
    parts = (passes + per_part - 1) / per_part;
    const long long ctas = (rows * parts + 7) / 8;
    return ctas <= 0x7FFFFFFFLL ? unsigned(ctas) : 0u;
}
int passes_of(int heads, int dim) { return (heads * dim + 127) / 128; }
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

int write_rows(const qmv_kv_cache* cache, const void* k, const void* v, int dtype, long long k_stride, long long v_stride,
               const long long* slots, long long rows, const float* cos_table, const float* sin_table, const long long* positions,
               long long n_positions, int rot_dim, int paired, const uint8_t* axes, int n_axes, const void* q, long long q_stride,
               int n_q, void* q_out, void* stream) {
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
    for (int f = 0; axes && f < rot_dim / 2; ++f) {
        if (axes[f] >= n_axes) return ST_BAD_SHAPE;
        P.axis_of[f >> 5] |= uint64_t(axes[f]) << (2 * (f & 31));
    }
    if (rows == 0) return ST_OK;
    P.n_axes = n_axes;
    P.k = k, P.v = v, P.q = q, P.q_out = q_out;
    P.k_stride = k_stride, P.v_stride = v_stride, P.q_stride = q_stride;
    P.slots = slots;
    P.cos_t = cos_table, P.sin_t = sin_table, P.pos = positions, P.n_pos = n_positions;
    P.rot = rot_dim, P.paired = paired, P.n_q = q ? n_q : 0;
    P.rows = int(rows);
    P.status = device_status_ptr();
    const unsigned ctas = cut_rows(rows, 2 * passes_of(P.c.n_kv, P.c.dim) + passes_of(P.n_q, P.c.dim), P.parts, P.per_part);
    if (!ctas) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return by_blocks(P.c.J, [&](auto j) {
            constexpr int DT = decltype(c)::value, J = decltype(j)::value;
            return axes ? launch_pdl(kv_write_kernel<DT, J, true>, dim3(ctas), dim3(256), static_cast<cudaStream_t>(stream), P)
                        : launch_pdl(kv_write_kernel<DT, J, false>, dim3(ctas), dim3(256), static_cast<cudaStream_t>(stream), P);
        });
    });
}

struct KvCopyParams {
    KvView c;
    const int* src;
    const int* dst;
    const int* used;                      // tokens of each copy (null: whole pages)
    int n;
    int* status;
};

// A CTA a copy and key head: the first tokens' K rows, V pairs and scales, each one run of bytes.
__global__ void __launch_bounds__(128) kv_copy_kernel(const __grid_constant__ KvCopyParams P) {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const int i = blockIdx.x / P.c.n_kv, head = blockIdx.x - i * P.c.n_kv, tid = threadIdx.x;
    const int from = __ldg(P.src + i), to = __ldg(P.dst + i);
    if (from < 0 || to < 0) return;
    const int page = P.c.page(), asked = P.used ? __ldg(P.used + i) : page, used = min(max(asked, 0), page);
    const bool bad = from >= P.c.n_pages || to >= P.c.n_pages;
    if ((bad || used != asked) && tid == 0 && head == 0 && P.status) atomicOr(P.status, DEV_BAD_ADDRESS);
    if (bad) return;
    // pieces of 16 bytes of K, V and scales in one list, the last words of the scales by themselves: two pieces of a thread in flight
    uint8_t* sc = reinterpret_cast<uint8_t*>(P.c.sc);
    const int n_k = used * 4 * P.c.J * P.c.kb / 16, n_v = (used + 1) / 2 * 8 * P.c.J * P.c.vb / 16, words = used * P.c.J, n_s = words / 4;
    const uint8_t* src[3] = {P.c.k + P.c.k_row(from, head, 0), P.c.v + P.c.v_pair(from, head, 0), sc + 2 * P.c.scale_row(from, head, 0)};
    uint8_t* dst[3] = {P.c.k + P.c.k_row(to, head, 0), P.c.v + P.c.v_pair(to, head, 0), sc + 2 * P.c.scale_row(to, head, 0)};
    if (tid < words % 4) reinterpret_cast<uint32_t*>(dst[2])[4 * n_s + tid] = reinterpret_cast<const uint32_t*>(src[2])[4 * n_s + tid];
    const int all = n_k + n_v + n_s;
#pragma unroll 4
    for (int x = tid; x < all; x += 128) {
        const int y = x < n_k ? x : x < n_k + n_v ? x - n_k : x - n_k - n_v;
        const uint8_t* f = x < n_k ? src[0] : x < n_k + n_v ? src[1] : src[2];
        uint8_t* t = x < n_k ? dst[0] : x < n_k + n_v ? dst[1] : dst[2];
        reinterpret_cast<uint4*>(t)[y] = __ldcg(reinterpret_cast<const uint4*>(f) + y);
    }
}

}  // namespace

extern "C" {

int qmv_kv_write(const qmv_kv_cache* cache, const void* k, const void* v, int dtype, long long k_stride,
                 long long v_stride, const long long* slots, long long rows, const float* cos_table,
                 const float* sin_table, const long long* positions, long long n_positions, int rot_dim, int paired,
                 const void* q, long long q_stride, int n_q, void* q_out, void* stream) {
    return write_rows(cache, k, v, dtype, k_stride, v_stride, slots, rows, cos_table, sin_table, positions, n_positions, rot_dim, paired,
                      nullptr, 0, q, q_stride, n_q, q_out, stream);
}

int qmv_kv_write_axes(const qmv_kv_cache* cache, const void* k, const void* v, int dtype, long long k_stride, long long v_stride,
                      const long long* slots, long long rows, const float* cos_table, const float* sin_table, const long long* positions,
                      long long n_positions, int rot_dim, int paired, const uint8_t* axes, int n_axes, const void* q, long long q_stride,
                      int n_q, void* q_out, void* stream) {
    if (!cos_table || !axes) return ST_NULL;
    if (n_axes < 1 || n_axes > 4) return ST_BAD_SHAPE;
    return write_rows(cache, k, v, dtype, k_stride, v_stride, slots, rows, cos_table, sin_table, positions, n_positions, rot_dim, paired,
                      axes, n_axes, q, q_stride, n_q, q_out, stream);
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
    const unsigned ctas = cut_rows(rows, 2 * passes_of(P.c.n_kv, P.c.dim), P.parts, P.per_part);
    if (!ctas) return ST_BAD_TOKENS;
    return by_elem(dtype, [&](auto c) {
        return by_blocks(P.c.J, [&](auto j) {
            return launch_pdl(kv_read_kernel<decltype(c)::value, decltype(j)::value>, dim3(ctas), dim3(256), static_cast<cudaStream_t>(stream), P);
        });
    });
}

int qmv_kv_copy(const qmv_kv_cache* cache, const int* src, const int* dst, const int* used, int n, void* stream) {
    KvCopyParams P{};
    const int st = kv_view(cache, P.c);
    if (st) return st;
    if (!src || !dst) return ST_NULL;
    if (n < 0 || (long long)n * P.c.n_kv > 0x7FFFFFFFLL) return ST_BAD_TOKENS;
    if (!aligned(src, 4) || !aligned(dst, 4) || !aligned(used, 4)) return ST_BAD_ALIGN;
    if (n == 0) return ST_OK;
    P.src = src, P.dst = dst, P.used = used, P.n = n;
    P.status = device_status_ptr();
    return launch_pdl(kv_copy_kernel, dim3(unsigned(n * P.c.n_kv)), dim3(128), static_cast<cudaStream_t>(stream), P);
}

}  // extern "C"
