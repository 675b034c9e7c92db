// What the quantized products on the matrix cores share (gemm.hip, moe_rows.hip): x as two fp16 parts, a lane's share
// of a weight block, and its decode to fp16 operands. The mathematics stands at the head of gemm.hip.
#pragma once

#include <cfloat>
#include <type_traits>
#include <utility>

#include "device_common.hpp"
#include "ggml_common.hpp"

namespace qk {
namespace {

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float wave_max_abs(float v) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}

__device__ __forceinline__ uint32_t half_bits_of(float v) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(v));
}

// Exponent slot of a token row holding an infinity: the fp16 split cannot carry
// it (h = inf, l = inf - inf = NaN would turn the whole output row into NaN),
// so the GEMM evaluates that row's outputs per element instead.
constexpr int kRowNonFinite = 0x7fffffff;

// e for a row whose largest |x| is m (NaN is ignored by the max; a NaN row's
// outputs are NaN either way): zero rows unscaled, rows with an infinity marked.
__device__ __forceinline__ int prep_exponent(float m) {
    if (!(m <= FLT_MAX)) return kRowNonFinite;
    int e = 0;
    if (m > 0.f) {
        int em;
        frexpf(m, &em);   // m in [2^(em-1), 2^em)
        e = 15 - em;
    }
    return e;
}

// y for (token row x, weight row at element `base`) when x holds an infinity:
// the reference's per-element fp32 products and sum (src/cuda/matmul_q4.cu:
// 140-167), so inf * w, 0 * inf = NaN and +inf + -inf = NaN give the same
// pattern of infinities and NaNs as its GEMV.
__device__ float row_dot_per_element(const uint8_t* __restrict__ w, int type, uint64_t base,
                                     const float* __restrict__ x, int K) {
    float s = 0.f;
    for (int k = 0; k < K; ++k) s = __builtin_fmaf(dequant_elem(w, type, base + k), x[k], s);
    return s;
}

__device__ __forceinline__ float max_abs4(float m, const float4& v) {
    return fmaxf(m, fmaxf(fmaxf(fabsf(v.x), fabsf(v.y)), fmaxf(fabsf(v.z), fabsf(v.w))));
}

// The fp16 parts of 8 values times 2^e, in the operand's order (packed pairs), and the sum of the scaled values.
__device__ __forceinline__ float split8(const float4& a, const float4& b, int e, uint32_t (&hi)[4], uint32_t (&lo)[4]) {
    const float f[8] = {ldexpf(a.x, e), ldexpf(a.y, e), ldexpf(a.z, e), ldexpf(a.w, e),
                        ldexpf(b.x, e), ldexpf(b.y, e), ldexpf(b.z, e), ldexpf(b.w, e)};
    uint32_t h[8], l[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const _Float16 hh = static_cast<_Float16>(f[i]);
        h[i] = __builtin_bit_cast(uint16_t, hh);
        l[i] = half_bits_of(f[i] - static_cast<float>(hh));
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int k = 4 * (i >> 1) + (i & 1);
        hi[i] = h[k] | (h[k + 2] << 16);
        lo[i] = l[k] | (l[k + 2] << 16);
    }
    return ((f[0] + f[1]) + (f[2] + f[3])) + ((f[4] + f[5]) + (f[6] + f[7]));
}

__device__ __forceinline__ f16x2_t h2(uint32_t w) { return __builtin_bit_cast(f16x2_t, w); }
__device__ __forceinline__ uint32_t w2(f16x2_t h) { return __builtin_bit_cast(uint32_t, h); }
__device__ __forceinline__ f16x2_t fma2(f16x2_t a, f16x2_t b, f16x2_t c) { return __builtin_elementwise_fma(a, b, c); }
__device__ __forceinline__ f16x2_t dup2(float v) {
    const _Float16 h = static_cast<_Float16>(v);
    return f16x2_t{h, h};
}

// 16 bytes at a 2-byte aligned address (gfx950 global loads take any byte
// alignment; Q6_K blocks are 210 bytes).
__device__ __forceinline__ uint4 ldg16_a2(const uint8_t* p) {
    uint4 v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 2), 16);
    return v;
}
__device__ __forceinline__ uint2 ldg8_a2(const uint8_t* p) {
    uint2 v;
    __builtin_memcpy(&v, __builtin_assume_aligned(p, 2), 8);
    return v;
}

// A lane's share of one block of its weight row (the mapping above). Q4_K, element i of a block
// (src/cuda/matmul_q4.cu:76-96): qs byte 16 + 32 (i / 64) + i % 32, low nibble if i % 64 < 32, scale i / 32:
// q[g] holds the bytes of depths u = 2 g, 2 g + 1 (both nibbles), hd the 16-byte header. Q6_K
// (src/cuda/matmul_q4.cu:105-126): ql byte 64 (i / 128) + 32 ((i % 128) / 32 & 1) + i % 32, low nibble in quarters
// 0, 1 of a half, qh byte 128 + 32 (i / 128) + i % 32 bits 2 quarter, scale byte 192 + i / 16, d at 208: q[0], q[1]
// the ql bytes of even and odd u, qh, the half's 8 scales and d.
template <int TYPE>
struct WBlock;
template <>
struct WBlock<kQ4_K> {
    uint4 q[2], hd;
    __device__ __forceinline__ void load(const uint8_t* base, uint32_t row, int lk) {
        const uint32_t o = row + 16u + 64u * (lk >> 1) + 16u * (lk & 1);
        hd = ld16(base + row);
        q[0] = ld16(base + o);
        q[1] = ld16(base + (o + 32u));
    }
};
template <>
struct WBlock<kQ6_K> {
    uint4 q[2], qh;
    uint2 sc;
    uint16_t d;
    __device__ __forceinline__ void load(const uint8_t* base, uint32_t row, int lk) {
        const uint32_t h = lk >> 1, l = lk & 1, o = row + 64u * h + 16u * l;
        q[0] = ldg16_a2(base + o);
        q[1] = ldg16_a2(base + (o + 32u));
        qh = ldg16_a2(base + (row + 128u + 32u * h + 16u * l));
        sc = ldg8_a2(base + (row + 192u + 8u * h));
        d = *reinterpret_cast<const uint16_t*>(base + (row + 208u));
    }
};

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) { return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w; }

// Scale of depth u of the lane's half-block, as the fp16 operands need it.
template <int TYPE>
struct WScale;
template <>
struct WScale<kQ4_K> {
    f16x2_t s, c;   // q sc = fma(1024 + q, sc, -1024 sc); high nibbles fma(1024 + 16 q, sc / 16, -64 sc): exact
    template <int U>
    __device__ __forceinline__ void set(const WBlock<kQ4_K>& b, int lk) {
        // scale_min_k4 (src/cuda/matmul_q4.cu:18-26): group 4 (lk / 2) + U
        const uint32_t lo = (b.hd.y >> (8 * U)) & 63u;
        const uint32_t hi = ((b.hd.w >> (8 * U)) & 15u) | ((b.hd.y >> (8 * U + 2)) & 0x30u);
        from<U>((lk & 2) ? hi : lo);
    }
    // (q - 8) sc = fma(16 + q, sc, -24 sc), exact
    template <int U>
    __device__ __forceinline__ void set_centred(const WBlock<kQ4_K>& b, int lk) {
        const uint32_t lo = (b.hd.y >> (8 * U)) & 63u;
        const uint32_t hi = ((b.hd.w >> (8 * U)) & 15u) | ((b.hd.y >> (8 * U + 2)) & 0x30u);
        s = h2(((lk & 2) ? hi : lo) * 0x00010001u + 0x64006400u) - dup2(1024.f);
        c = s * dup2(-24.f);
    }
    template <int U>
    __device__ __forceinline__ void from(uint32_t v) {
        const f16x2_t sc = h2(v * 0x00010001u + 0x64006400u) - dup2(1024.f);   // exact
        s = (U & 1) ? sc * dup2(0.0625f) : sc;
        c = sc * ((U & 1) ? dup2(-64.f) : dup2(-1024.f));
    }
};
template <>
struct WScale<kQ6_K> {
    f16x2_t s;
    template <int U>
    __device__ __forceinline__ void set(const WBlock<kQ6_K>& b, int lk) {
        const uint32_t w = U < 2 ? b.sc.x : b.sc.y;   // scales 2 U, 2 U + 1 of the half
        s = from((w >> (16 * (U & 1) + 8 * (lk & 1))) & 0xffu);
    }
    static __device__ __forceinline__ f16x2_t from(uint32_t byte) {
        return h2((byte ^ 0x80u) * 0x00010001u + 0x64006400u) - dup2(1152.f);   // signed 8 bits, exact
    }
};

// B operand(s) of depth (U, J). Bits 0x64bb are the fp16 1024 + bb, so quants placed under 0x64 by one and-or
// become exact small integers by one packed add or fused multiply-add.
template <int U, int J>
__device__ __forceinline__ void decode_q4(const uint4& q, const WScale<kQ4_K>& sc, uint32_t k64, f16x8_t (&B)[1]) {
    constexpr uint32_t mask = (U & 1) ? 0x00f000f0u : 0x000f000fu;
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = word_of(q, 2 * J + i);
        e[2 * i] = w2(fma2(h2((w & mask) | k64), sc.s, sc.c));
        e[2 * i + 1] = w2(fma2(h2(((w >> 8) & mask) | k64), sc.s, sc.c));
    }
    __builtin_memcpy(&B[0], e, 16);
}

template <int U, int J>
__device__ __forceinline__ void decode(const WBlock<kQ4_K>& b, const WScale<kQ4_K>& sc, uint32_t k64, f16x8_t (&B)[1]) {
    decode_q4<U, J>(b.q[U >> 1], sc, k64, B);
}

// (q - 8) sc: a nibble in the top four mantissa bits under 0x4c00 is the fp16 16 + q.
template <int U, int J>
__device__ __forceinline__ void decode_centred(const WBlock<kQ4_K>& b, const WScale<kQ4_K>& sc, f16x8_t (&B)[1]) {
    constexpr int lo = (U & 1) ? 2 : 6, hi = (U & 1) ? 6 : 2;   // left shift of bytes 0, 2; right shift of bytes 1, 3
    uint32_t e[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const uint32_t w = word_of(b.q[U >> 1], 2 * J + i);
        e[2 * i] = w2(fma2(h2(((w << lo) & 0x03c003c0u) | 0x4c004c00u), sc.s, sc.c));
        e[2 * i + 1] = w2(fma2(h2(((w >> hi) & 0x03c003c0u) | 0x4c004c00u), sc.s, sc.c));
    }
    __builtin_memcpy(&B[0], e, 16);
}

// (q - 32) sc in two fp16 parts, exactly: magnitudes up to 2048 fit the first one. wd, hd: the ql and qh words of the
// operand's quants.
template <int U>
__device__ __forceinline__ void decode_q6(const uint32_t (&wd)[2], const uint32_t (&hd)[2], f16x2_t s, uint32_t k64,
                                          uint32_t kf, uint32_t k30, f16x8_t (&B)[2]) {
    f16x2_t q[4], p[4];
    uint32_t e[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {   // bytes (0, 2), (1, 3) of both words
        const int o = i & 1;
        constexpr int up = 4 - 2 * U;   // bits 2 U of qh to bits 4, 5
        const int sh = up - 8 * o;
        const uint32_t h = hd[i >> 1];
        uint32_t t = ((sh >= 0 ? h << (sh & 31) : h >> (-sh & 31)) & k30) | k64;
        asm("" : "+v"(t));   // two v_and_or_b32 rather than two ands and an or3
        q[i] = h2(((wd[i >> 1] >> (8 * o + 4 * (U >> 1))) & kf) | t) - dup2(1056.f);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        p[i] = q[i] * s;
        e[i] = w2(p[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) l[i] = w2(fma2(q[i], s, -p[i]));
    __builtin_memcpy(&B[0], e, 16);
    __builtin_memcpy(&B[1], l, 16);
}

template <int U, int J>
__device__ __forceinline__ void decode(const WBlock<kQ6_K>& b, const WScale<kQ6_K>& sc, uint32_t k64, f16x8_t (&B)[2]) {
    const uint32_t wd[2] = {word_of(b.q[U & 1], 2 * J), word_of(b.q[U & 1], 2 * J + 1)};
    const uint32_t hd[2] = {word_of(b.qh, 2 * J), word_of(b.qh, 2 * J + 1)};
    decode_q6<U>(wd, hd, sc.s, k64, 0x000f000fu, 0x00300030u, B);
}

// Q4_K's min terms, sum_g m_g S_g of a block, as one v_mfma_f32_16x16x16_f16 per tile: k = 8 groups x the two fp16
// parts of S_g 2^-5 (|S_g| < 2^20) against m_g twice. Lane (lr, lk): groups 2 lk, 2 lk + 1 of token (row) lr.
__device__ __forceinline__ f16x4_t min_operand(const float2& v) {
    const float s0 = v.x * 0.03125f, s1 = v.y * 0.03125f;
    const _Float16 a0 = static_cast<_Float16>(s0), a1 = static_cast<_Float16>(s1);
    return f16x4_t{a0, static_cast<_Float16>(s0 - static_cast<float>(a0)), a1,
                   static_cast<_Float16>(s1 - static_cast<float>(a1))};
}
__device__ __forceinline__ f16x4_t min_weights(const uint4& h, int lk) {
    const uint32_t sh = 16u * (lk & 1);
    const uint32_t l = (h.z >> sh) & 0x3f3fu;
    const uint32_t g = ((h.w >> (sh + 4)) & 0x0f0fu) | ((h.z >> (sh + 2)) & 0x3030u);
    const uint32_t m = lk < 2 ? l : g;
    const f16x2_t p = h2(((m & 0xffu) | ((m >> 8) << 16)) + 0x64006400u) - dup2(1024.f);   // exact
    return f16x4_t{p[0], p[0], p[1], p[1]};
}

// The same form with the block's scales in the place of its minima.
__device__ __forceinline__ f16x4_t scale_weights(const uint4& h, int lk) {
    const uint32_t sh = 16u * (lk & 1);
    const uint32_t l = (h.y >> sh) & 0x3f3fu;
    const uint32_t g = ((h.w >> sh) & 0x0f0fu) | ((h.y >> (sh + 2)) & 0x3030u);
    const uint32_t m = lk < 2 ? l : g;
    const f16x2_t p = h2(((m & 0xffu) | ((m >> 8) << 16)) + 0x64006400u) - dup2(1024.f);   // exact
    return f16x4_t{p[0], p[0], p[1], p[1]};
}

// A value the compiler may not fold into its users (keeps v_fmac_f32 from
// becoming v_fma_mix_f32, which issues at half the rate).
__device__ __forceinline__ float opaque(float v) {
    asm volatile("" : "+v"(v));
    return v;
}

template <int S>
using IC = std::integral_constant<int, S>;

template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
    (f(IC<I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
    static_for_impl(f, std::make_integer_sequence<int, N>{});
}

}  // namespace
}  // namespace qk
