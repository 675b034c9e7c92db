// The paged 4-bit key / value cache on gfx950: storing fresh keys and values, reading slots back. Layout and quantization:
// kv4_common.hpp. Page bookkeeping is that of any paged cache (kv8_plan). The attention that reads it: kv4_attn.hip.
//
// The reference keeps one sequence's keys and values in fp32 rows of a fixed array (src/layer_attn.cpp:44-46, copied to
// row pos at :99-100); these entry points have no counterpart there.
#include <algorithm>
#include <cfloat>

#include "capi_common.hpp"
#include "kv4_common.hpp"

namespace qk {
namespace {

// ------------------------------------------------------------------ store
// A row of a head lies on D / 4 lanes, 4 dims each: the groups' smallest and largest values by lane exchanges, every lane its 4 codes.
// Keys: the row's words, one per pair of lanes. Values lie 8 tokens to a word, so a workgroup takes the pieces that begin in
// its 8 rows (a piece: neighbouring rows with neighbouring slots of an octet of tokens; of a prompt one whole octet), hands
// the codes over in LDS and writes an octet's words whole. A piece that fills only a part of them clears and sets its own
// nibbles by two 32-bit atomics: other rows, of any workgroup, may have the others, and no order shows in the result.
// Bound by latency: one round of loads, the reductions, the stores.
constexpr int kStore4Rows = 8;
constexpr int kStore4Block = 512;

template <bool ALIGNED>
__device__ __forceinline__ float4 row4(const float* p) {
    if constexpr (ALIGNED) return ld4(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

template <int G>
__device__ __forceinline__ float group_min(float v) {
#pragma unroll
    for (int o = 1; o < G; o <<= 1) v = fminf(v, __shfl_xor(v, o));
    return v;
}

// Codes of a lane's 4 dims of a group on G lanes.
template <int G>
__device__ __forceinline__ void quantize4(const float4 x, Kv4Group& g, uint32_t (&c)[4]) {
    const float v[4] = {x.x, x.y, x.z, x.w};
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) bad |= !(fabsf(v[i]) <= FLT_MAX);
    const uint64_t mine = (G == 64 ? ~0ull : ((1ull << (G & 63)) - 1)) << ((threadIdx.x & 63) & ~(G - 1));
    bad = (__ballot(bad) & mine) != 0;
    const float lo = group_min<G>(fminf(fminf(v[0], v[1]), fminf(v[2], v[3])));
    const float hi = -group_min<G>(fminf(fminf(-v[0], -v[1]), fminf(-v[2], -v[3])));
    g = kv4_group(lo, hi, bad);
#pragma unroll
    for (int i = 0; i < 4; ++i) c[i] = bad ? 0u : kv4_code(v[i], g);
}

__device__ __forceinline__ uint16_t bf16_bits(float f) { return static_cast<uint16_t>(__float_as_uint(f) >> 16); }

// Grid: x = shares of kStore4Rows rows, y = head, z = keys, values of the first gridDim.x shares, of the next ones, and so on.
template <int D, bool ALIGNED>
__global__ __launch_bounds__(kStore4Block) void kv4_store_kernel(const float* __restrict__ k, const float* __restrict__ v,
                                                                 int64_t k_stride, int64_t v_stride,
                                                                 const int32_t* __restrict__ slots, int rows, const Kv4Cache c) {
    constexpr int LPR = D / 4, RPW = kWave / LPR, NG = D / 64, WAVES = kStore4Block / kWave;
    __shared__ uint32_t codes[2 * kStore4Rows][LPR];   // a value row's codes, a byte a dim
    const int lane = threadIdx.x & 63, l = lane % LPR, h = blockIdx.y, P = c.page;
    const int total = c.pages * P;
    const uint32_t share = (blockIdx.z >> 1) * gridDim.x + blockIdx.x;
    if (static_cast<int64_t>(share) * kStore4Rows >= rows) return;   // the whole workgroup
    const int base = static_cast<int>(share) * kStore4Rows;
    // Lane i of every wave looks at row base - 1 + i; `cont`: the row goes on with the piece of the one before it.
    const int64_t seen = static_cast<int64_t>(base) - 1 + lane;
    int slot = -1;
    if (lane <= 2 * kStore4Rows && seen >= 0 && seen < rows) slot = slots[seen];
    const bool in = slot >= 0 && slot < total;
    const int before = __shfl_up(slot, 1);
    const uint64_t cont = __ballot(lane > 0 && in && (slot & 7) != 0 && before == slot - 1);
    const uint64_t live = __ballot(in);
    const int wv = wave_in_block();
    if ((blockIdx.z & 1) == 0) {
#pragma unroll
        for (int i0 = 0; i0 < kStore4Rows; i0 += WAVES * RPW) {
            const int i = i0 + wv * RPW + lane / LPR, s = __shfl(slot, 1 + i);
            if (i >= kStore4Rows || !((live >> (1 + i)) & 1)) continue;
            const float4 x = row4<ALIGNED>(k + (base + i) * k_stride + h * D + 4 * l);
            Kv4Group g;
            uint32_t q[4];
            quantize4<16>(x, g, q);
            const uint32_t part = q[0] | (q[1] << 16) | (q[2] << 4) | (q[3] << 20);   // elements 4 (l % 2) + 0..3 of a word
            const uint32_t other = static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(part), 0xB1, 0xF, 0xF, false));
            const int pg = s / P, t = s - pg * P;
            const size_t at = static_cast<size_t>(pg) * c.heads + h, tok = at * P + t;
            if ((l & 1) == 0) {
                const int d = 4 * l, word = (d % 64) / 16 * (2 * NG) + 2 * (d / 64) + (d % 16) / 8;
                reinterpret_cast<uint32_t*>(c.k)[tok * (D / 8) + word] = part | (other << 8);
            }
            if (l % 16 == 0) {
                c.ks[((at * P + (t & ~7)) * NG) + (l / 16) * 8 + (t & 7)] = bf16_bits(g.scale);
                c.km[tok * NG + l / 16] = bf16_bits(g.low);
            }
        }
        return;
    }
    // rows lo .. hi - 1 (as lanes): the pieces that begin in this share
    const int lo = 1 + __builtin_ctzll(~(cont >> 1));
    const int hi = 1 + kStore4Rows + __builtin_ctzll(~(cont >> (1 + kStore4Rows)));
#pragma unroll
    for (int i0 = 0; i0 < 2 * kStore4Rows; i0 += WAVES * RPW) {
        const int i = i0 + wv * RPW + lane / LPR, at_lane = lo + i, s = __shfl(slot, at_lane & 63);
        const bool take = i < 2 * kStore4Rows && at_lane < hi && ((live >> at_lane) & 1);
        if (!take) continue;   // whole rows: the reductions below stay inside one
        const float4 x = row4<ALIGNED>(v + (static_cast<int64_t>(base) - 1 + at_lane) * v_stride + h * D + 4 * l);
        Kv4Group g;
        uint32_t q[4];
        quantize4<LPR>(x, g, q);
        codes[i][l] = q[0] | (q[1] << 8) | (q[2] << 16) | (q[3] << 24);
        if (l == 0) {
            const int pg = s / P;
            const size_t tok = (static_cast<size_t>(pg) * c.heads + h) * P + (s - pg * P);
            c.vs[tok] = bf16_bits(g.scale);
            c.vm[tok] = bf16_bits(g.low);
        }
    }
    __syncthreads();
    uint64_t starts = live & ~cont & ((1ull << hi) - 1) & ~((1ull << lo) - 1);
    for (int skip = threadIdx.x / D; skip > 0; --skip) starts &= starts - 1;   // the pieces of this thread's dims, in turn
    const int d = threadIdx.x % D;
    while (starts) {
        const int first = __builtin_ctzll(starts);
        const int n = 1 + __builtin_ctzll(~(cont >> (first + 1)));
        const int s = __builtin_amdgcn_readlane(slot, first), pg = s / P, t = s - pg * P;
        uint32_t w = 0, mask = 0;
        for (int j = 0; j < n; ++j) {
            const int sh = kv4_shift((t & 7) + j);
            w |= ((codes[first - lo + j][d >> 2] >> (8 * (d & 3))) & 15u) << sh;
            mask |= 15u << sh;
        }
        uint32_t* p = reinterpret_cast<uint32_t*>(c.v) +
                      ((static_cast<size_t>(pg) * c.heads + h) * (P >> 3) + static_cast<size_t>(t >> 3)) * D + d;
        if (n == 8) {
            *p = w;
        } else {
            __hip_atomic_fetch_and(p, ~mask, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            __hip_atomic_fetch_or(p, w, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int i = 0; i < kStore4Block / D; ++i) starts &= starts - 1;
    }
}

// ------------------------------------------------------------------ read
// Slots back as fp32 rows: a thread takes 4 dims of a row's head; a negative slot gives zeros, one past the cache NaN.
// Write-bound (8 bytes out per byte of codes); the values' words are read once per token of their octet, from L1 where the
// tokens are neighbours.
__global__ __launch_bounds__(256) void kv4_read_kernel(const Kv4Cache c, const int32_t* __restrict__ slots, int rows,
                                                       float* __restrict__ k, float* __restrict__ v) {
    const int d_shift = __builtin_ctz(c.dim) - 2, p_shift = __builtin_ctz(c.page), ng = c.dim >> 6;
    const uint32_t per_row = static_cast<uint32_t>(c.heads) << d_shift, n = static_cast<uint32_t>(rows) * per_row;   // below 2^31
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
        const uint32_t r = i / per_row, rest = i - r * per_row;
        const int h = static_cast<int>(rest >> d_shift), d = 4 * (static_cast<int>(rest) & ((1 << d_shift) - 1));
        const int s = slots[r];
        float a[4] = {0.f, 0.f, 0.f, 0.f}, b[4] = {0.f, 0.f, 0.f, 0.f};
        if (s >= c.pages * c.page) {
#pragma unroll
            for (int j = 0; j < 4; ++j) a[j] = b[j] = __builtin_nanf("");
        } else if (s >= 0) {
            const int pg = s >> p_shift, t = s & (c.page - 1);
            const size_t at = static_cast<size_t>(pg) * c.heads + h, tok = (at << p_shift) + t;
            const int word = (d % 64) / 16 * (2 * ng) + 2 * (d / 64) + (d % 16) / 8;
            const uint32_t kw = reinterpret_cast<const uint32_t*>(c.k)[tok * (c.dim / 8) + word];
            const uint4 vw = ld16(c.v + ((((at << p_shift) + (t & ~7)) >> 3) * c.dim + d) * 4);
            const float ks = bf16_value(c.ks[((at << p_shift) + (t & ~7)) * ng + (d >> 6) * 8 + (t & 7)]);
            const float km = bf16_value(c.km[tok * ng + (d >> 6)]), vs = bf16_value(c.vs[tok]), vm = bf16_value(c.vm[tok]);
            const uint32_t w[4] = {vw.x, vw.y, vw.z, vw.w};
#pragma unroll
            for (int j = 0; j < 4; ++j) {   // one rounding; 15 scale by itself may pass the largest number
                a[j] = __builtin_fmaf(ks, static_cast<float>((kw >> kv4_shift((d & 4) + j)) & 15u), km);
                b[j] = __builtin_fmaf(vs, static_cast<float>((w[j] >> kv4_shift(t & 7)) & 15u), vm);
            }
        }
        st4(k + 4 * static_cast<size_t>(i), make_float4(a[0], a[1], a[2], a[3]));
        st4(v + 4 * static_cast<size_t>(i), make_float4(b[0], b[1], b[2], b[3]));
    }
}

template <int D>
void launch_store(const float* k, const float* v, int64_t ks, int64_t vs, const int32_t* slots, int rows, const Kv4Cache& c,
                  bool vec, hipStream_t s) {
    const dim3 shares = grid_of(blocks_for(rows, kStore4Rows)), grid(shares.x, static_cast<unsigned>(c.heads), 2 * shares.y);
    const auto kernel = vec ? kv4_store_kernel<D, true> : kv4_store_kernel<D, false>;
    kernel<<<grid, kStore4Block, 0, s>>>(k, v, ks, vs, slots, rows, c);
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qwen_kv4_store_rows(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* slots, int rows,
                        uint8_t* k_codes, uint8_t* v_codes, uint16_t* k_scale, uint16_t* k_min, uint16_t* v_scale,
                        uint16_t* v_min, int pages, int page_size, int kv_heads, int dim, void* stream) {
    const Kv4Cache c{k_codes, v_codes, k_scale, k_min, v_scale, v_min, pages, page_size, kv_heads, dim};
    if (const int rc = kv4_check("kv4_store_rows", c)) return rc;
    QK_REQUIRE(rows >= 0, "kv4_store_rows: negative rows %d", rows);
    if (rows == 0) return ok();
    QK_REQUIRE(k && v && slots, "kv4_store_rows: null pointer");
    const int64_t width = static_cast<int64_t>(kv_heads) * dim;
    QK_REQUIRE(rows == 1 || (k_stride >= width && v_stride >= width), "kv4_store_rows: row strides below kv_heads x dim");
    const bool vec = aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0;
    const hipStream_t s = as_stream(stream);
    if (dim == 64)
        launch_store<64>(k, v, k_stride, v_stride, slots, rows, c, vec, s);
    else if (dim == 128)
        launch_store<128>(k, v, k_stride, v_stride, slots, rows, c, vec, s);
    else
        launch_store<256>(k, v, k_stride, v_stride, slots, rows, c, vec, s);
    return check_launch("kv4_store_rows");
}

int qwen_kv4_read_rows(const uint8_t* k_codes, const uint8_t* v_codes, const uint16_t* k_scale, const uint16_t* k_min,
                       const uint16_t* v_scale, const uint16_t* v_min, int pages, int page_size, int kv_heads, int dim,
                       const int32_t* slots, int rows, float* k, float* v, void* stream) {
    const Kv4Cache c{const_cast<uint8_t*>(k_codes),  const_cast<uint8_t*>(v_codes),  const_cast<uint16_t*>(k_scale),
                     const_cast<uint16_t*>(k_min),   const_cast<uint16_t*>(v_scale), const_cast<uint16_t*>(v_min),
                     pages, page_size, kv_heads, dim};
    if (const int rc = kv4_check("kv4_read_rows", c)) return rc;
    QK_REQUIRE(rows >= 0, "kv4_read_rows: negative rows %d", rows);
    if (rows == 0) return ok();
    QK_REQUIRE(slots && k && v, "kv4_read_rows: null pointer");
    QK_REQUIRE(aligned16(k) && aligned16(v), "kv4_read_rows: outputs must be 16-byte aligned");
    const int64_t items = static_cast<int64_t>(rows) * kv_heads * (dim / 4);
    QK_REQUIRE(items <= 0x7fffffff, "kv4_read_rows: %d rows exceed one call", rows);
    QK_REQUIRE(apart(k, static_cast<size_t>(items) * 16, v, static_cast<size_t>(items) * 16), "kv4_read_rows: k and v overlap");
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((items + 255) / 256, 8192));
    kv4_read_kernel<<<grid, 256, 0, as_stream(stream)>>>(c, slots, rows, k, v);
    return check_launch("kv4_read_rows");
}

}  // extern "C"
