// Attention over the paged 4-bit cache (kv4_common.hpp) on gfx950: the rows of several requests in one call, single tokens
// and prompts mixed. Row i of a request with n rows and kv_len keys stands at position kv_len - n + i and sees keys
// 0 .. position:
//   score_t = (sum_g scale_tg (q . code_t)_g + min_tg sum(q)_g) / sqrt(D) over the groups g of 64 dims,
//   out = (sum_t p_t scale_t code_t + sum_t p_t min_t) / sum_t p_t, p = exp(score - max)  (x sigmoid(gate)),
// zeros where no key is seen. The reference has the one-token form over an fp32 cache (src/cuda/attn_kernels.cu:72-195,
// src/layer_attn.cpp:103-108).
//
// Both products run on the matrix cores with an fp32 dot product's accuracy: a code is exact in fp16, and the other operand
// (a query row scaled by a power of two; the softmax weights) is two fp16 parts, 22 bits. 8 codes take 9 instructions: a
// nibble under 0x64 is the fp16 1024 + code, or 1024 + 16 code one nibble up, and a packed addition or fma brings it down.
// (Nibbles as they are, subnormal fp16 numbers code * 2^-24, take 5 and are multiplied exactly, but the matrix core aligns a
// product by its operands' exponents as if they were normal: beside a larger weight a smaller one's products lost all but 13
// bits.)
//
// The parts of a score: the products of each group of 64 dims come out of the matrix core by themselves and are scaled in
// fp32; sum_g min_tg sum(q)_g is one product more, of the bf16 minima as they lie in the cache with three bf16 parts, 24
// bits, of each sum. Values are summed as code - 8, with min + 8 scale in the place of min: codes 0..15 would add up to
// numbers as large as the context is long, of which the mean of thousands of values of either sign keeps few bits
// (200000 keys: 2e-3 off, now as near as fp32 values).
//
// Both products are computed transposed, scores^T = K q^T and out^T = V^T p^T, because then the scores that a lane holds (4
// tokens of one row in each half of a tile) are already the p^T operand of the second product: with key row lr of half `x`
// standing for token 8 (lr / 4) + 4 x + lr % 4, lane group lk holds tokens 8 lk .. 8 lk + 7, whose value codes of one dim are
// one word of the cache. Nothing crosses lanes or LDS between the products.
//
// The running reference m of the exponentials bounds score + log2(size), size = max(16 scale, |min|, 2^-40) of the token's
// values, so that a weight p * scale as an fp16 number cannot overflow, and what its last bit loses (2^-30 of the largest
// p * size) is small beside the sum, whatever tokens with sizes far apart a row sees. It moves, and the sums are rescaled, only
// when a token passes it by 8. log2 comes from the bf16 bits, linear between powers of two: below it by at most 0.09. Sizes
// count from 2^-40 up: counted as 2^-100, tokens of zeros would fall out of the softmax's sum when larger ones come.
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "capi_common.hpp"
#include "device_common.hpp"
#include "kv4_common.hpp"

namespace qk {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;              // tokens of a step
constexpr int kSplitWaves = 4;
constexpr int kSplitBlock = kSplitWaves * kWave;
constexpr int kRows = 8;               // (row, head) pairs of a split workgroup
constexpr int kTargetItems = 1024;     // pieces of the whole call
constexpr int kMinTiles = 4;           // of a piece
constexpr int kMaxItems = 1 << 24;     // more than any call has
constexpr float kMoves = 8.0f;         // a token past the reference by more moves it
constexpr float kWeightUp = 0x1p10f;   // weights (p scale up to 2^4) enter fp16 times this

struct Attn4Args {
    const float* q;
    const float* gate;   // or null
    float* out;
    Kv4Cache c;
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* kv_len;
    int max_pages, page_shift, requests, rows, heads, group;
    float* part;         // [item][kRows][D] sums of p v
    float2* stat;        // [item][kRows] (m, l)
    int2* info;          // [row][head] (first item * kRows + row in item, pieces); written for the requests' rows alone
    int items;           // the grid, and what `part` and `stat` hold
    float scale;         // log2(e) / sqrt(D)
};

// A request as the kernels see it, whatever the arrays hold: rows inside q, lengths from 0 to what the table row holds
// (`bad` marks a longer one, whose rows come out NaN). Starts that do not decrease give every row between the first and the
// last one request; of others the rows are not defined, but nothing is read or written out of bounds.
struct Request4 {
    int first, n, len;
    bool bad;
};
__device__ __forceinline__ Request4 request(const Attn4Args& a, int b) {
    const int s = min(max(a.row_start[b], 0), a.rows), e = min(max(a.row_start[b + 1], s), a.rows);
    const int len = a.kv_len[b], most = a.max_pages << a.page_shift;
    return Request4{s, e - s, min(max(len, 0), most), len > most};
}

// ------------------------------------------------------------------ pieces of a call
// Inclusive prefix over the wave.
__device__ __forceinline__ int wave_prefix(int v) {
#define QK_STEP(ctrl, rows) v += __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false)
    QK_STEP(0x111, 0xF);   // row_shr 1, 2, 4, 8
    QK_STEP(0x112, 0xF);
    QK_STEP(0x114, 0xF);
    QK_STEP(0x118, 0xF);
    QK_STEP(0x142, 0xA);   // row 0's last lane to row 1, row 2's to row 3
    QK_STEP(0x143, 0xC);   // lane 31 to the upper half
#undef QK_STEP
    return v;
}

// Piece `item` of the call: request, which of its units (KV head, row block), which piece of the unit's tiles. Every wave
// finds it by itself from the lengths, 64 requests at a time: the whole call, ragged requests and all, is cut into about
// kTargetItems pieces of the same number of tiles.
struct Piece {
    int b, unit, split, splits, tiles;   // tiles: of one piece
    Request4 r;
};
__device__ __forceinline__ int tiles_of(const Request4& r) { return max(1, (r.len + kTile - 1) / kTile); }
__device__ __forceinline__ float units_of(const Attn4Args& a, const Request4& r) {
    return static_cast<float>((static_cast<int64_t>(r.n) * a.group + kRows - 1) / kRows) * static_cast<float>(a.c.heads);
}
__device__ bool find_piece(const Attn4Args& a, int item, Piece& p) {
    const int lane = threadIdx.x & 63;
    Request4 r{0, 0, 0, false};
    if (lane < a.requests) r = request(a, lane);
    float total = units_of(a, r) * static_cast<float>(tiles_of(r));
    for (int b = lane + kWave; b < a.requests; b += kWave) {
        const Request4 s = request(a, b);
        total += units_of(a, s) * static_cast<float>(tiles_of(s));
    }
    total = group_sum<kWave>(total);
    // (rounded sums: the pieces may be one or two more than kTargetItems and one for every unit)
    const int cut = max(static_cast<int>(fminf(ceilf(total * (1.0f / kTargetItems)), 0x1p26f)), kMinTiles);
    p.tiles = cut;
    for (int b0 = 0; b0 < a.requests; b0 += kWave) {
        if (b0) {
            r = Request4{0, 0, 0, false};
            if (b0 + lane < a.requests) r = request(a, b0 + lane);
        }
        const int splits = (tiles_of(r) + cut - 1) / cut;
        const int n = static_cast<int>(fminf(units_of(a, r) * static_cast<float>(splits), static_cast<float>(kMaxItems)));
        const int upto = wave_prefix(n);
        const uint64_t hit = __ballot(item < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int local = item - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
            p.b = b0 + l;
            p.splits = __builtin_amdgcn_readlane(splits, l);
            p.unit = __builtin_amdgcn_readfirstlane(local / p.splits);
            p.split = local - p.unit * p.splits;
            p.r.first = __builtin_amdgcn_readlane(r.first, l);
            p.r.n = __builtin_amdgcn_readlane(r.n, l);
            p.r.len = __builtin_amdgcn_readlane(r.len, l);
            p.r.bad = __builtin_amdgcn_readlane(static_cast<int>(r.bad), l) != 0;
            return true;
        }
        item -= __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// ------------------------------------------------------------------ codes and numbers
// A word's 8 codes less LESS as the fp16 operand.
template <int LESS>
__device__ __forceinline__ f16x8_t codes8(uint32_t w) {
    const f16x2_t down = {(_Float16)(-1024.0f - LESS), (_Float16)(-1024.0f - LESS)}, sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const f16x2_t down16 = {(_Float16)(-64.0f - LESS), (_Float16)(-64.0f - LESS)};
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = i & 2 ? w >> 8 : w;
        f16x2_t h;
        if (i & 1)
            h = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (x & 0x00f000f0u) | 0x64006400u), sixteenth, down16);
        else
            h = __builtin_bit_cast(f16x2_t, (x & 0x000f000fu) | 0x64006400u) + down;
        r[2 * i] = h[0];
        r[2 * i + 1] = h[1];
    }
    return r;
}

// The fp32 product behind a value that is then split in two fp16 parts: kept from being fused into the conversion
// (v_fma_mixlo_f16 rounds once where the other part's subtraction has rounded twice, and the parts miss by an fp16 ulp
// of one weight in some thousands).
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}
__device__ __forceinline__ float low_part(float v) { return v - static_cast<float>(static_cast<_Float16>(v)); }
__device__ __forceinline__ float bf16_part(float v, int part) {   // bf16 part 0, 1, 2 of v, as an fp32 number
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float r = static_cast<float>(static_cast<__bf16>(v));
        if (part == i) return r;
        v -= r;
    }
    return static_cast<float>(static_cast<__bf16>(v));
}
__device__ __forceinline__ float max_over_lk(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
// Two tokens' sizes max(16 scale, |min|, 2^-40) as bf16 bits, from their scales and minima.
__device__ __forceinline__ uint32_t sizes2(uint32_t scale, uint32_t low) {
    const u16x2_t s = __builtin_bit_cast(u16x2_t, scale) + u16x2_t{0x0200, 0x0200};
    const u16x2_t m = __builtin_bit_cast(u16x2_t, low & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_elementwise_max(s, m), u16x2_t{0x2b80, 0x2b80}));
}
__device__ __forceinline__ float log2_of_bits(uint32_t b) { return static_cast<float>(b) * 0x1p-7f - 127.0f; }

// An output from its sums: zero where no key was seen (a weight may be 0 beside a NaN).
__device__ __forceinline__ float finished(const Attn4Args& a, float m, float sum, float tot, size_t o) {
    const float v = m == -FLT_MAX && tot == 0.f ? 0.f : sum / tot;
    return a.gate ? v * sigmoid(a.gate[o]) : v;
}

// ------------------------------------------------------------------ few rows
// Bound by the cache's bytes. A workgroup takes 8 (row, head) pairs that share a KV head - 16 columns: 8 rows x 2 fp16 parts -
// and a range of 32-token tiles, its 4 waves every fourth tile, straight from the cache to operand registers.
// WIDE: pages of 32 tokens and more, so that a tile lies in one page and its addresses are the wave's.
template <int D, bool WIDE>
__global__ __launch_bounds__(kSplitBlock, 2) void split4_kernel(const Attn4Args a) {
    constexpr int NG = D / 64, NV = D / 64, LD = D + 2;
    __shared__ float sums[kSplitWaves][kRows * LD];
    __shared__ float stat[kSplitWaves][kRows][2];
    __shared__ __align__(16) _Float16 qs[2 * kRows][D + 8];   // the queries' parts; 16 bytes more, and 16 rows meet no bank twice
    __shared__ float factors[kRows], qsum[kRows][NG];
    Piece pc;
    if (!find_piece(a, static_cast<int>(blockIdx.x), pc)) return;   // the whole workgroup
    const Request4 r = pc.r;
    const int G = a.group, pairs = r.n * G;
    const int blocks = (pairs + kRows - 1) / kRows;
    const int h = pc.unit / blocks, rb = pc.unit - h * blocks;
    const int lane = threadIdx.x & 63, lr = lane & 15, lk = lane >> 4, part = lr & 1;
    const int wv = wave_in_block();
    const int ti = min(rb * kRows + (lr >> 1), pairs - 1) / G;   // columns past the last pair repeat it
    const int limit = r.len - r.n + ti;                      // this column's last key
    const int first_limit = r.len - r.n + rb * kRows / G;    // the smallest of the workgroup
    const int seen = max(r.len - r.n + min(rb * kRows + kRows - 1, pairs - 1) / G + 1, 0);   // keys that some column sees
    const int t_end = min((pc.split + 1) * pc.tiles, (seen + kTile - 1) / kTile);
    int t = pc.split * pc.tiles + wv;
    const int P = a.c.page;

    // Where a lane's parts of a tile lie, as tokens of the head's cache: `kt` of its octet of key rows (octet lr / 4), `vt` of
    // octet lk (values, scales). Octets that no row sees are read from page 0, a page id outside the cache is not followed.
    struct Where {
        size_t kt, vt;
        bool bad;
    };
    const int32_t* row_table = a.table + static_cast<size_t>(pc.b) * a.max_pages;
    auto where = [&](int tile) {
        Where w;
        const int t0 = tile * kTile;
        if constexpr (WIDE) {
            int id = row_table[t0 >> a.page_shift];   // the wave's; below max_pages since t0 < seen
            w.bad = id < 0 || id >= a.c.pages;
            id = w.bad ? 0 : id;
            const size_t at = (static_cast<size_t>(id) * a.c.heads + h) * P + (t0 & (P - 1));
            w.kt = w.vt = at;
        } else {
            auto octet = [&](int tok, bool& bad) {
                bad = false;
                int id = 0;
                if (tok < seen) {
                    id = row_table[tok >> a.page_shift];
                    bad = id < 0 || id >= a.c.pages;
                    id = bad ? 0 : id;
                }
                return (static_cast<size_t>(id) * a.c.heads + h) * P + (tok & (P - 1));
            };
            bool unused;
            w.kt = octet(t0 + 8 * (lr >> 2), unused);
            w.vt = octet(t0 + 8 * lk, w.bad);
        }
        return w;
    };
    constexpr int KW = NG * 2;   // words of a lane's share of a token's keys
    uint32_t K[2][KW];
    uint4 V[NV], ksc[NG], vsc, vmn;
    bf16x8_t kmn[2];
    bool bad_page = false;
    auto load_k = [&](const Where& w) {
        const size_t tok = w.kt + (WIDE ? 8 * (lr >> 2) : 0) + (lr & 3);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t* p = a.c.k + (tok + 4 * x) * (D / 2) + lk * (4 * KW);
            if constexpr (KW == 8) {
                const uint4 u = ld16(p), v = ld16(p + 16);
                K[x][0] = u.x, K[x][1] = u.y, K[x][2] = u.z, K[x][3] = u.w;
                K[x][4] = v.x, K[x][5] = v.y, K[x][6] = v.z, K[x][7] = v.w;
            } else if constexpr (KW == 4) {
                const uint4 u = ld16(p);
                K[x][0] = u.x, K[x][1] = u.y, K[x][2] = u.z, K[x][3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(p);
                K[x][0] = u.x, K[x][1] = u.y;
            }
            const uint16_t* m = a.c.km + (tok + 4 * x) * NG;
            u32x4_t z = {0u, 0u, 0u, 0u};
            if constexpr (NG == 4) {
                const uint2 u = *reinterpret_cast<const uint2*>(m);
                z[0] = u.x, z[1] = u.y;
            } else if constexpr (NG == 2) {
                z[0] = *reinterpret_cast<const uint32_t*>(m);
            } else {
                z[0] = *m;
            }
            kmn[x] = __builtin_bit_cast(bf16x8_t, z);
        }
        const size_t oct = w.vt + (WIDE ? 8 * lk : 0);   // a multiple of 8
#pragma unroll
        for (int g = 0; g < NG; ++g) ksc[g] = ld16(a.c.ks + oct * NG + 8 * g);
        bad_page = w.bad;
    };
    auto load_v = [&](const Where& w) {
        const size_t oct = w.vt + (WIDE ? 8 * lk : 0);
#pragma unroll
        for (int m = 0; m < NV; ++m) V[m] = ld16(a.c.v + oct * (D / 2) + (64 * m + 4 * lr) * 4);
        vsc = ld16(a.c.vs + oct);
        vmn = ld16(a.c.vm + oct);
    };
    // The rows' queries, scaled by 2^e so that a row's largest magnitude is in [2^14, 2^15), as two fp16 parts: 2 rows a wave,
    // requested before the first tile.
    const int qr = 2 * wv + (lane >> 5), qp = min(rb * kRows + qr, pairs - 1), qt = qp / G;
    const float* qrow = a.q + (static_cast<size_t>(r.first + qt) * a.heads + h * G + (qp - qt * G)) * D + (lane & 31) * (D / 32);
    constexpr int QN = D / 32;
    float qf[QN];
    if constexpr (QN >= 4) {
#pragma unroll
        for (int i = 0; i < QN / 4; ++i) {
            const float4 x = ld4(qrow + 4 * i);
            qf[4 * i] = x.x, qf[4 * i + 1] = x.y, qf[4 * i + 2] = x.z, qf[4 * i + 3] = x.w;
        }
    } else {
        qf[0] = qrow[0], qf[1] = qrow[1];
    }
    const bool any = t < t_end;
    Where next{};
    if (any) {
        const Where w = where(t);
        load_k(w);
        load_v(w);
        if (t + kSplitWaves < t_end) next = where(t + kSplitWaves);
    }
    {
        float m = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            m = fmaxf(m, fabsf(qf[i]));
            bad |= !(fabsf(qf[i]) <= FLT_MAX);
        }
        if (bad) m = INFINITY;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) m = fmaxf(m, __shfl_xor(m, o));
        const bool ok = m <= FLT_MAX;
        int e = 0;
        if (m > 0.f && ok) {
            int em;
            frexpf(m, &em);
            e = 15 - em;
        }
        float s = 0.f;
        const int d0 = (lane & 31) * QN;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const float v = ok ? ldexpf(qf[i], e) : 0.f;
            s += v;
            qs[2 * qr][d0 + i] = static_cast<_Float16>(v);
            qs[2 * qr + 1][d0 + i] = static_cast<_Float16>(low_part(v));
        }
        s = group_sum<64 / QN>(s);
        if ((lane & (64 / QN - 1)) == 0) qsum[qr][d0 / 64] = s;
        if ((lane & 31) == 0) factors[qr] = ok ? ldexpf(a.scale, -e) : __builtin_nanf("");   // products to log2 scores; NaN: a row
    }                                                                                        // with infinities or NaNs
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the tile's loads stay in flight
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f16x8_t Q[2 * NG];   // dims 64 g + 16 lk + 8 (d % 2) + 0..7 of depth d = 2 g + d % 2
#pragma unroll
    for (int d = 0; d < 2 * NG; ++d)
        Q[d] = *reinterpret_cast<const f16x8_t*>(&qs[lr][64 * (d >> 1) + 16 * lk + 8 * (d & 1)]);
    bf16x8_t Qs;   // depth 8 lk + g: bf16 part lk of the sum over group g, in the row's first column
#pragma unroll
    for (int g = 0; g < 8; ++g)
        Qs[g] = static_cast<__bf16>(g < NG && lk < 3 && part == 0 ? bf16_part(qsum[lr >> 1][g < NG ? g : 0], lk) : 0.f);
    const float factor = factors[lr >> 1];
    f32x4_t acc[NV][4];
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[m][e] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float mu = -FLT_MAX, l = 0.f, low = 0.f;
    for (; t < t_end; t += kSplitWaves) {
        const bool more = t + kSplitWaves < t_end;
        f32x4_t S[2];
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) S[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kmn[x], Qs, zero, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint32_t w[4] = {ksc[g].x, ksc[g].y, ksc[g].z, ksc[g].w};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f32x4_t T = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<0>(K[x][2 * g]), Q[2 * g], zero, 0, 0, 0);
                T = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<0>(K[x][2 * g + 1]), Q[2 * g + 1], T, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    S[x][i] = __builtin_fmaf(T[i], i & 1 ? bf16_hi(w[2 * x + (i >> 1)]) : bf16_lo(w[2 * x + (i >> 1)]), S[x][i]);
            }
        }
        const float f = bad_page ? __builtin_nanf("") : factor;
        if (more) load_k(next);
        float s[8], sv[8], mv[8];
        uint32_t size[4];
        const uint32_t vs[4] = {vsc.x, vsc.y, vsc.z, vsc.w}, vm[4] = {vmn.x, vmn.y, vmn.z, vmn.w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = S[i >> 2][i & 3];
            s[i] = (v + dpp_move<0xB1>(v)) * f;   // both fp16 parts of the query
            sv[i] = i & 1 ? bf16_hi(vs[i >> 1]) : bf16_lo(vs[i >> 1]);
            mv[i] = __builtin_fmaf(8.0f, sv[i], i & 1 ? bf16_hi(vm[i >> 1]) : bf16_lo(vm[i >> 1]));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) size[i] = sizes2(vs[i], vm[i]);
        if (t * kTile + kTile - 1 > first_limit) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (t * kTile + 8 * lk + i > limit) {   // what lies there is anything: no 0 * NaN
                    s[i] = -INFINITY;
                    sv[i] = mv[i] = 0.f;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = fmaxf(top, s[i] + log2_of_bits(i & 1 ? size[i >> 1] >> 16 : size[i >> 1] & 0xffffu));
        if (__ballot(top > mu + kMoves)) {
            const float now = fmaxf(mu, max_over_lk(top));
            const float shrink = __builtin_amdgcn_exp2f(mu - now);
            mu = now;
            l *= shrink;
            low *= shrink;
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][e][i] *= shrink;
        }
        f16x8_t W;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] - mu);
            l += p;
            low = __builtin_fmaf(p, mv[i], low);
            const float w = rounded(p * (sv[i] * kWeightUp));
            W[i] = static_cast<_Float16>(part ? low_part(w) : w);
        }
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            const uint32_t w[4] = {V[m].x, V[m].y, V[m].z, V[m].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[m][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<8>(w[e]), W, acc[m][e], 0, 0, 0);
        }
        if (more) {
            load_v(next);
            if (t + 2 * kSplitWaves < t_end) next = where(t + 2 * kSplitWaves);
        }
    }
    // The waves' sums meet in LDS; the two parts of a row are neighbouring columns, each lane of a pair writes every
    // other dim of both. Row 4 lk + i of value tile (m, e) is dim 64 m + 4 (4 lk + i) + e.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    low += __shfl_xor(low, 16);
    low += __shfl_xor(low, 32);
    float* mine = sums[wv] + (lr >> 1) * LD;
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float u = acc[m][e][i] + dpp_move<0xB1>(acc[m][e][i]);
                const float v = acc[m][e + 1][i] + dpp_move<0xB1>(acc[m][e + 1][i]);
                mine[64 * m + 4 * (4 * lk + i) + e + part] = __builtin_fmaf(part ? v : u, 1.0f / kWeightUp, low);
            }
    if (lane < 16 && part == 0) {
        stat[wv][lr >> 1][0] = mu;
        stat[wv][lr >> 1][1] = l;
    }
    __syncthreads();
    const int rows = min(kRows, pairs - rb * kRows);
    for (int i = threadIdx.x; i < rows * D; i += kSplitBlock) {
        const int row = i / D, d = i - row * D;
        float m = stat[0][row][0];
#pragma unroll
        for (int w = 1; w < kSplitWaves; ++w) m = fmaxf(m, stat[w][row][0]);
        float sum = 0.f, tot = 0.f;
#pragma unroll
        for (int w = 0; w < kSplitWaves; ++w) {
            const float k = __builtin_amdgcn_exp2f(stat[w][row][0] - m);
            sum += k * sums[w][row * LD + d];
            tot += k * stat[w][row][1];
        }
        if (r.bad) tot = __builtin_nanf("");
        const int at = rb * kRows + row, tok = at / G;
        const size_t o = (static_cast<size_t>(r.first + tok) * a.heads + h * G + (at - tok * G)) * D + d;
        if (pc.splits == 1) {
            a.out[o] = finished(a, m, sum, tot, o);
        } else {
            a.part[(static_cast<size_t>(blockIdx.x) * kRows + row) * D + d] = sum;
            if (d == 0) a.stat[static_cast<size_t>(blockIdx.x) * kRows + row] = make_float2(m, tot);
        }
        if (d == 0 && pc.split == 0) a.info[o / D] = make_int2(static_cast<int>(blockIdx.x) * kRows + row, pc.splits);
    }
}

// ------------------------------------------------------------------ join
// Joins the pieces of (row, head) pairs: a workgroup of NW waves per pair, wave w takes pieces w, w + NW, ... Lanes hold the
// dims.
template <int D, int NW>
__global__ __launch_bounds__(NW* kWave) void join4_kernel(const Attn4Args a) {
    constexpr int V = D / kWave;
    __shared__ float sums[NW][D], ls[NW], ms[NW];
    const int lane = threadIdx.x & 63, wv = wave_in_block();
    // Pairs of the requests' rows alone: only those have an entry of this call (the workspace may hold an earlier one's).
    const int from = min(max(a.row_start[0], 0), a.rows) * a.heads, live = min(max(a.row_start[a.requests], 0), a.rows) * a.heads;
    const int pair = static_cast<int>(blockIdx.x);
    if (pair < from || pair >= live) return;   // the whole workgroup
    const int2 in = a.info[pair];
    if (in.y <= 1 || in.x < 0 || in.y > a.items - in.x / kRows) return;   // one piece; or starts that decrease
    const int slot = in.x % kRows, first = in.x / kRows;
    float m = -FLT_MAX, l = 0.f, s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.f;
    constexpr int U = 4;   // pieces in flight
    for (int p0 = wv; p0 < in.y; p0 += U * NW) {
        float2 st[U];
        float x[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const size_t q = static_cast<size_t>(first + min(p0 + u * NW, in.y - 1)) * kRows + slot;
            st[u] = a.stat[q];
            const float* p = a.part + q * D + V * lane;
            if constexpr (V == 4) {
                const float4 y = ld4(p);
                x[u][0] = y.x, x[u][1] = y.y, x[u][2] = y.z, x[u][3] = y.w;
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) x[u][i] = p[i];
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // all U loads before the first use
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p0 + u * NW >= in.y) break;
            const float now = fmaxf(m, st[u].x);
            const float was = __builtin_amdgcn_exp2f(m - now), f = __builtin_amdgcn_exp2f(st[u].x - now);
            m = now;
            l = l * was + st[u].y * f;
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] = s[i] * was + x[u][i] * f;
        }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) sums[wv][V * lane + i] = s[i];
    if (lane == 0) {
        ms[wv] = m;
        ls[wv] = l;
    }
    __syncthreads();
    for (int d = threadIdx.x; d < D; d += NW * kWave) {
        float top = ms[0];
#pragma unroll
        for (int w = 1; w < NW; ++w) top = fmaxf(top, ms[w]);
        float sum = 0.f, tot = 0.f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            const float f = __builtin_amdgcn_exp2f(ms[w] - top);
            sum += f * sums[w][d];
            tot += f * ls[w];
        }
        const size_t o = static_cast<size_t>(pair) * D + d;
        a.out[o] = finished(a, top, sum, tot, o);
    }
}

// ------------------------------------------------------------------ host
// split4_kernel's pieces are at most kTargetItems (and a few for rounding) plus one per unit; units at most one per 8 pairs
// plus one per request that has rows.
int64_t item_bound(int rows, int requests, int heads, int kv_heads) {
    const int64_t pairs = static_cast<int64_t>(rows) * (heads / kv_heads);
    return kTargetItems + 8 + (pairs / kRows + std::min(rows, requests)) * kv_heads;
}
size_t align_up(size_t b) { return (b + 255) & ~size_t{255}; }

struct Layout {
    int64_t items;
    size_t stat, info, bytes;
};
Layout layout(int rows, int requests, int heads, int kv_heads, int dim) {
    Layout l;
    l.items = item_bound(rows, requests, heads, kv_heads);
    l.stat = align_up(static_cast<size_t>(l.items) * kRows * dim * 4);
    l.info = l.stat + align_up(static_cast<size_t>(l.items) * kRows * 8);
    l.bytes = l.info + align_up(static_cast<size_t>(rows) * heads * 8);
    return l;
}

template <int D>
void launch(const Attn4Args& a, hipStream_t s) {
    const auto split = a.c.page >= kTile ? split4_kernel<D, true> : split4_kernel<D, false>;
    split<<<static_cast<unsigned>(a.items), kSplitBlock, 0, s>>>(a);
    const unsigned pairs = static_cast<unsigned>(a.rows) * static_cast<unsigned>(a.heads);
    if (pairs <= 128)   // few rows: many pieces each
        join4_kernel<D, 16><<<pairs, 16 * kWave, 0, s>>>(a);
    else
        join4_kernel<D, 4><<<pairs, 4 * kWave, 0, s>>>(a);
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qwen_attn_kv4_workspace_bytes(int rows, int requests, int heads, int kv_heads, int dim) {
    if (rows <= 0 || requests <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dim <= 0) return 0;
    return layout(rows, requests, heads, kv_heads, dim).bytes;
}

int qwen_attn_kv4_rows(const float* q, const uint8_t* k_codes, const uint8_t* v_codes, const uint16_t* k_scale,
                       const uint16_t* k_min, const uint16_t* v_scale, const uint16_t* v_min, int pages, int page_size,
                       const int32_t* block_table, int max_pages, const int32_t* row_start, const int32_t* kv_len,
                       int requests, const float* gate, float* out, int rows, int heads, int kv_heads, int dim,
                       void* workspace, size_t workspace_bytes, void* stream) {
    const Kv4Cache c{const_cast<uint8_t*>(k_codes),  const_cast<uint8_t*>(v_codes),  const_cast<uint16_t*>(k_scale),
                     const_cast<uint16_t*>(k_min),   const_cast<uint16_t*>(v_scale), const_cast<uint16_t*>(v_min),
                     pages, page_size, kv_heads, dim};
    if (const int rc = kv4_check("attn_kv4_rows", c)) return rc;
    QK_REQUIRE(heads > 0 && heads % kv_heads == 0, "attn_kv4_rows: %d query heads over %d KV heads", heads, kv_heads);
    QK_REQUIRE(rows >= 0 && requests >= 0 && max_pages >= 0, "attn_kv4_rows: negative size");
    QK_REQUIRE(requests <= kKv4MaxRequests, "attn_kv4_rows: %d requests (at most %d)", requests, kKv4MaxRequests);
    // (tokens a few tiles past a row's end are computed in 32 bits too)
    QK_REQUIRE(static_cast<int64_t>(max_pages) * page_size <= (1 << 30), "attn_kv4_rows: table rows of %d pages", max_pages);
    if (rows == 0 || requests == 0) return ok();
    QK_REQUIRE(q && out && row_start && kv_len && (block_table || max_pages == 0), "attn_kv4_rows: null pointer");
    QK_REQUIRE(static_cast<int64_t>(rows) * heads <= (int64_t{1} << 24), "attn_kv4_rows: %d rows of %d heads exceed one call",
               rows, heads);
    QK_REQUIRE(aligned16(q) && aligned16(out) && (!gate || aligned16(gate)),
               "attn_kv4_rows: q, gate and out must be 16-byte aligned");
    const size_t row_bytes = static_cast<size_t>(rows) * heads * dim * 4;
    QK_REQUIRE(apart(out, row_bytes, q, row_bytes), "attn_kv4_rows: out is q or overlaps it");
    QK_REQUIRE(!gate || gate == out || apart(out, row_bytes, gate, row_bytes), "attn_kv4_rows: out overlaps gate out of place");
    const Layout l = layout(rows, requests, heads, kv_heads, dim);
    QK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= l.bytes,
               "attn_kv4_rows: workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, l.bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    Attn4Args a;
    a.q = q;
    a.gate = gate;
    a.out = out;
    a.c = c;
    a.table = block_table;
    a.row_start = row_start;
    a.kv_len = kv_len;
    a.max_pages = max_pages;
    a.page_shift = __builtin_ctz(static_cast<unsigned>(page_size));
    a.requests = requests;
    a.rows = rows;
    a.heads = heads;
    a.group = heads / kv_heads;
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(dim)));
    a.part = reinterpret_cast<float*>(ws);
    a.stat = reinterpret_cast<float2*>(ws + l.stat);
    a.info = reinterpret_cast<int2*>(ws + l.info);
    a.items = static_cast<int>(l.items);
    const hipStream_t s = as_stream(stream);
    if (dim == 64)
        launch<64>(a, s);
    else if (dim == 128)
        launch<128>(a, s);
    else
        launch<256>(a, s);
    return check_launch("attn_kv4_rows");
}

}  // extern "C"
