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
// bits, of each sum. Values are summed as code - 8 of even tokens and code - 7 of odd ones, with min + 8 scale and min + 7 scale in
// the place of min: codes 0..15 would add up to numbers as large as the context is long, of which the mean of thousands of values
// of either sign keeps few bits (one row at 200000 keys: 2e-3 off). So would code - 8 alone, at half a code a token: where a row's
// keys come one after the other, 5.7e-6 of the outputs at 5000 of them and 1.5e-5 at 12000, now 0.8e-6 and 1.3e-6 (fp32 values in
// a library's products: 0.9e-6 and 1.1e-6).
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
#include <numeric>
#include <type_traits>
#include <utility>

#include "capi_common.hpp"
#include "device_common.hpp"
#include "kv4_common.hpp"
#include "kv4_places.hpp"

namespace qk {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2_t __attribute__((ext_vector_type(2)));

constexpr int kTile = 32;              // tokens of a step
constexpr int kSplitWaves = 4;
constexpr int kWholeWaves = 8;
constexpr int kMaxItems = 1 << 24;     // more than any call has
constexpr int kSplitMax = 64;          // (row, head) pairs of a request and KV head that always take split4_kernel; a row does
constexpr int kSplitOnly = 1024;       // and of a whole call that has no more rows than requests
constexpr int kLightUnits = 1024;      // of a light call, see Weight
constexpr int kLightWork = 25 * 1024;  // its units x (tiles + kUnitCost) at D = 256
constexpr int kUnitCost = 8;
constexpr int kEvenLess = 8, kOddLess = 7;   // what a value's code is less when it is summed, see above
constexpr int kMaxUp = 110;             // tiny queries are taken times 2^110 at most, so that what undoes it is a normal number
constexpr float kMoves = 8.0f;         // a token past the reference by more moves it
constexpr float kWeightUp = 10.0f;     // log2 of what exponentials, and so all sums, are taken times: weights fill fp16

struct Attn4Args {
    const float* q;
    const float* gate;   // or null
    float* out;
    Kv4Cache c;
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* kv_len;
    int max_pages, page_shift, requests, rows, heads, group;
    float* part;         // [place][D] sums of p v, where Places says
    float2* stat;        // [place] (m, l)
    int2* info;          // [row][head] (place of the first piece, pieces); written for the requests' rows alone
    int items;           // split4_kernel's pieces that have places, kRows each
    int all_places;      // of the workspace
    int places;          // split4_kernel's workgroups that the card holds at once
    int split_all;       // every request takes split4_kernel
    int light_work;      // of a light call at most
    int light;           // the call is light whatever its lengths are (and split_all)
    int whole;           // and every unit's tiles are one piece: nothing is joined
    int prompt_step;     // tiles of a step of prompt4_kernel's line (a power of two)
    float scale;         // log2(e) / sqrt(D)
};

// A request as the kernels see it, whatever the arrays hold: rows inside q, lengths from 0 to what the table row holds
// (`bad` marks a longer one, whose rows come out NaN). Starts that do not decrease give every row between the first and the
// last one request; of others the rows are not defined, but nothing is read or written out of bounds.
struct Request4 {
    int first, n, len;
    bool bad;
};
__device__ __forceinline__ Request4 request_of(const Attn4Args& a, int start, int end, int len) {
    const int s = min(max(start, 0), a.rows), e = min(max(end, s), a.rows), most = a.max_pages << a.page_shift;
    return Request4{s, e - s, min(max(len, 0), most), len > most};
}
__device__ __forceinline__ Request4 request(const Attn4Args& a, int b) {
    return request_of(a, a.row_start[b], a.row_start[b + 1], a.kv_len[b]);
}

__device__ __forceinline__ Request4 of_lane(const Request4& r, int l) {
    return Request4{__builtin_amdgcn_readlane(r.first, l), __builtin_amdgcn_readlane(r.n, l), __builtin_amdgcn_readlane(r.len, l),
                    __builtin_amdgcn_readlane(static_cast<int>(r.bad), l) != 0};
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
__device__ __forceinline__ int wave_max(int v) {
#define QK_STEP(ctrl, rows) v = max(v, __builtin_amdgcn_update_dpp(v, v, ctrl, rows, 0xF, false))
    QK_STEP(0x111, 0xF);
    QK_STEP(0x112, 0xF);
    QK_STEP(0x114, 0xF);
    QK_STEP(0x118, 0xF);
    QK_STEP(0x142, 0xA);
    QK_STEP(0x143, 0xC);
#undef QK_STEP
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_total(int v) { return __builtin_amdgcn_readlane(wave_prefix(v), 63); }

// Piece `item` of the call: request, which of its units (KV head, row block), which piece of the unit's tiles. Every wave
// finds it by itself from the lengths. No piece has more than `cut` tiles, a unit's pieces are of one size, and both are whole
// turns of the waves. `cut` is the least that still gives each of the card's places one piece at most, since a place that takes a
// second one makes the call half as long again; with more units than places, four pieces. Lengths are held in registers, 64
// requests to one, up to HELD x 64 (16 for all calls cost one token 1 us, 4 for all 1000 requests 170 us where they take 90).
struct Piece {
    int b, unit, split, splits, tiles;   // tiles: of one piece
    Request4 r;
};
__device__ __forceinline__ int tiles_of(const Request4& r) { return max(1, (r.len + kTile - 1) / kTile); }
__device__ __forceinline__ bool is_small(const Attn4Args& a, const Request4& r) {
    return a.split_all || r.n * a.group <= max(kSplitMax, a.group);   // rows * heads <= 2^24
}
__device__ __forceinline__ float units_of(const Attn4Args& a, const Request4& r) {
    const uint32_t blocks = (static_cast<uint32_t>(r.n) * static_cast<uint32_t>(a.group) + kRows - 1) / kRows;
    return static_cast<float>(blocks) * static_cast<float>(a.c.heads);
}
// Whether a call is light: whether split4_kernel takes its larger requests too. A unit of 8 pairs and a tile cost a CU 0.3 us
// there, and the unit's start and end as much as 8 tiles; 128 pairs and a tile 2.2 us in prompt4_kernel, which begins and ends
// with 20 us and has more pieces to join. (100 rows of a prompt 7 us for 33, 11 with a table row of 200 pages, 500 rows 30 for 44, 12
// rows at 3000 keys 15 for 33, 20 requests of 20 rows at 500 keys 36 for 47; past it, 130 rows at 4000 keys 69 for 52, 30 of 12 rows
// at 2000 keys 76 for 66.) Both kernels weigh a call's requests alike: sums of whole numbers, exact where they matter.
struct Weight {
    float work = 0.f, units = 0.f;
    __device__ __forceinline__ void add(const Attn4Args& a, const Request4& r) {
        const float u = units_of(a, r);
        units += u;
        if (!is_small(a, r)) work += u * static_cast<float>(tiles_of(r) + kUnitCost);
    }
    __device__ __forceinline__ bool light(const Attn4Args& a) const {   // over the wave's lanes
        return a.light_work > 0 && group_sum<kWave>(work) <= static_cast<float>(a.light_work) &&
               group_sum<kWave>(units) <= static_cast<float>(kLightUnits);
    }
};
// n / d, both below 2^27, the quotient below 2^20; inverse within 2^-22 of 1 / d.
__device__ __forceinline__ int quotient(int n, int d, float inverse) {
    int q = static_cast<int>(static_cast<float>(n) * inverse);
    q -= q * d > n;
    return q + (n - q * d >= d);
}
template <int HELD>
__device__ __forceinline__ bool find_piece(const Attn4Args& a, int item, Piece& p) {
    const int lane = threadIdx.x & 63;
    auto lane_request = [&](int b) { return b < a.requests ? request(a, b) : Request4{0, 0, 0, false}; };
    // The requests' numbers, all loads of a lane in flight together.
    int start[HELD], end[HELD], len[HELD];
    auto load = [&](int c) {
        const int b = min(c * kWave + lane, a.requests - 1);
        start[c] = a.row_start[b];
        end[c] = a.row_start[b + 1];
        len[c] = a.kv_len[b];
    };
#pragma unroll
    for (int c = 0; c < HELD; ++c)
        if (c * kWave < a.requests) load(c);
    float units[HELD];
    int tiles[HELD];
    uint32_t large = 0;
    Weight weight;
#pragma unroll
    for (int c = 0; c < HELD; ++c) {
        units[c] = 0.f;
        tiles[c] = 0;
        if (c * kWave < a.requests) {
            const Request4 r = c * kWave + lane < a.requests ? request_of(a, start[c], end[c], len[c]) : Request4{0, 0, 0, false};
            units[c] = units_of(a, r);
            tiles[c] = tiles_of(r);
            large |= is_small(a, r) ? 0u : 1u << c;
            weight.add(a, r);
        }
    }
    if (!a.split_all)
        for (int b = HELD * kWave + lane; b < a.requests; b += kWave) weight.add(a, request(a, b));
    const bool light = a.light || (!a.split_all && weight.light(a));
    auto units_here = [&](const Request4& r) { return light || is_small(a, r) ? units_of(a, r) : 0.f; };
#pragma unroll
    for (int c = 0; c < HELD; ++c)
        if (((large >> c) & 1) && !light) units[c] = 0.f;
    auto sum = [&](auto&& of) {   // rounded, but the same in every wave
        float v = 0.f;
#pragma unroll
        for (int c = 0; c < HELD; ++c)
            if (c * kWave < a.requests) v += of(units[c], static_cast<float>(tiles[c]));
        for (int b = HELD * kWave + lane; b < a.requests; b += kWave) {
            const Request4 r = request(a, b);
            v += of(units_here(r), static_cast<float>(tiles_of(r)));
        }
        return group_sum<kWave>(v);
    };
    int cut = 1 << 26;
    float step = 0x1p-26f;
    if (!a.whole) {
        const float total = sum([](float u, float t) { return u * t; }), all_units = sum([](float u, float) { return u; });
        const bool many = all_units > static_cast<float>(a.places);
        const float want = static_cast<float>(a.places) * (many ? 4.0f : 1.0f);
        const float per_want = __builtin_amdgcn_rcpf(want);
        auto limited = [](float t) {   // whole turns
            return max(static_cast<int>(fminf(ceilf(t * (1.0f / kSplitWaves)), 0x1p24f)), 1) * kSplitWaves;
        };
        cut = limited(total * per_want);
        step = __builtin_amdgcn_rcpf(static_cast<float>(cut));
        for (int i = 0; i < 3; ++i) {
            const float pieces = sum([=](float u, float t) { return u * ceilf(t * step * 0.99999f); });   // (step may be an ulp high)
            if (pieces <= want) break;
            cut = max(limited(static_cast<float>(cut) * pieces * per_want), cut + kSplitWaves);
            step = __builtin_amdgcn_rcpf(static_cast<float>(cut));
        }
        cut = __builtin_amdgcn_readfirstlane(cut);
        if (light && many) {   // whole units: the workspace has no places for more pieces
            cut = 1 << 26;
            step = 0x1p-26f;
        }
    }
    bool found = false;
    auto look = [&](int b0, float u, int t) {
        const int splits = quotient(t + cut - 1, cut, step);
        const int n = static_cast<int>(fminf(u * static_cast<float>(splits), static_cast<float>(kMaxItems)));
        const int upto = wave_prefix(n);
        const uint64_t hit = __ballot(item < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int local = item - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
            p.b = b0 + l;
            p.splits = __builtin_amdgcn_readlane(splits, l);
            p.unit = __builtin_amdgcn_readfirstlane(quotient(local, p.splits, __builtin_amdgcn_rcpf(static_cast<float>(p.splits))));
            p.split = local - p.unit * p.splits;
            const int turns = (__builtin_amdgcn_readlane(t, l) + kSplitWaves - 1) / kSplitWaves;
            const float per_split = __builtin_amdgcn_rcpf(static_cast<float>(p.splits));
            p.tiles = p.splits == 1 ? 1 << 26 : quotient(turns + p.splits - 1, p.splits, per_split) * kSplitWaves;
            p.r = b0 == 0 ? request_of(a, __builtin_amdgcn_readlane(start[0], l), __builtin_amdgcn_readlane(end[0], l),
                                       __builtin_amdgcn_readlane(len[0], l))
                          : request(a, p.b);
            found = true;
        } else {
            item -= __builtin_amdgcn_readlane(upto, 63);
        }
    };
#pragma unroll
    for (int c = 0; c < HELD; ++c)
        if (!found && c * kWave < a.requests) look(c * kWave, units[c], tiles[c]);
    for (int b0 = HELD * kWave; !found && b0 < a.requests; b0 += kWave) {
        const Request4 r = lane_request(b0 + lane);
        look(b0, units_here(r), tiles_of(r));
    }
    return found;
}

// ------------------------------------------------------------------ codes and numbers
// A word's 8 codes as the fp16 operand, the even ones less EVEN, the odd ones less ODD. `magic` is 0x64006400 from a vector
// register: v_and_or_b32 takes one constant only, and the compiler makes two instructions of a mask and a literal.
__device__ __forceinline__ uint32_t code_magic() {
    uint32_t m = 0x64006400u;
    asm("" : "+v"(m));
    return m;
}
template <int EVEN, int ODD = EVEN>
__device__ __forceinline__ f16x8_t codes8(uint32_t w, uint32_t magic) {
    const f16x2_t down = {(_Float16)(-1024.0f - EVEN), (_Float16)(-1024.0f - ODD)};
    const f16x2_t sixteenth = {(_Float16)0.0625f, (_Float16)0.0625f};
    const f16x2_t down16 = {(_Float16)(-64.0f - EVEN), (_Float16)(-64.0f - ODD)};
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t x = i & 2 ? w >> 8 : w;
        f16x2_t h;
        if (i & 1)
            h = __builtin_elementwise_fma(__builtin_bit_cast(f16x2_t, (x & 0x00f000f0u) | magic), sixteenth, down16);
        else
            h = __builtin_bit_cast(f16x2_t, (x & 0x000f000fu) | magic) + down;
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
// Two values' high parts as a word, and the rest of one of them behind its high part: exact, and in one instruction, which takes
// the half number as it lies in the word. (The compiler turns that fma to a conversion of its own and a subtraction.)
__device__ __forceinline__ uint32_t high_parts(float a, float b) {
    const f16x2_t h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, h);
}
template <int HALF>
__device__ __forceinline__ float rest_of(uint32_t high, float v) {
    float r;
    if constexpr (HALF == 0)
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(high), "v"(v));
    else
        asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(high), "v"(v));
    return r;
}
// v less its own fp16 part, exact
__device__ __forceinline__ float low_part(float v) { return __builtin_fmaf(static_cast<float>(static_cast<_Float16>(v)), -1.0f, v); }
__device__ __forceinline__ float bf16_part(float v, int part) {   // bf16 part 0, 1, 2 of v, as an fp32 number
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float r = static_cast<float>(static_cast<__bf16>(v));
        if (part == i) return r;
        v -= r;
    }
    return static_cast<float>(static_cast<__bf16>(v));
}
// A sum of thousands of tiles' sums, and what its additions have rounded away. Where a row's weights are all the same, each of them
// rounds the same way: token by token and without the second number, rows of 12000 equal weights were 5e-5 off and of 40000 4e-4.
// (It costs the prompts' kernel 1.3%.)
struct Sum {
    float high = 0.f, rest = 0.f;
    __device__ __forceinline__ void add(float v) {
        const float t = high + v;
        rest += v - (t - high);   // exact while |v| <= |high|
        high = t;
    }
    __device__ __forceinline__ void scale(float f) {
        high *= f;
        rest *= f;
    }
    __device__ __forceinline__ float value() const { return high + rest; }
};
// The largest over the 8 lanes that share a row: its two columns, four lane groups.
__device__ __forceinline__ float max_over_row(float v) {
    v = fmaxf(v, dpp_move<0xB1>(v));
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}
// Two tokens' sizes max(16 scale, |min|, 2^-40) as bf16 bits, from their scales and minima.
__device__ __forceinline__ uint32_t sizes2(uint32_t scale, uint32_t low) {
    const u16x2_t s = __builtin_bit_cast(u16x2_t, scale) + u16x2_t{0x0200, 0x0200};
    const u16x2_t m = __builtin_bit_cast(u16x2_t, low & 0x7fff7fffu);
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_elementwise_max(s, m), u16x2_t{0x2b80, 0x2b80}));
}
// score + log2(size) + 127
__device__ __forceinline__ float log2_over(float score, uint32_t b) { return __builtin_fmaf(static_cast<float>(b), 0x1p-7f, score); }

// v / (1 + e^-x). Below kFarGate, where e^-x leaves the range, e^x as the square of e^(x/2): subnormal results too. Without a
// branch a value, with which the prompts' outputs took 4500 instructions a wave.
constexpr float kFarGate = -80.0f;
__device__ __forceinline__ float near_gated(float v, float x) {
    return v * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-x * kLog2e));
}
__device__ __forceinline__ float gated_by(float v, float x) {
    const float t = __builtin_amdgcn_exp2f(x * (0.5f * kLog2e));
    return x < kFarGate ? v * (t * t) : near_gated(v, x);
}
// An output from its sums: zero where no key was seen (a weight may be 0 beside a NaN).
__device__ __forceinline__ float finished(float m, float sum, float tot, bool gated, float gate) {
    const float v = m == -FLT_MAX && tot == 0.f ? 0.f : sum / tot;
    return gated ? gated_by(v, gate) : v;
}
// 2, 4 or 8 neighbouring floats, as aligned as they are many
template <int N>
__device__ __forceinline__ void load_floats(const float* p, float (&x)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const float4 y = ld4(p + i);
            x[i] = y.x, x[i + 1] = y.y, x[i + 2] = y.z, x[i + 3] = y.w;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = p[i];
    }
}
template <int N>
__device__ __forceinline__ void store_floats(float* p, const float (&x)[N]) {
    if constexpr (N >= 4) {
#pragma unroll
        for (int i = 0; i < N; i += 4) st4(p + i, make_float4(x[i], x[i + 1], x[i + 2], x[i + 3]));
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) p[i] = x[i];
    }
}

// ------------------------------------------------------------------ few rows
// Bound by bytes and by vector instructions about alike: at 200000 keys the cache comes at 3.9 TB/s (5.8 more keys added to a long
// call), and 600 instructions a tile and wave, 290 of them from codes to fp16 numbers, take 15 of the 29 us.
// A workgroup takes 8 (row, head) pairs that share a KV head - 16 columns: 8 rows x 2 fp16 parts - and a range of 32-token
// tiles, its NW waves every NW-th tile. A wave's tiles go straight from the cache to a ring of two places in LDS (no
// registers wait for them), the next but one requested as soon as a tile has been taken to registers: one and a half tiles,
// 13 KB at D = 256, are under way per wave. The two columns of a row share the work of the softmax: each of the two lanes takes
// half of the tokens that both hold.
// WIDE: pages of 32 tokens and more, so that a tile lies in one page.
//
// A tile's place: keys, values, then k_scale, k_min, v_scale, v_min, each with its tokens in order. The keys' 16-byte pieces
// are exchanged within a token's row (piece q of token t lies where q ^ key_turn(t) would), so that the 8 lanes that LDS
// serves at once, which read one piece of 8 rows, meet no bank twice.
template <int D>
struct Ring {
    static constexpr int NG = D / 64;
    static constexpr int keys = 32 * D / 2, values = 32 * D / 2, scales = 32 * 2 * NG;   // bytes
    static constexpr int at_ks = keys + values, at_km = at_ks + scales, at_vs = at_km + scales, at_vm = at_vs + 64;
    static constexpr int bytes = at_vm + 64;
    static constexpr int pieces = keys / 1024;              // loads of 1 KB for the keys, and for the values
    static constexpr int loads = 2 * pieces + 1;            // of a tile
    static constexpr int small_lanes = (bytes - at_ks) / 16;
};
template <int D>
__device__ __forceinline__ int key_turn(int t) {
    if constexpr (D == 256) return (t & 3) | ((t >> 1) & 4);
    if constexpr (D == 128) return ((t >> 1) & 1) | ((t >> 2) & 2);
    return (t >> 3) & 1;
}

template <int D, bool WIDE, int NW>
__global__ __launch_bounds__(NW* kWave, 2) void split4_kernel(const Attn4Args a) {
    constexpr int NG = D / 64, NV = D / 64, LD = D + 4;   // rows of sums: 16-byte aligned
    constexpr int QL = kWave * NW / kRows, QN = D / QL;   // threads of a row, in its query and in its output, and their dims
    using R = Ring<D>;
    static_assert(kRows * LD * 4 <= 2 * R::bytes, "a wave's sums go where its ring was");
    __shared__ __align__(16) uint8_t ring[NW][2][R::bytes];
    __shared__ __align__(16) _Float16 qs[2 * kRows][D + 8];   // the queries' parts; 16 bytes more, and 16 rows meet no bank twice
    __shared__ float2 stat[NW][kRows];
    __shared__ float factors[kRows], qsum[kRows][NG];
    Piece pc;
    const int item = static_cast<int>(blockIdx.x);
    if (!(a.requests <= kWave       ? find_piece<1>(a, item, pc)
          : a.requests <= 4 * kWave ? find_piece<4>(a, item, pc)
                                    : find_piece<16>(a, item, pc)))
        return;   // the whole workgroup
    const Request4 r = of_lane(pc.r, 0);
    pc.b = __builtin_amdgcn_readfirstlane(pc.b);
    pc.unit = __builtin_amdgcn_readfirstlane(pc.unit);
    pc.split = __builtin_amdgcn_readfirstlane(pc.split);
    pc.tiles = __builtin_amdgcn_readfirstlane(pc.tiles);
    const int G = a.group, pairs = r.n * G;
    const float per_g = __builtin_amdgcn_rcpf(static_cast<float>(G));
    auto over_g = [&](int pair) { return quotient(pair, G, per_g); };
    const int blocks = (pairs + kRows - 1) / kRows;
    const int h = __builtin_amdgcn_readfirstlane(quotient(pc.unit, blocks, __builtin_amdgcn_rcpf(static_cast<float>(blocks))));
    const int rb = pc.unit - h * blocks;
    const int lane = threadIdx.x & 63, lr = lane & 15, lk = lane >> 4, part = lr & 1;
    const int wv = wave_in_block();
    const uint32_t magic = code_magic();
    const int limit = r.len - r.n + over_g(min(rb * kRows + (lr >> 1), pairs - 1));   // this column's last key; columns past
                                                                                      // the last pair repeat it
    const int first_limit = r.len - r.n + over_g(rb * kRows);    // the smallest of the workgroup
    const int seen = max(r.len - r.n + over_g(min(rb * kRows + kRows - 1, pairs - 1)) + 1, 0);   // keys that some column sees
    const int t_end = __builtin_amdgcn_readfirstlane(min((pc.split + 1) * pc.tiles, (seen + kTile - 1) / kTile));
    int t = pc.split * pc.tiles + wv;
    const int P = a.c.page;

    // The pages of a tile's octets of tokens, requested a tile before they are needed. Octets that no row sees are read from
    // page 0, a page id outside the cache is not followed.
    constexpr int OCT = WIDE ? 1 : 4;
    const int32_t* row_table = a.table + static_cast<size_t>(pc.b) * a.max_pages;
    int ids[OCT];
    auto request_ids = [&](int tile) {
#pragma unroll
        for (int j = 0; j < OCT; ++j) {
            const int tok = tile * kTile + 8 * j;
            ids[j] = tile < t_end && tok < seen ? row_table[tok >> a.page_shift] : 0;   // below max_pages since tok < seen
        }
    };
    uint32_t bad_octets[2] = {0, 0};   // of the tiles in the ring
    const uint32_t ring_at = lds_address(&ring[wv][0][0]);
    // A lane's part of the keys: token L / PR of a load, 16-byte piece L % PR of its row, exchanged; as offset in its octet.
    constexpr int PR = D / 32;   // pieces of a row
    const int ktok = lane / PR;
    const uint32_t koff = (ktok & 7) * (D / 2) + 16 * ((lane % PR) ^ key_turn<D>(ktok)), voff = 16 * (lane % (D / 4));
    const int lane_oct = lane / (D / 4);   // the octet that a lane has in a load, after the first of the load
    // and of the rest: NG pieces of an octet's key scales, as many of its minima, one each of the values'
    const uint8_t* small_base;
    int small_oct, small_mul;
    uint32_t small_off;
    {
        const int s = lane < 8 * NG ? lane % (4 * NG) : lane & 3, big = lane < 8 * NG;
        small_base = reinterpret_cast<const uint8_t*>(lane < 4 * NG ? a.c.ks : big ? a.c.km : lane < 8 * NG + 4 ? a.c.vs : a.c.vm);
        small_oct = big ? s / NG : s;
        small_mul = big ? 2 * NG : 2;
        small_off = big ? 16 * (s % NG) : 0;
    }
    auto request_tile = [&](int tile, int slot) {   // from `ids`; for tile < t_end
        size_t at[OCT];   // the octets' first tokens, in the head's cache
        uint32_t bad = 0;
#pragma unroll
        for (int j = 0; j < OCT; ++j) {
            const bool b = static_cast<uint32_t>(ids[j]) >= static_cast<uint32_t>(a.c.pages);
            bad |= b ? (WIDE ? 15u : 1u << j) : 0u;
            at[j] = (static_cast<size_t>(b ? 0u : static_cast<uint32_t>(ids[j])) * a.c.heads + h) * P +
                    ((tile * kTile + 8 * j) & (P - 1));
        }
        bad_octets[slot] = bad;
        auto octet = [&](int j) {   // for a lane
            if constexpr (WIDE) return at[0] + 8 * j;
            else return j == 0 ? at[0] : j == 1 ? at[1] : j == 2 ? at[2] : at[3];
        };
        const uint32_t to = ring_at + slot * R::bytes;
#pragma unroll
        for (int i = 0; i < R::pieces; ++i) {
            constexpr int per = 4 / R::pieces;   // octets of a load
            if constexpr (WIDE || per == 1) {
                const size_t base = (WIDE ? at[0] + 8 * per * i : at[WIDE ? 0 : i]) * (D / 2);
                const uint32_t turn = D == 256 ? 64 * (i & 1) : 0;   // key_turn's bit of the octet
                dma16((koff ^ turn) + lane_oct * (4 * D), a.c.k + base, to + 1024 * i);
                dma16(voff + lane_oct * (4 * D), a.c.v + base, to + R::keys + 1024 * i);
            } else {
                const size_t base = octet(per * i + lane_oct) * (D / 2);
                dma16(a.c.k + base + koff, to + 1024 * i);
                dma16(a.c.v + base + voff, to + R::keys + 1024 * i);
            }
        }
        if (lane < R::small_lanes) dma16(small_base + octet(small_oct) * small_mul + small_off, to + R::at_ks);
    };
    // The rows' queries, scaled by 2^e so that a row's largest magnitude is in [2^14, 2^15), as two fp16 parts: requested
    // before the first tile.
    const int qr = static_cast<int>(threadIdx.x) / QL, qp = min(rb * kRows + qr, pairs - 1), qt = over_g(qp);
    const float* qrow = a.q + (static_cast<size_t>(r.first + qt) * a.heads + h * G + (qp - qt * G)) * D + (threadIdx.x % QL) * QN;
    float qf[QN];
    load_floats(qrow, qf);
    request_ids(t);
#pragma unroll
    for (int i = 0; i < QN; ++i) asm volatile("" : "+v"(qf[i]));   // here: behind the tile's loads it would wait for those too
    if (t < t_end) request_tile(t, 0);
    request_ids(t + NW);
    {
        float m = 0.f;
        bool bad = false;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            m = fmaxf(m, fabsf(qf[i]));
            bad |= !(fabsf(qf[i]) <= FLT_MAX);
        }
        if (bad) m = INFINITY;
        m = fmaxf(m, dpp_move<0xB1>(m));   // over the row's lanes
        m = fmaxf(m, dpp_move<0x4E>(m));
        m = fmaxf(m, dpp_move<0x141>(m));
        m = fmaxf(m, dpp_move<0x140>(m));
        const auto two = __builtin_amdgcn_permlane16_swap(__float_as_uint(m), __float_as_uint(m), false, false);
        m = fmaxf(__uint_as_float(two[0]), __uint_as_float(two[1]));
        if constexpr (QL == 64) {
            const auto halves = __builtin_amdgcn_permlane32_swap(__float_as_uint(m), __float_as_uint(m), false, false);
            m = fmaxf(__uint_as_float(halves[0]), __uint_as_float(halves[1]));
        }
        const bool ok = m <= FLT_MAX;
        int e = 0;
        if (m > 0.f && ok) {
            int em;
            frexpf(m, &em);
            e = min(15 - em, kMaxUp);
        }
        float s = 0.f;
        const int d0 = (threadIdx.x % QL) * QN;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const float v = ok ? ldexpf(qf[i], e) : 0.f;
            s += v;
            qs[2 * qr][d0 + i] = static_cast<_Float16>(v);
            qs[2 * qr + 1][d0 + i] = static_cast<_Float16>(low_part(v));
        }
        s = group_sum<64 / QN>(s);
        if ((lane & (64 / QN - 1)) == 0) qsum[qr][d0 / 64] = s;
        if (d0 == 0) factors[qr] = ok ? ldexpf(a.scale, -e) : __builtin_nanf("");   // products to log2 scores; NaN: a row
    }                                                                                        // with infinities or NaNs
    if (t + NW < t_end) request_tile(t + NW, 1);
    request_ids(t + 2 * NW);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the tiles' loads stay in flight
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
    float mu = -FLT_MAX;   // the reference less kWeightUp
    Sum sum_l, sum_low;
    const int my_turn = key_turn<D>(8 * (lr >> 2) + (lr & 3));
    const uint32_t k_at = (8 * (lr >> 2) + (lr & 3)) * (D / 2);
    for (int slot = 0; t < t_end; t += NW, slot ^= 1) {
        if (t + NW < t_end)
            wait_vm<R::loads>();   // the next tile stays under way
        else
            wait_vm<0>();
        asm volatile("" ::: "memory");
        const uint8_t* in = ring[wv][slot];
        constexpr int KW = NG * 2;   // words of a lane's share of a token's keys
        uint32_t K[2][KW];
        uint4 V[NV], ksc[NG];
        bf16x8_t kmn[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const uint8_t* p = in + k_at + x * (4 * D / 2);
            if constexpr (KW == 8) {
                const uint4 u = ld16(p + 16 * ((2 * lk) ^ my_turn)), v = ld16(p + 16 * ((2 * lk + 1) ^ my_turn));
                K[x][0] = u.x, K[x][1] = u.y, K[x][2] = u.z, K[x][3] = u.w;
                K[x][4] = v.x, K[x][5] = v.y, K[x][6] = v.z, K[x][7] = v.w;
            } else if constexpr (KW == 4) {
                const uint4 u = ld16(p + 16 * (lk ^ my_turn));
                K[x][0] = u.x, K[x][1] = u.y, K[x][2] = u.z, K[x][3] = u.w;
            } else {
                const uint2 u = *reinterpret_cast<const uint2*>(p + 16 * ((lk >> 1) ^ my_turn) + 8 * (lk & 1));
                K[x][0] = u.x, K[x][1] = u.y;
            }
            const uint8_t* m = in + R::at_km + (8 * (lr >> 2) + 4 * x + (lr & 3)) * (2 * NG);
            u32x4_t z = {0u, 0u, 0u, 0u};
            if constexpr (NG == 4) {
                const uint2 u = *reinterpret_cast<const uint2*>(m);
                z[0] = u.x, z[1] = u.y;
            } else if constexpr (NG == 2) {
                z[0] = *reinterpret_cast<const uint32_t*>(m);
            } else {
                z[0] = *reinterpret_cast<const uint16_t*>(m);
            }
            kmn[x] = __builtin_bit_cast(bf16x8_t, z);
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) ksc[g] = ld16(in + R::at_ks + lk * (16 * NG) + 16 * g);
        f32x4_t S[2];
        const f32x4_t zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int x = 0; x < 2; ++x) S[x] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kmn[x], Qs, zero, 0, 0, 0);
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint32_t w[4] = {ksc[g].x, ksc[g].y, ksc[g].z, ksc[g].w};
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                f32x4_t T = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<0>(K[x][2 * g], magic), Q[2 * g], zero, 0, 0, 0);
                T = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<0>(K[x][2 * g + 1], magic), Q[2 * g + 1], T, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    S[x][i] = __builtin_fmaf(T[i], i & 1 ? bf16_hi(w[2 * x + (i >> 1)]) : bf16_lo(w[2 * x + (i >> 1)]), S[x][i]);
            }
        }
#pragma unroll
        for (int m = 0; m < NV; ++m) V[m] = ld16(in + R::keys + lk * (4 * D) + 256 * m + 16 * lr);
        const uint2 vsc = *reinterpret_cast<const uint2*>(in + R::at_vs + 16 * lk + 8 * part);
        const uint2 vmn = *reinterpret_cast<const uint2*>(in + R::at_vm + 16 * lk + 8 * part);
        const float f = (bad_octets[slot] >> lk) & 1 ? __builtin_nanf("") : factor;
        if (t + 2 * NW < t_end) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the place has been read
            request_tile(t + 2 * NW, slot);
            request_ids(t + 3 * NW);
        }
        // This lane's tokens 8 lk + 4 part + 0..3: both fp16 parts of the query, the other one from the lane beside.
        const int tok = t * kTile + 8 * lk + 4 * part;
        float s[4], sv[4], mv[4];
        const uint32_t vs[2] = {vsc.x, vsc.y}, vm[2] = {vmn.x, vmn.y};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float mine = part ? S[1][i] : S[0][i], other = part ? S[0][i] : S[1][i];
            s[i] = (mine + dpp_move<0xB1>(other)) * f;
            sv[i] = i & 1 ? bf16_hi(vs[i >> 1]) : bf16_lo(vs[i >> 1]);
            mv[i] = __builtin_fmaf(i & 1 ? kOddLess : kEvenLess, sv[i], i & 1 ? bf16_hi(vm[i >> 1]) : bf16_lo(vm[i >> 1]));
        }
        if (t * kTile + kTile - 1 > first_limit) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (tok + i > limit) {   // what lies there is anything: no 0 * NaN
                    s[i] = -INFINITY;
                    sv[i] = mv[i] = 0.f;
                }
        }
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const uint32_t z = sizes2(vs[i >> 1], vm[i >> 1]);
            top = fmaxf(top, fmaxf(log2_over(s[i], z & 0xffffu), log2_over(s[i + 1], z >> 16)));
        }
        top -= 127.0f + kWeightUp;
        if (__ballot(top > mu + kMoves)) {
            const float now = fmaxf(mu, max_over_row(top));
            const float shrink = __builtin_amdgcn_exp2f(mu - now);
            mu = now;
            sum_l.scale(shrink);
            sum_low.scale(shrink);
#pragma unroll
            for (int m = 0; m < NV; ++m)
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][e][i] *= shrink;
        }
        uint32_t high[2], rest[2];
        float w0 = 0.f, tile_l = 0.f, tile_low = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] - mu);
            tile_l = i == 0 ? p : tile_l + p;
            tile_low = i == 0 ? p * mv[0] : __builtin_fmaf(p, mv[i], tile_low);
            const float w = rounded(p * sv[i]);
            if (i & 1) {
                high[i >> 1] = high_parts(w0, w);
                rest[i >> 1] = high_parts(rest_of<0>(high[i >> 1], w0), rest_of<1>(high[i >> 1], w));
            }
            w0 = w;
        }
        sum_l.add(tile_l);
        sum_low.add(tile_low);
        u32x4_t W;   // tokens 8 lk + 0..7 of this column's part: half of them from the lane beside
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t x = high[j], y = rest[j];
            const uint32_t got = __float_as_uint(dpp_move<0xB1>(__uint_as_float(part ? x : y)));
            W[j] = part ? got : x;
            W[2 + j] = part ? y : got;
        }
#pragma unroll
        for (int m = 0; m < NV; ++m) {
            const uint32_t w[4] = {V[m].x, V[m].y, V[m].z, V[m].w};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                acc[m][e] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8<kEvenLess, kOddLess>(w[e], magic), __builtin_bit_cast(f16x8_t, W),
                                                                   acc[m][e], 0, 0, 0);
        }
    }
    // The waves' sums meet in LDS; the two parts of a row are neighbouring columns, each lane of a pair writes every
    // other dim of both. Row 4 lk + i of value tile (m, e) is dim 64 m + 4 (4 lk + i) + e.
    float l = sum_l.value(), low = sum_low.value();
    l += dpp_move<0xB1>(l);
    low += dpp_move<0xB1>(low);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    low += __shfl_xor(low, 16);
    low += __shfl_xor(low, 32);
    float* mine = reinterpret_cast<float*>(ring[wv]) + (lr >> 1) * LD;   // the wave's loads have all come
#pragma unroll
    for (int m = 0; m < NV; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; e += 2) {
                const float u = acc[m][e][i] + dpp_move<0xB1>(acc[m][e][i]);
                const float v = acc[m][e + 1][i] + dpp_move<0xB1>(acc[m][e + 1][i]);
                mine[64 * m + 4 * (4 * lk + i) + e + part] = (part ? v : u) + low;
            }
    if (lane < 16 && part == 0) stat[wv][lr >> 1] = make_float2(mu, l);
    __syncthreads();
    const int row = static_cast<int>(threadIdx.x) / QL, d = (threadIdx.x % QL) * QN, at = rb * kRows + row;
    if (at >= pairs) return;
    float2 st[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) st[w] = stat[w][row];
    float m = st[0].x, tot = 0.f, sum[QN];
#pragma unroll
    for (int w = 1; w < NW; ++w) m = fmaxf(m, st[w].x);
#pragma unroll
    for (int i = 0; i < QN; ++i) sum[i] = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
        const float k = __builtin_amdgcn_exp2f(st[w].x - m);
        tot += k * st[w].y;
        const float* from = reinterpret_cast<const float*>(ring[w]) + row * LD + d;
        float x[QN];
        load_floats(from, x);
#pragma unroll
        for (int i = 0; i < QN; ++i) sum[i] += k * x[i];
    }
    if (r.bad) tot = __builtin_nanf("");
    const int n = over_g(at);
    const size_t pair = static_cast<size_t>(r.first + n) * a.heads + h * G + (at - n * G);
    const size_t o = pair * D + d, place = static_cast<size_t>(item) * kRows + row;
    if (pc.splits == 1) {
        float gate[QN];
        if (a.gate) load_floats(a.gate + o, gate);
#pragma unroll
        for (int i = 0; i < QN; ++i) sum[i] = finished(m, sum[i], tot, a.gate, a.gate ? gate[i] : 0.f);
        store_floats(a.out + o, sum);
    } else {
        store_floats(a.part + place * D + d, sum);
        if (d == 0) a.stat[place] = make_float2(m, tot);
    }
    if (d == 0 && pc.split == 0 && !a.whole) a.info[pair] = make_int2(static_cast<int>(place), pc.splits);
}

// ------------------------------------------------------------------ many rows
// Bound by instruction issue: of the 4990 cycles that a wave has a tile of 32 tokens, the matrix products take 2180 and its 430
// other vector instructions 1820. 128 rows a workgroup, 4 waves, one a SIMD, of 32 rows each, on v_mfma_f32_32x32x16_f16: codes are
// turned to fp16 once per workgroup, into LDS, and an operand of keys or values, 1 KB of LDS, feeds 2 products (both parts of
// 32 rows). A wave holds its rows' query parts (128 registers at D = 256, pinned in accumulation registers) and sums (128).
// Its vector work - softmax, turning codes to fp16 - is laid between its own products: while tile t + 1's scores are computed,
// tile t's are exponentiated; while tile t's values are summed, the codes of the next tiles go to LDS. All waves run all tiles
// of the workgroup, though a wave's own rows may end one earlier: with a branch around the products the compiler moves the sums
// between register files at each. (5000 rows by exponents for each 8 tokens in place of each token's 506 us, codes to LDS beside
// the scores 510, where this took 492; with the roundings of `Sum` and the values' middle 500.)
// The keys' scales are in the operand: code - 8 has at most 3 bits and a bf16 scale 8, so scale (code - 8) is an fp16 number, and
// all dims of a head are one sum. What is left of a key, min + 8 scale of each group times the sum of its queries, is two
// products more, of bf16 numbers (the minima, 8 scale) with the sums' three parts. A token's numbers are taken times a power of
// two that brings the largest max(16 scale, |min|) of its groups below 2^16; the scores are multiplied by its inverse. (Each
// group's products scaled by themselves, in fp32, took 64 fmas a lane and tile and 64 registers: 506 us where this took 490.)
// The scores^T tile has token rho = 8 b + 4 g + j of the 32 in register 4 b + j of lane half g; key row rho stands for token
// 16 (b / 2) + 8 g + 4 (b % 2) + j, so that a lane's registers 8 s .. 8 s + 7 are octet 2 s + g, its share of the second
// product's depth s.

// A workgroup has its CU to itself at D = 256 (registers). A unit (a row tile and a KV head) costs 20 us beside its tiles' 2.2 us
// each: its queries, the first tiles' way to the products, its outputs. How a call's units meet the CUs:
// - pieces: up to kPromptFill units, each cut in pieces of at most so many tiles that all pieces are at most kPromptFill;
// - a line: all units' tiles one after the other, kPromptCost more in front of each unit, cut in kPromptFill equal parts. A
//   workgroup takes its part's segments of units in turn. Of fewer than kPromptCut units, where a part is shorter than the
//   longest piece would be;
// - of more, a workgroup a unit, the longest first.
// (Every unit in the same number of pieces, as many as fit: 2048 rows 144 us where this took 124; 1100 rows 91 for 66; 777 behind
// 6000 keys 220 for 193. A cost of 5, 7 or 15 tiles in the line: 153, 134, 131 us where 10 took 124.)
struct Line {
    int over, parts, base, more;   // steps in front of a unit; the first `more` parts have base + 1 steps, the others base
    __device__ __forceinline__ Line(int over, int steps, int most) : over(over) {
        parts = __builtin_amdgcn_readfirstlane(min(most, steps));
        base = __builtin_amdgcn_readfirstlane(steps / max(parts, 1));
        more = __builtin_amdgcn_readfirstlane(steps - base * parts);
    }
    __device__ __forceinline__ int start(int i) const { return i * base + min(i, more); }
    __device__ __forceinline__ int part_of(int step) const {
        const int wide = more * (base + 1);
        return step < wide ? step / (base + 1) : more + (step - wide) / base;
    }
    // The pieces of a unit that starts at `at`.
    __device__ __forceinline__ int pieces(int at, int steps) const { return part_of(at + over + steps - 1) - part_of(at + over) + 1; }
};
constexpr int kPromptWaves = 4;
static_assert(kPromptRows == 32 * kPromptWaves, "32 rows a wave");
constexpr int kPromptMinTiles = 4;   // of a piece
constexpr int kPromptCut = 2 * kPromptFill;   // units that are still a line
constexpr int kPromptCost = 10;  // of a unit, in tiles
typedef float f32x16_t __attribute__((ext_vector_type(16)));

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

template <int D>
__global__ __launch_bounds__(kPromptWaves* kWave, 1) void prompt4_kernel(const Attn4Args a) {
    constexpr int ND = D / 16, DT = D / 32, NG = D / 64, E = D / 64, NTH = kPromptWaves * kWave;   // E: a lane's words of a tile's
    constexpr int GL = D == 256 ? 2 : 1;                                                           // keys, and of its values;
    __shared__ __align__(16) f16x8_t ks[2][ND][kWave];                                             // GL: groups of those words
    __shared__ __align__(16) f16x8_t vs[2][DT][2][kWave];
    __shared__ __align__(16) uint16_t kmin[4][kTile][8];   // [tile % 4][key row]: bf16, the groups' minima (4) and 8 scale (4)
    __shared__ __align__(16) float outs[kPromptWaves][32][64 + 4];   // a wave's rows, 64 dims; 4 more, and 8 rows meet no bank twice
    __shared__ int2 out_rows[kPromptWaves][32];            // what a row's sums are taken times, where they go (-1: nowhere)
    __shared__ __align__(16) float tok[4][4][kTile];       // [tile % 4][key factor, value scale, min + 8 or 7 scale, log2 size][token]
    // which request, KV head and row tile: the last row tiles (the longest rows) first
    const int G = a.group;
    const float per_g = 1.0f / static_cast<float>(G);
    auto over_g = [&](int pair) { return quotient(pair, G, per_g); };
    auto row_tiles = [&](const Request4& r) { return is_small(a, r) ? 0 : (r.n * G + kPromptRows - 1) / kPromptRows; };
    auto keys_seen = [&](const Request4& r, int rt) {   // by some row of a row tile
        return max(r.len - r.n + over_g(min(rt * kPromptRows + kPromptRows - 1, r.n * G - 1)) + 1, 0);
    };
    const int step_bits = __builtin_ctz(a.prompt_step);
    auto steps_of = [&](int seen) { return max(1, (seen + kTile * a.prompt_step - 1) >> (5 + step_bits)); };
    auto lane_request = [&](int b) { return b < a.requests ? request(a, b) : Request4{0, 0, 0, false}; };
    const int lane0 = threadIdx.x & 63;
    const Request4 held = lane_request(lane0);   // every look is at these first
    float units = static_cast<float>(row_tiles(held)) * static_cast<float>(a.c.heads);
    Weight weight;
    weight.add(a, held);
    for (int b0 = kWave; b0 < a.requests; b0 += kWave) {
        const Request4 q = lane_request(b0 + lane0);
        units += static_cast<float>(row_tiles(q)) * static_cast<float>(a.c.heads);
        weight.add(a, q);
    }
    units = group_sum<kWave>(units);
    if (units == 0.f || weight.light(a)) return;   // the whole workgroup
    const bool cut = units < static_cast<float>(kPromptCut);
    Line line(0, 1, 1);
    int cut_at = 0;   // steps of a piece at most; 0: not in pieces
    int line_at = 0, line_end = 1;
    int b = 0, unit = 0, unit_steps = 1, unit_at = 0;   // unit_at: where the line has it
    Request4 r{0, 0, 0, false};
    {
        bool found = false;
        if (cut) {
            // `of`: what a unit of so many steps counts. Of lane's request q, all its units together: the row tiles one after the
            // other, or, where that is less, request by request with a lane a row tile.
            auto here = [&](const Request4& q, int k, auto&& of) {   // the units of row tile k, the longest first
                const int n = row_tiles(q);
                return k < n ? of(steps_of(keys_seen(q, n - 1 - k))) * a.c.heads : 0;
            };
            auto looks = [&](const Request4& q) {   // of the first way, and of the other
                return make_int2(wave_max(row_tiles(q)), wave_total((row_tiles(q) + kWave - 1) / kWave));
            };
            const int2 held_looks = looks(held);
            auto of_request = [&](const Request4& q, int2 ways, auto&& of) {
                const int n = row_tiles(q);
                int v = 0;
                if (ways.y < ways.x) {
                    for (uint64_t hit = __ballot(n > 0); hit; hit &= hit - 1) {
                        const int l = __builtin_ctzll(hit);
                        const Request4 one = of_lane(q, l);
                        int sum = 0;
                        for (int k0 = 0; k0 < row_tiles(one); k0 += kWave) sum += wave_total(here(one, k0 + lane0, of));
                        if (lane0 == l) v = sum;
                    }
                } else {
                    for (int k = 0; k < ways.x; ++k) v += here(q, k, of);
                }
                return v;
            };
            auto all = [&](auto&& of) {
                int v = of_request(held, held_looks, of);
                for (int b0 = kWave; b0 < a.requests; b0 += kWave) {
                    const Request4 q = lane_request(b0 + lane0);
                    v += of_request(q, looks(q), of);
                }
                return wave_total(v);
            };
            auto longest_of = [&](const Request4& q) { return row_tiles(q) ? steps_of(keys_seen(q, row_tiles(q) - 1)) : 0; };
            int longest = longest_of(held);
            for (int b0 = kWave; b0 < a.requests; b0 += kWave) longest = max(longest, longest_of(lane_request(b0 + lane0)));
            longest = wave_max(longest);
            const int steps = all([](int t) { return t; });
            int pieces = kPromptFill + 1;
            auto pieces_of = [&](int t) { return quotient(t + cut_at - 1, cut_at, __builtin_amdgcn_rcpf(static_cast<float>(cut_at))); };
            if (units <= static_cast<float>(kPromptFill)) {
                cut_at = max((steps + kPromptFill - 1) / kPromptFill, (kPromptMinTiles + a.prompt_step - 1) >> step_bits);
                for (int i = 0; i < 4; ++i) {
                    pieces = all(pieces_of);
                    if (pieces <= kPromptFill) break;
                    const float longer = static_cast<float>(cut_at) * static_cast<float>(pieces) * (1.0f / kPromptFill);
                    cut_at = max(static_cast<int>(longer), cut_at + 1);
                }
                if (pieces > kPromptFill) {
                    cut_at = longest;
                    pieces = static_cast<int>(units);
                }
            }
            const int cost = max(kPromptCost >> step_bits, 1), in_line = steps + cost * static_cast<int>(units);
            if (pieces > kPromptFill || max(in_line / kPromptFill, kPromptMinTiles >> step_bits) < min(cut_at, longest)) cut_at = 0;
            line = cut_at ? Line(0, pieces, pieces) : Line(cost, in_line, kPromptFill);
            if (static_cast<int>(blockIdx.x) >= line.parts) return;   // the whole workgroup
            line_at = line.start(blockIdx.x);
            line_end = line.start(blockIdx.x + 1);
            int left = line_at;
            auto of = [&](int t) { return cut_at ? pieces_of(t) : t + line.over; };
            for (int b0 = 0; b0 < a.requests && !found; b0 += kWave) {
                const Request4 q = b0 ? lane_request(b0 + lane0) : held;
                const int n = of_request(q, b0 ? looks(q) : held_looks, of), upto = wave_prefix(n);
                const uint64_t hit = __ballot(left < upto);
                if (!hit) {
                    left -= __builtin_amdgcn_readlane(upto, 63);
                    continue;
                }
                const int l = __builtin_ctzll(hit);
                left -= __builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l);
                b = b0 + l;
                r = of_lane(q, l);
                for (int k0 = 0; k0 < row_tiles(r) && !found; k0 += kWave) {
                    const int m = here(r, k0 + lane0, of), last = wave_prefix(m);
                    const uint64_t in = __ballot(left < last);
                    if (!in) {
                        left -= __builtin_amdgcn_readlane(last, 63);
                        continue;
                    }
                    const int k = __builtin_ctzll(in), each = __builtin_amdgcn_readlane(m, k) / a.c.heads;
                    left -= __builtin_amdgcn_readlane(last, k) - __builtin_amdgcn_readlane(m, k);
                    const int head = left / each;
                    unit = (k0 + k) * a.c.heads + head;
                    unit_steps = each - line.over;
                    unit_at = line_at - (left - head * each);
                    found = true;
                }
            }
        } else {
            int left = blockIdx.x;
            for (int b0 = 0; b0 < a.requests && !found; b0 += kWave) {
                const Request4 q = b0 ? lane_request(b0 + lane0) : held;
                const int n = row_tiles(q) * a.c.heads, upto = wave_prefix(n);
                const uint64_t hit = __ballot(left < upto);
                if (hit) {
                    const int l = __builtin_ctzll(hit);
                    unit = left - (__builtin_amdgcn_readlane(upto, l) - __builtin_amdgcn_readlane(n, l));
                    b = b0 + l;
                    r = of_lane(q, l);
                    found = true;
                } else {
                    left -= __builtin_amdgcn_readlane(upto, 63);
                }
            }
        }
        if (!found) return;   // the whole workgroup
    }
    for (;;) {
        int tid = threadIdx.x;
        asm("" : "+v"(tid));   // what follows from it is not held from one segment to the next
        const int lane = tid & 63, col = lane & 31, g = lane >> 5;
        r = of_lane(r, 0);
        b = __builtin_amdgcn_readfirstlane(b);
        unit = __builtin_amdgcn_readfirstlane(unit);
        unit_at = __builtin_amdgcn_readfirstlane(unit_at);
        unit_steps = __builtin_amdgcn_readfirstlane(unit_steps);
        const int pairs = r.n * G, tiles = row_tiles(r);
        const int h = unit % a.c.heads, rt = tiles - 1 - unit / a.c.heads;
        const int wv = wave_in_block();
        const int row0 = rt * kPromptRows + 32 * wv;             // the wave's first pair
        const int rr = min(row0 + col, pairs - 1);
        const int ti = over_g(rr), head = h * G + (rr - ti * G);
        const int limit = r.len - r.n + ti;
        const int wave_first = r.len - r.n + over_g(min(row0, pairs - 1));
        const int seen = keys_seen(r, rt);
        const int all_steps = (seen + kTile - 1) / kTile;
        const int from = max(line_at - unit_at - line.over, 0), to = min(line_end - unit_at - line.over, unit_steps);
        if (to <= 0) return;   // the part ends before the unit's first step
        const bool begins = from == 0, whole = begins && to == unit_steps;
        const int step = (cut_at ? (steps_of(seen) + unit_steps - 1) / unit_steps : 1) * a.prompt_step;   // tiles
        const int first_tile = whole ? 0 : __builtin_amdgcn_readfirstlane(from * step);
        // this segment's tiles
        const int steps = __builtin_amdgcn_readfirstlane(whole ? all_steps : max(min(to * step, all_steps) - first_tile, 0));
        const uint32_t magic = code_magic();

        // A wave brings one octet of tokens of each tile: page and offset are the same for its lanes. A lane's words: of keys
        // (token lane % 8, words E (lane / 8) .. of its row), of values (dims E lane ..). Octets past the last are loaded from
        // page 0 and never read from LDS. Page ids are read a tile ahead of the codes they lead to.
        uint32_t kr[E], vr[E];
        // bf16, of token lane % 8: the key scales of the lane's words, value scale and minimum, and its element of the token's row of
        // kmin (the minimum of group lane / 8, from lane 32 on the scale of group lane / 8 - 4)
        uint32_t ksr[GL], vsr, vmr, own;
        const int piece = lane >> 3, own_group = piece & 3;
        const uint16_t* own_at = piece < 4 ? a.c.km + (lane & 7) * NG + min(own_group, NG - 1)
                                           : a.c.ks + 8 * min(own_group, NG - 1) + (lane & 7);
        bool sdead = false, sbad = false;
        int id = 0;
        size_t at[3];   // the octet in tiles st + 1, st + 2, st + 3: its first token in the head's cache
        auto words = [](const uint8_t* p, uint32_t(&w)[E]) {
            if constexpr (E == 4) {
                const uint4 x = ld16(p);
                w[0] = x.x, w[1] = x.y, w[2] = x.z, w[3] = x.w;
            } else if constexpr (E == 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(p);
                w[0] = x.x, w[1] = x.y;
            } else {
                w[0] = *reinterpret_cast<const uint32_t*>(p);
            }
        };
        auto next_id = [&](int st) {   // the table's entry for the octet (any in-bounds entry past the row's end)
            const int page = min((kTile * (first_tile + st) + 8 * wv) >> a.page_shift, a.max_pages - 1);
            id = a.table[static_cast<size_t>(b) * a.max_pages + page];
        };
        auto k_load = [&](int st) {
            const int tok = kTile * (first_tile + st) + 8 * wv, page = __builtin_amdgcn_readfirstlane(id);
            sdead = tok >= seen;
            sbad = !sdead && (page < 0 || page >= a.c.pages);
            at[0] = at[1];
            at[1] = at[2];
            at[2] = (static_cast<size_t>(static_cast<uint32_t>(sdead || sbad ? 0 : page)) * a.c.heads + h) * a.c.page +
                    static_cast<uint32_t>(tok & (a.c.page - 1));
            words(a.c.k + at[2] * (D / 2) + (lane & 7) * (D / 2) + (lane >> 3) * (4 * E), kr);
#pragma unroll
            for (int j = 0; j < GL; ++j) ksr[j] = a.c.ks[at[2] * NG + 8 * ((GL * piece + j) % NG) + (lane & 7)];
            own = own_at[at[2] * NG];
            vsr = a.c.vs[at[2] + (lane & 7)];
            vmr = a.c.vm[at[2] + (lane & 7)];
        };
        auto v_load = [&](int n) {   // n: how many tiles behind the keys
            words(a.c.v + at[2 - n] * (D / 2) + lane * (4 * E), vr);
        };
        const int ktok = 8 * wv + (lane & 7), rho = (ktok & 16) + 8 * ((ktok >> 2) & 1) + 4 * ((ktok >> 3) & 1) + (ktok & 3);
        // The token's power of two, over its 8 lanes, and the lane's scales with it.
        int up = 0;
        _Float16 scale16[GL];
        auto k_scale = [&]() {
            uint32_t z = own_group < NG ? (piece < 4 ? own & 0x7fffu : own + 0x0200u) : 0u;   // |min|, 16 scale
            z = max(z, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(z), 0x128, 0xF, 0xF, false)));   // row_ror 8
            const auto x = __builtin_amdgcn_permlane16_swap(z, z, false, false);
            z = max(x[0], x[1]);
            const auto y = __builtin_amdgcn_permlane32_swap(z, z, false, false);
            up = 142 - max(static_cast<int>(max(y[0], y[1]) >> 7), 20);
#pragma unroll
            for (int j = 0; j < GL; ++j) scale16[j] = static_cast<_Float16>(ldexpf(bf16_value(static_cast<uint16_t>(ksr[j])), up));
        };
        auto k_put = [&](int st, int j) {   // word E (lane / 8) + j of the token's row: its place among [4][NG][2]
            const int w = E * piece + j, dims = 4 * ((w % (2 * NG)) >> 1) + w / (2 * NG);
            const _Float16 f = scale16[GL == 2 ? j >> 1 : 0];
            ks[st & 1][dims][32 * (w & 1) + rho] = codes8<8>(kr[j], magic) * f16x8_t{f, f, f, f, f, f, f, f};
        };
        auto v_put = [&](int st, int j) {   // dim 32 E m + E row + j is row `row` of value tile E m + j
            vs[st & 1][E * g + j][wv >> 1][32 * (wv & 1) + col] = codes8<kEvenLess, kOddLess>(vr[j], magic);
        };
        auto s_put = [&](int st) {
            const float mine = own_group < NG ? ldexpf(bf16_value(static_cast<uint16_t>(own)), piece < 4 ? up : up + 3) : 0.f;
            kmin[st & 3][rho][piece] = static_cast<uint16_t>(__float_as_uint(mine) >> 16);
            if (lane < 8) {
                // A page outside the cache, or values that are not finite, make the token's scores NaN: of the rows that see it.
                float scale = bf16_value(static_cast<uint16_t>(vsr));
                float rest = __builtin_fmaf(lane & 1 ? kOddLess : kEvenLess, scale, bf16_value(static_cast<uint16_t>(vmr)));
                const bool bad = sbad || !(fabsf(rest) <= FLT_MAX);
                if (sdead || bad) scale = rest = 0.f;
                tok[st & 3][0][ktok] = bad ? __builtin_nanf("") : __uint_as_float(static_cast<uint32_t>(127 - up) << 23);
                tok[st & 3][1][ktok] = scale;
                tok[st & 3][2][ktok] = rest;
                tok[st & 3][3][ktok] = log2_over(0.f, sizes2(vsr, vmr) & 0xffffu) - (127.0f + kWeightUp);
            }
        };
        auto k_store = [&](int st) {
            k_scale();
#pragma unroll
            for (int j = 0; j < E; ++j) k_put(st, j);
            s_put(st);
        };
        auto barrier = []() {   // LDS is written and read; the loads stay in flight
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_s_barrier();
            asm volatile("" ::: "memory");
        };
        if (steps > 0) {
            next_id(0);
            at[1] = at[2] = 0;
            k_load(0);
            next_id(1);
            v_load(0);
        }
        // the row's query, times 2^e, in two parts: dims 16 d + 8 g + 0..7 of depth d; and its groups' sums in three bf16 parts:
        // depth 8 g + e has part g of group e % 4, in a second product part 2 + g
        f16x8_t Qh[ND], Ql[ND];
        bf16x8_t Qs[2];
        float factor;
        {
            const float* q = a.q + (static_cast<size_t>(r.first + ti) * a.heads + head) * D + 8 * g;
            float f[ND][8];   // all of it requested before the first is looked at
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const float4 x = ld4(q + 16 * d + 4 * i);
                    f[d][4 * i] = x.x, f[d][4 * i + 1] = x.y, f[d][4 * i + 2] = x.z, f[d][4 * i + 3] = x.w;
                }
            float m = 0.f, bad = 0.f;   // 0, or NaN with an infinity or NaN
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    m = fmaxf(m, fabsf(f[d][i]));
                    bad = __builtin_fmaf(f[d][i], 0.f, bad);
                }
            if (bad != 0.f) m = INFINITY;
            m = fmaxf(m, __shfl_xor(m, 32));
            const bool ok = m <= FLT_MAX;
            int e = 0;
            if (m > 0.f && ok) {
                int em;
                frexpf(m, &em);
                e = min(15 - em, kMaxUp);
            }
            float sum[4] = {0.f, 0.f, 0.f, 0.f};
            const float by = ldexpf(1.0f, e);   // what a row with infinities or NaNs gives here does not matter: factor is NaN
#pragma unroll
            for (int d = 0; d < ND; ++d) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float v = f[d][i] * by;
                    Qh[d][i] = static_cast<_Float16>(v);
                    Ql[d][i] = static_cast<_Float16>(low_part(v));
                    sum[d >> 2] += v;
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (i < NG) sum[i] += __shfl_xor(sum[i], 32);
                const float p0 = bf16_part(sum[i], 0), p1 = bf16_part(sum[i], 1), p2 = bf16_part(sum[i], 2);
                Qs[0][i] = Qs[0][4 + i] = static_cast<__bf16>(g ? p1 : p0);
                Qs[1][i] = Qs[1][4 + i] = static_cast<__bf16>(g ? 0.f : p2);
            }
            // A row that sees no key keeps a factor that is a number, for scores of -inf that it meets.
            factor = ok || limit < 0 ? ldexpf(a.scale, -e) : __builtin_nanf("");
#pragma unroll
            for (int d = 0; d < ND; ++d) {   // only products read them: accumulation registers, the others are full
                asm("" : "+a"(Qh[d]));
                asm("" : "+a"(Ql[d]));
            }
        }
        f32x16_t acc[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[d][i] = 0.f;
        float mu = -FLT_MAX;
        Sum l, low;
        float tile_l = 0.f, tile_low = 0.f;
        f32x16_t zero;
#pragma unroll
        for (int i = 0; i < 16; ++i) zero[i] = 0.f;
        f32x16_t S, N;          // a tile's scores over `factor`; the next tile's products
        u32x4_t Wh[2], Wl[2];   // weights of the last tile, pairs of fp16 numbers
        // the numbers of a lane's tokens 4 j .. 4 j + 3
        auto of_tokens = [&](const float* p, int j) { return ld4(p + 16 * (j >> 1) + 8 * g + 4 * (j & 1)); };
        // The operands of a step's products are one sequence, the last tile's values (2 DT of them), then the next tile's keys
        // (ND = 2 DT); each is requested AP products' pairs ahead, into the register that the one before it has left. fill(i) goes
        // between the two products of an operand and after them.
        constexpr int AP = 4;
        f16x8_t A[AP];
        auto value_at = [&](int slot, int k) { return vs[slot][k >> 1][k & 1][lane]; };
        auto key_at = [&](int slot, int d) { return ks[slot][d][lane]; };
        auto minima = [&](int tile) { return *reinterpret_cast<const bf16x8_t*>(&kmin[tile & 3][col][0]); };
        // A tile's products into N. ahead(d): what to request when operand d has been taken.
        auto scores = [&](const bf16x8_t mins, auto&& ahead, auto&& fill) {
            N = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mins, Qs[0], zero, 0, 0, 0);
            N = __builtin_amdgcn_mfma_f32_32x32x16_bf16(mins, Qs[1], N, 0, 0, 0);
            static_for<ND>([&](auto dI) {
                constexpr int d = decltype(dI)::value;
                const f16x8_t x = A[d % AP];
                N = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Qh[d], N, 0, 0, 0);
                fill(IC<2 * d>{});
                __builtin_amdgcn_sched_barrier(0);
                N = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Ql[d], N, 0, 0, 0);
                ahead(dI);
                fill(IC<2 * d + 1>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        auto values = [&](auto&& ahead, auto&& fill) {
            static_for<ND>([&](auto kI) {
                constexpr int k = decltype(kI)::value, d = k >> 1, s = k & 1;
                const f16x8_t x = A[k % AP];
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, __builtin_bit_cast(f16x8_t, Wh[s]), acc[d], 0, 0, 0);
                fill(IC<2 * k>{});
                __builtin_amdgcn_sched_barrier(0);
                acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, __builtin_bit_cast(f16x8_t, Wl[s]), acc[d], 0, 0, 0);
                ahead(kI);
                fill(IC<2 * k + 1>{});
                __builtin_amdgcn_sched_barrier(0);
            });
        };
        for (int i = tid; i < DT * 2 * kWave; i += NTH) (&vs[1][0][0][0])[i] = f16x8_t{};   // the values before the first tile
#pragma unroll
        for (int s = 0; s < 2; ++s) Wh[s] = Wl[s] = u32x4_t{};
        if (steps > 0) {
            k_store(0);
            k_load(1);
            next_id(2);
            barrier();
            static_for<AP>([&](auto dI) { A[decltype(dI)::value] = key_at(0, decltype(dI)::value); });
            scores(minima(0), [&](auto dI) {
                constexpr int d = decltype(dI)::value;
                if constexpr (d + AP < ND) A[d % AP] = key_at(0, d + AP);
            }, [](auto) {});
            k_store(1);
            k_load(2);
            next_id(3);
        }
        barrier();
#pragma unroll
        for (int k = 0; k < AP; ++k) A[k] = value_at(1, k);
        // Step st: tile st's products are in N. Its values and the keys of st + 2 go to LDS (slots whose last readers passed
        // the barrier before); the values of st - 1 are summed beside that and beside the scaling and maximum of the scores,
        // the scores of st + 1 beside the exponentials. One step more than tiles; before the first the weights are zero.
        float top = 0.f, w0 = 0.f, z0 = 0.f;
        float4 kf[2], sz[2], sv[2], mv[2];   // of 4 tokens, and the 4 after them, requested when those come up
        auto pick = [](const float4& x, int i) { return i == 0 ? x.x : i == 1 ? x.y : i == 2 ? x.z : x.w; };
        auto ask_scales = [&](int st, int j) {
            kf[j & 1] = of_tokens(tok[st & 3][0], j);
            sz[j & 1] = of_tokens(tok[st & 3][3], j);
        };
        auto scale_max = [&](int st, int i) {
            if (i % 4 == 0 && i < 12) ask_scales(st, i / 4 + 1);
            S[i] = N[i] * pick(kf[(i / 4) & 1], i & 3);
            const float z = __builtin_fmaf(S[i], factor, pick(sz[(i / 4) & 1], i & 3));
            if (i & 1)
                top = i == 1 ? fmaxf(z0, z) : fmaxf(fmaxf(z0, z), top);   // one instruction
            else
                z0 = z;
            asm volatile("" : "+v"(S[i]), "+v"(top), "+v"(z0));   // here, not where they are used
        };
        auto weight = [&](int st, int i) {
            if (i % 4 == 0 && i < 12) {
                sv[(i / 4 + 1) & 1] = of_tokens(tok[st & 3][1], i / 4 + 1);
                mv[(i / 4 + 1) & 1] = of_tokens(tok[st & 3][2], i / 4 + 1);
            }
            const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(S[i], factor, -mu));
            const float m = pick(mv[(i / 4) & 1], i & 3);
            tile_l = i == 0 ? p : tile_l + p;
            tile_low = i == 0 ? p * m : __builtin_fmaf(p, m, tile_low);
            if (i == 15) {
                l.add(tile_l);
                low.add(tile_low);
            }
            const float w = rounded(p * pick(sv[(i / 4) & 1], i & 3));
            if (i & 1) {
                const uint32_t h = high_parts(w0, w);
                Wh[i >> 3][(i & 7) / 2] = h;
                Wl[i >> 3][(i & 7) / 2] = high_parts(rest_of<0>(h, w0), rest_of<1>(h, w));
            }
            w0 = w;
        };
        for (int st = 0; steps > 0 && st <= steps; ++st) {
            bf16x8_t mins;
            {
                constexpr int SLOTS = 4 * DT, PER = 32 / SLOTS;   // places between products; scores at a place of the second half
                values([&](auto kI) {
                    constexpr int k = decltype(kI)::value;
                    A[k % AP] = k + AP < ND ? value_at((st + 1) & 1, k + AP) : key_at((st + 1) & 1, k + AP - ND);
                }, [&](auto kI) {
                    constexpr int k = decltype(kI)::value;
                    constexpr int EVERY = SLOTS / (4 * E);   // a word to LDS at every so many places of the first half
                    if constexpr (k == 0) k_scale();
                    if constexpr (k < SLOTS / 2 && k % EVERY == 0) {
                        if constexpr ((k / EVERY) & 1)
                            k_put(st + 2, (k / EVERY) >> 1);
                        else
                            v_put(st, (k / EVERY) >> 1);
                    }
                    if constexpr (k == SLOTS / 2 - 2) {
                        ask_scales(st, 0);
                        mins = minima(st + 1);
                    }
                    if constexpr (k == SLOTS / 2) {
                        s_put(st + 2);
                        v_load(1);
                    }
                    if constexpr (k == SLOTS / 2 + 2) {
                        k_load(st + 3);
                        next_id(st + 4);
                    }
                    if constexpr (k >= SLOTS / 2) {
#pragma unroll
                        for (int i = (k - SLOTS / 2) * PER; i < (k - SLOTS / 2 + 1) * PER; ++i) scale_max(st, i);
                    }
                    if constexpr (k == SLOTS - 2) {
                        sv[0] = of_tokens(tok[st & 3][1], 0);
                        mv[0] = of_tokens(tok[st & 3][2], 0);
                    }
                });
            }
            {
                const int t0 = kTile * (first_tile + st);
                if (t0 + kTile - 1 > wave_first || st == steps) {   // past the piece's last tile nothing is seen
                    const int last = st == steps ? -1 : limit;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float4 size = of_tokens(tok[st & 3][3], i / 4);
                        if (t0 + 16 * (i >> 3) + 8 * g + (i & 7) > last) S[i] = -INFINITY;
                        const float z = __builtin_fmaf(S[i], factor, pick(size, i & 3));
                        top = i ? fmaxf(top, z) : z;
                    }
                }
                if (__ballot(top > mu + kMoves)) {
                    const float now = fmaxf(mu, fmaxf(top, __shfl_xor(top, 32)));
                    const float shrink = __builtin_amdgcn_exp2f(mu - now);
                    mu = now;
                    l.scale(shrink);
                    low.scale(shrink);
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
                }
                // (past the wave's last tile these scores are of an old one, and unused)
                scores(mins, [&](auto dI) {
                    constexpr int d = decltype(dI)::value;
                    if constexpr (d + AP < ND) A[d % AP] = key_at((st + 1) & 1, d + AP);
                    // The tile's keys have been read, its values and the next keys are written: the next values can be read.
                    if constexpr (d == ND - 2) {
                        barrier();
#pragma unroll
                        for (int k = 0; k < AP - 1; ++k) A[k] = value_at(st & 1, k);
                    }
                    if constexpr (d == ND - 1) A[AP - 1] = value_at(st & 1, AP - 1);
                }, [&](auto kI) {
                    constexpr int k = decltype(kI)::value, PLACES = 2 * ND;
#pragma unroll
                    for (int i = k * 16 / PLACES; i < (k + 1) * 16 / PLACES; ++i) weight(st, i);
                });
            }
        }
        const float row_l = l.value() + __shfl_xor(l.value(), 32), row_low = low.value() + __shfl_xor(low.value(), 32);
        // The outputs, or the sums of a piece, by way of LDS: a lane of the sums has 16 bytes of each of many rows, the lanes that
        // write have whole lines.
        if (g == 0) {
            const bool none = mu == -FLT_MAX && row_l == 0.f, live = row0 + col < pairs;
            const int pair = (r.first + ti) * a.heads + head, k = static_cast<int>(blockIdx.x) * kPromptRows + 32 * wv + col;
            const int first = a.items * kRows + k, place = first + (begins ? kPromptRegion : 0);
            const float by = !whole ? 1.f : none ? 0.f : 1.f / (r.bad ? __builtin_nanf("") : row_l);
            out_rows[wv][col] = make_int2(__float_as_int(by), !live ? -1 : whole ? pair : place);
            if (live && !whole) a.stat[place] = make_float2(mu, r.bad ? __builtin_nanf("") : row_l);
            if (live && begins) a.info[pair] = whole ? make_int2(0, 1) : make_int2(first, line.pieces(unit_at, unit_steps));
        }
        // 4 neighbouring dims, the n-th of DT * 4: of E value tiles of one register, or 2 of two, or one of four
        auto four = [&](int n, int& dim) {
            const int m = n * 4 / (16 * E), rest = n - m * 4 * E;   // tile group; 4 registers' 16 rows x E dims as 4 E fours
            float x[4];
            if constexpr (E == 4) {
                const int i = rest;   // register
                dim = 128 * m + 4 * (8 * (i >> 2) + 4 * g + (i & 3));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[4 * m + e][i];
            } else if constexpr (E == 2) {
                const int i = 2 * rest;
                dim = 64 * m + 2 * (8 * (i >> 2) + 4 * g + (i & 3));
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[2 * m + (e & 1)][i + (e >> 1)];
            } else {
                const int i = 4 * rest;
                dim = 32 * m + 8 * (i >> 2) + 4 * g;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = acc[m][i + e];
            }
            return make_float4(x[0] + row_low, x[1] + row_low, x[2] + row_low, x[3] + row_low);
        };
        {
            auto meet = []() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); };   // of one wave
            meet();
            float* to_rows = whole ? a.out : a.part;
            const bool gated = whole && a.gate;
            const int dim0 = 4 * (lane & 15);
            float by[8];
            int64_t goes[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const int2 x = out_rows[wv][4 * j + (lane >> 4)];
                by[j] = __int_as_float(x.x);
                goes[j] = x.y < 0 ? -1 : static_cast<int64_t>(x.y) * D + dim0;
            }
            float4 gates[2][8];   // of 64 dims, requested before the 64 before them
            auto ask_gates = [&](int c) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    if (gated && goes[j] >= 0) gates[c & 1][j] = ld4(a.gate + goes[j] + 64 * c);
            };
            ask_gates(0);
#pragma unroll
            for (int c = 0; c < D / 64; ++c) {
                if (c + 1 < D / 64) ask_gates(c + 1);
#pragma unroll
                for (int n = 8 * c; n < 8 * c + 8; ++n) {
                    int dim;
                    const float4 x = four(n, dim);
                    st4(&outs[wv][col][dim - 64 * c], x);
                }
                meet();
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float4 x = ld4(&outs[wv][4 * j + (lane >> 4)][dim0]);
                    x = make_float4(x.x * by[j], x.y * by[j], x.z * by[j], x.w * by[j]);
                    if (gated) {
                        const float4 y = gates[c & 1][j];
                        if (__ballot(fminf(fminf(y.x, y.y), fminf(y.z, y.w)) < kFarGate))
                            x = make_float4(gated_by(x.x, y.x), gated_by(x.y, y.y), gated_by(x.z, y.z), gated_by(x.w, y.w));
                        else
                            x = make_float4(near_gated(x.x, y.x), near_gated(x.y, y.y), near_gated(x.z, y.z), near_gated(x.w, y.w));
                    }
                    if (goes[j] >= 0) st4(to_rows + goes[j] + 64 * c, x);
                }
                meet();
            }
        }
        if (!cut) return;
        line_at = unit_at = unit_at + line.over + unit_steps;   // the unit's end
        if (cut_at || line_at >= line_end) return;
        if (++unit == tiles * a.c.heads) {   // the next request that has row tiles
            unit = 0;
            uint64_t hit = 0;
            for (int b0 = b + 1; b0 < a.requests; b0 += kWave) {
                const Request4 q = b0 + lane < a.requests ? request(a, b0 + lane) : Request4{0, 0, 0, false};
                hit = __ballot(row_tiles(q) > 0);
                if (hit) {
                    const int l = __builtin_ctzll(hit);
                    b = b0 + l;
                    r = of_lane(q, l);
                    break;
                }
            }
            if (!hit) return;
        }
        unit_steps = steps_of(keys_seen(r, row_tiles(r) - 1 - unit / a.c.heads));
        __syncthreads();   // the last tile has been read from LDS
    }
}

// ------------------------------------------------------------------ join
// Joins the pieces of (row, head) pairs. `entry`: where a pair's pieces are, (0, 0) where nothing is to be joined.
__device__ __forceinline__ Places places(const Attn4Args& a, int first) { return places_of(first, a.items * kRows); }
__device__ __forceinline__ int2 entry(const Attn4Args& a, int64_t pair, bool live) {
    // Pairs of the requests' rows alone: only those have an entry of this call (the workspace may hold an earlier one's).
    const int from = min(max(a.row_start[0], 0), a.rows) * a.heads, end = min(max(a.row_start[a.requests], 0), a.rows) * a.heads;
    int2 in = make_int2(0, 0);
    if (live && pair >= from && pair < end) in = a.info[pair];
    return joinable(in.x, in.y, a.items * kRows, a.all_places) ? in : make_int2(0, 0);
}
// The join of two parts of a sum with their references: (m, l, s) takes in (n, k, x).
template <int V>
__device__ __forceinline__ void join_in(float& m, float& l, float (&s)[V], float n, float k, const float (&x)[V]) {
    const float now = fmaxf(m, n);
    const float was = __builtin_amdgcn_exp2f(m - now), f = __builtin_amdgcn_exp2f(n - now);
    m = now;
    l = l * was + k * f;
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = s[i] * was + x[i] * f;
}

// Few pairs, each of perhaps hundreds of pieces: a workgroup of 8 waves per pair and 64 dims, 16 lanes a piece. (A workgroup per
// pair, whole rows: what one CU can read bounded it, 7.7 us for 16 pairs of 256 pieces.)
constexpr int kJoinWaves = 8;
template <int D>
__global__ __launch_bounds__(kJoinWaves* kWave) void join4_few(const Attn4Args a) {
    __shared__ __align__(16) float sums[kJoinWaves][64];
    __shared__ float ls[kJoinWaves], ms[kJoinWaves];
    constexpr int PARTS = D / 64, LANES = 4 * kJoinWaves;   // pieces looked at together
    const int lane = threadIdx.x & 63, wv = wave_in_block(), mine = static_cast<int>(threadIdx.x) >> 4;
    const int pair = static_cast<int>(blockIdx.x) / PARTS, d = 64 * (static_cast<int>(blockIdx.x) % PARTS) + 4 * (lane & 15);
    const int2 in = entry(a, pair, true);
    if (in.y == 0) return;   // the whole workgroup
    const int pieces = in.y;
    const Places place = places(a, in.x);
    float m = -FLT_MAX, l = 0.f, s[4] = {0.f, 0.f, 0.f, 0.f};
    constexpr int U = 8;   // in flight
    for (int p0 = mine; p0 < pieces; p0 += U * LANES) {
        float2 st[U];
        float x[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p0 + u * LANES < pieces) {
                const size_t q = place.of(p0 + u * LANES);
                st[u] = a.stat[q];
                load_floats(a.part + q * D + d, x[u]);
            } else {
                st[u] = make_float2(-FLT_MAX, 0.f);
                x[u][0] = x[u][1] = x[u][2] = x[u][3] = 0.f;
            }
        }
        __builtin_amdgcn_sched_barrier(0);   // all U loads before the first use
#pragma unroll
        for (int u = 0; u < U; ++u) join_in(m, l, s, st[u].x, st[u].y, x[u]);
    }
    // the wave's four pieces, then the waves
    auto over_rows = [](float v, auto&& op) {
        const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        v = op(__uint_as_float(p[0]), __uint_as_float(p[1]));
        const auto q = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
        return op(__uint_as_float(q[0]), __uint_as_float(q[1]));
    };
    auto add = [](float x, float y) { return x + y; };
    const float top = over_rows(m, [](float x, float y) { return fmaxf(x, y); }), f = __builtin_amdgcn_exp2f(m - top);
    l = over_rows(l * f, add);
#pragma unroll
    for (int i = 0; i < 4; ++i) s[i] = over_rows(s[i] * f, add);
    if (lane < 16) st4(&sums[wv][4 * lane], make_float4(s[0], s[1], s[2], s[3]));
    if (lane == 0) {
        ms[wv] = top;
        ls[wv] = l;
    }
    __syncthreads();
    if (threadIdx.x >= 64) return;
    const size_t o = static_cast<size_t>(pair) * D + d - 4 * (lane & 15) + lane;
    const float gate = a.gate ? a.gate[o] : 0.f;
    float all = ms[0], sum = 0.f, tot = 0.f;
#pragma unroll
    for (int w = 1; w < kJoinWaves; ++w) all = fmaxf(all, ms[w]);
#pragma unroll
    for (int w = 0; w < kJoinWaves; ++w) {
        const float k = __builtin_amdgcn_exp2f(ms[w] - all);
        sum += k * sums[w][lane];
        tot += k * ls[w];
    }
    a.out[o] = finished(all, sum, tot, a.gate, gate);
}

// Many pairs. NW > 1: a workgroup of NW waves per pair, wave w takes pieces w, w + NW, ...; NW = 1: a wave per pair, and each wave
// looks at `per` pairs at once, because in a prompt's call most are there already. Lanes hold the dims.
template <int D, int NW>
__global__ __launch_bounds__(NW == 1 ? 4 * kWave : NW * kWave) void join4_kernel(const Attn4Args a, int per) {
    constexpr int V = D / kWave;
    __shared__ float sums[NW][NW == 1 ? 1 : D], ls[NW], ms[NW];
    const int lane = threadIdx.x & 63, wv = NW == 1 ? 0 : wave_in_block();
    const int64_t pair0 = NW == 1 ? (static_cast<int64_t>(blockIdx.x) * 4 + wave_in_block()) * per : blockIdx.x;
    const int2 in = entry(a, pair0 + lane, lane < (NW == 1 ? per : 1));
    uint64_t todo = __ballot(in.y > 0);   // the same in every wave of a pair
    while (todo) {
        const int k = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int pieces = __builtin_amdgcn_readlane(in.y, k);
        const Places place = places(a, __builtin_amdgcn_readlane(in.x, k));
        const size_t o = static_cast<size_t>(pair0 + k) * D;
        float m = -FLT_MAX, l = 0.f, s[V], gate[V];
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = gate[i] = 0.f;
        if (NW == 1 && a.gate) load_floats(a.gate + o + V * lane, gate);
        constexpr int U = 4;   // pieces in flight
        for (int p0 = wv; p0 < pieces; p0 += U * NW) {
            float2 st[U];
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t q = place.of(min(p0 + u * NW, pieces - 1));
                st[u] = a.stat[q];
                load_floats(a.part + q * D + V * lane, x[u]);
            }
            __builtin_amdgcn_sched_barrier(0);   // all U loads before the first use
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p0 + u * NW >= pieces) break;
                join_in(m, l, s, st[u].x, st[u].y, x[u]);
            }
        }
        if constexpr (NW == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] = finished(m, s[i], l, a.gate, gate[i]);
            store_floats(a.out + o + V * lane, s);
        } else {
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
                a.out[o + d] = finished(top, sum, tot, a.gate, a.gate ? a.gate[o + d] : 0.f);
            }
        }
    }
}

// ------------------------------------------------------------------ host
// Whether a call can have requests for prompt4_kernel; if not, split4_kernel takes them all. A call with no more rows than
// requests is taken for a batch of single tokens, up to kSplitOnly (row, head) pairs of a KV head, and spared the launch;
// should one request have all the rows, split4_kernel answers it too.
bool may_prompt(int rows, int requests, int group) {
    const int64_t pairs = static_cast<int64_t>(rows) * group;
    return rows > 1 && pairs > kSplitMax && (rows > requests || pairs > kSplitOnly);
}
// split4_kernel's workgroups of 4 waves on a CU, by their registers.
int places_on_cu(int dim) { return dim == 256 ? 2 : dim == 128 ? 3 : 4; }
constexpr int kCus = 256;
// Its pieces are at most as many as wanted (and a few for rounding) plus one per unit; units at most one per 8 pairs and what each
// request's last one lacks, and, where larger requests go to prompt4_kernel, at most one per 8 of the pairs with which one does not
// (plus one, so that the bound does not fall where the first request goes there).
int64_t all_units(int rows, int requests, int heads, int kv_heads) {
    const int group = heads / kv_heads;   // a request's last block lacks a multiple of what group and kRows have in common
    const int64_t lacking = kRows - std::gcd(group, kRows), busy = std::min(rows, requests);
    return (static_cast<int64_t>(rows) * group + busy * lacking) / kRows * kv_heads;
}
int64_t unit_bound(int rows, int requests, int heads, int kv_heads) {
    const int group = heads / kv_heads;
    const int64_t units = all_units(rows, requests, heads, kv_heads);
    if (!may_prompt(rows, requests, group)) return units;
    const int64_t busy = std::min(rows, requests);
    return std::min(units, busy * (blocks_for(std::max(kSplitMax, group), kRows) + 1) * kv_heads);
}
int64_t item_bound(int64_t units, int dim) {
    const int64_t places = kCus * places_on_cu(dim);
    return (units > places ? 4 : 1) * places + 8 + units;
}
size_t align_up(size_t b) { return (b + 255) & ~size_t{255}; }

struct Layout {
    int64_t items, places;   // pieces of split4_kernel that have places; places of the workspace
    size_t stat, info, bytes;
};
Layout layout(int rows, int requests, int heads, int kv_heads, int dim) {
    Layout l;
    l.items = item_bound(unit_bound(rows, requests, heads, kv_heads), dim);
    // Room for cut prompts, and for a light call's pieces (which has them only with no more units than the card has places), by the
    // rows alone, though a call with no more rows than requests has neither: a workspace for some rows and requests has to serve
    // fewer of either.
    const bool large = rows > 1 && static_cast<int64_t>(rows) * (heads / kv_heads) > kSplitMax;
    if (large) l.items = std::max<int64_t>(l.items, 2 * kCus * places_on_cu(dim) + 8);
    l.places = l.items * kRows + (large ? 2 * kPromptRegion : 0);
    l.stat = align_up(static_cast<size_t>(l.places) * dim * 4);
    l.info = l.stat + align_up(static_cast<size_t>(l.places) * 8);
    l.bytes = l.info + align_up(static_cast<size_t>(rows) * heads * 8);
    return l;
}

// Table rows that hold no more tiles than this make calls whose units are not cut: a workgroup's eight waves take them in kWhole / 8
// turns, less than the launch that joins pieces.
constexpr int kWhole = 16;

template <int D, int NW>
void launch_split(const Attn4Args& a, int grid, hipStream_t s) {
    const auto split = a.c.page >= kTile ? split4_kernel<D, true, NW> : split4_kernel<D, false, NW>;
    split<<<static_cast<unsigned>(grid), NW * kWave, 0, s>>>(a);
}

template <int D>
void launch(const Attn4Args& a, int grid, hipStream_t s) {
    if (a.whole) return launch_split<D, kWholeWaves>(a, grid, s);
    launch_split<D, kSplitWaves>(a, grid, s);
    if (!a.split_all) {
        const int64_t pairs = static_cast<int64_t>(a.rows) * a.group;
        const int64_t tiles = (pairs / kPromptRows + std::min<int64_t>(a.requests, pairs / kSplitMax + 1)) * a.c.heads;
        prompt4_kernel<D><<<static_cast<unsigned>(std::max<int64_t>(tiles, kPromptFill)), kPromptWaves * kWave, 0, s>>>(a);
    }
    const unsigned pairs = static_cast<unsigned>(a.rows) * static_cast<unsigned>(a.heads);
    if (pairs <= 128)   // few rows: many pieces each
        join4_few<D><<<pairs * (D / 64), kJoinWaves * kWave, 0, s>>>(a);
    else if (pairs <= 2048)
        join4_kernel<D, 4><<<pairs, 4 * kWave, 0, s>>>(a, 1);
    else if (pairs <= kPromptCut * kPromptRows)   // many of them in pieces
        join4_kernel<D, 1><<<blocks_for(pairs, 4), 4 * kWave, 0, s>>>(a, 1);
    else
        join4_kernel<D, 1><<<blocks_for(pairs, 16), 4 * kWave, 0, s>>>(a, 4);
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
    a.all_places = static_cast<int>(l.places);
    a.places = kCus * places_on_cu(dim);
    a.light_work = kLightWork * (256 / dim);
    const int64_t tiles = (static_cast<int64_t>(max_pages) * page_size + kTile - 1) / kTile;
    const int64_t units = unit_bound(rows, requests, heads, kv_heads), every = all_units(rows, requests, heads, kv_heads);
    const bool prompts = may_prompt(rows, requests, a.group);
    a.light = prompts && every <= kLightUnits && every * (tiles + kUnitCost) <= a.light_work;
    a.split_all = !prompts || a.light;
    a.whole = a.split_all && tiles <= kWhole && (!a.light || every <= kCus);   // more units: the card has places for more small ones
    // pieces of no more units than places, or whole units
    const int64_t light_grid = std::max(a.places + 8 + std::min<int64_t>(every, a.places), std::min<int64_t>(every, kLightUnits));
    const int64_t grid = a.whole ? every : prompts ? std::max(item_bound(units, dim), light_grid) : item_bound(units, dim);
    QK_REQUIRE(grid * (a.whole ? kWholeWaves : kSplitWaves) * kWave < (int64_t{1} << 32),
               "attn_kv4_rows: %d rows of %d KV heads in %d requests exceed one call", rows, kv_heads, requests);
    a.prompt_step = 1;   // a line is below 2^30 steps, in 32 bits
    while (kPromptCut * (tiles / a.prompt_step + 1 + kPromptCost) >= (1 << 30)) a.prompt_step *= 2;
    const hipStream_t s = as_stream(stream);
    if (dim == 64)
        launch<64>(a, static_cast<int>(grid), s);
    else if (dim == 128)
        launch<128>(a, static_cast<int>(grid), s);
    else
        launch<256>(a, static_cast<int>(grid), s);
    return check_launch("attn_kv4_rows");
}

}  // extern "C"
