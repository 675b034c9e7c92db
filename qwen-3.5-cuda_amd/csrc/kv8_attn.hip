// Attention over the paged 8-bit cache (kv8_common.hpp) on gfx950: the rows of several requests in one call, single
// tokens and prompts mixed. Row i of a request with n rows and kv_len keys stands at position kv_len - n + i and sees
// keys 0 .. position:
//   out = sum_t softmax_t(q . k_t / sqrt(D)) v_t  (x sigmoid(gate)),  zeros where no key is seen.
// The reference has the one-token form over an fp32 cache (src/cuda/attn_kernels.cu:72-195, src/layer_attn.cpp:103-108).
//
// Both products run on v_mfma_f32_16x16x32_f16 with an fp32 dot product's accuracy: a code is exact in fp16, and the
// other operand (a query row scaled by a power of two; the softmax weights) is two fp16 parts, 22 bits. Both are
// computed transposed, scores^T = K q^T and out^T = V^T p^T, because then the scores that a lane holds (4 tokens of one
// row in each tile) are already the p^T operand of the second product: with key row lr of tile `half` standing for token
// 8 (lr / 4) + 4 half + lr % 4, lane group lk holds tokens 8 lk .. 8 lk + 7, whose value codes of one dim are 8
// neighbouring bytes of the cache. Nothing crosses lanes or LDS between the products.
//
// Scales: score = S * (2^-e / sqrt(D) log2(e) * k_scale); the value scale rides on the weights, w = p * v_scale, so that
// tokens of pages with different scales share one accumulator. The running reference m of the exponentials therefore
// bounds score + log2(v_scale); it moves, and the sums are rescaled, only when a score passes it by 8 (weights up to
// 2^8 are as exact as weights up to 1). A page of zeros has the smallest scale, 2^-100, and counts there as one of 2^-40:
// counted as 2^-100 its keys' weights fell below the smallest fp32 number, and out of the softmax's sum, when a page with
// values came into the same row (512 zeros with weights of 2^-10 beside values of 2^30: outputs off by a hundredth). What is
// left of that: of two scales 2^d apart the smaller one's keys lose weights below 2^(d - 126), and beside zeros of the
// same score a scale below 2^-49 loses a bit at each halving.
//
// Two kernels. split_kernel (few rows per request): bound by the cache's bytes. A workgroup takes 8 (row, head) pairs
// that share a KV head - 16 columns: 8 rows x 2 fp16 parts - and a range of 32-token tiles, its 4 waves every fourth tile,
// straight from the cache to operand registers. The ranges are cut so that the whole call, ragged requests and all, is
// about kTargetItems equal pieces; every workgroup works that out from the lengths, so nothing is planned on the host.
// combine_kernel joins the pieces. prompt_kernel (many rows): bound by the MFMAs. 128 rows per workgroup on
// v_mfma_f32_32x32x16_f16, the codes turned to fp16 once per workgroup into LDS.
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <type_traits>
#include <utility>

#include "capi_common.hpp"
#include "device_common.hpp"
#include "kv8_common.hpp"

namespace qk {
namespace {

typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

constexpr int kTile = 32;              // tokens of a step
constexpr int kSplitWaves = 4;
constexpr int kSplitBlock = kSplitWaves * kWave;
constexpr int kRows = 8;               // (row, head) pairs of a split workgroup
constexpr int kTargetItems = 1024;     // pieces of the whole call
constexpr int kMinTiles = 8;           // of a piece: two steps per wave; one in calls that then still have at most kFewItems
constexpr int kFewItems = 256;         // pieces, one a CU (4 tokens at 4000 keys 14.9 us with 4 tiles, 16.2 with 8; one token
                                       // at 30000 keys 22.7, 19.0)
constexpr int kSplitMax = 32;          // (row, head) pairs of a request and KV head that still take the split kernel (100
                                       // requests of 64 at 1500 keys: 205 us, with the prompt kernel 108); a single row does
constexpr int kSplitOnly = 1024;       // and of a whole call that has no more rows than requests
constexpr float kMoves = 8.0f;         // a score past the reference by more moves it
constexpr float kWeightUp = 64.0f;     // weights (up to 2^8) enter fp16 times 2^6

struct AttnArgs {
    const float* q;
    const float* gate;   // or null
    float* out;
    Kv8Cache c;
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* kv_len;
    int max_pages, page_shift, requests, rows, heads, group;
    int split_all;       // every request takes the split kernel
    float* part;         // [item][kRows][D] sums
    float2* stat;        // [item][kRows] (m, l)
    int2* info;          // [row][head] (first item * kRows + row in item, pieces); written for the requests' rows alone
    int items;           // capacity: the split kernel's grid
    int all_items;       // and with the cut prompts' pieces
    float scale;         // log2(e) / sqrt(D)
};

// A request as the kernels see it, whatever the arrays hold: rows inside q, lengths from 0 to what the table row holds
// (`bad` marks a longer one, whose rows come out NaN). Starts that do not decrease give every row between the first and the
// last one request; of others the rows are not defined, but nothing is read or written out of bounds.
struct Request {
    int first, n, len;
    bool bad;
};
__device__ __forceinline__ Request request(const AttnArgs& a, int b) {
    const int s = min(max(a.row_start[b], 0), a.rows), e = min(max(a.row_start[b + 1], s), a.rows);
    const int len = a.kv_len[b], most = a.max_pages << a.page_shift;
    return Request{s, e - s, min(max(len, 0), most), len > most};
}
__device__ __forceinline__ bool takes_split(const AttnArgs& a, const Request& r) {
    return a.split_all || static_cast<int64_t>(r.n) * a.group <= max(kSplitMax, a.group);
}

// Inclusive prefix over the wave.
__device__ __forceinline__ int64_t wave_prefix(int64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int64_t up = __shfl_up(v, o);
        if (lane >= o) v += up;
    }
    return v;
}

// Piece `item` of the call: request, which of its units (KV head, row block), which piece of the unit's tiles. Every wave
// finds it by itself from the lengths (64 requests at a time).
struct Piece {
    int b, unit, split, splits, tiles;   // tiles: of one piece
};
__device__ __forceinline__ int tiles_of(const Request& r) { return max(1, (r.len + kTile - 1) / kTile); }
__device__ __forceinline__ int64_t units_of(const AttnArgs& a, const Request& r) {
    return takes_split(a, r) ? (static_cast<int64_t>(r.n) * a.group + kRows - 1) / kRows * a.c.heads : 0;
}
__device__ bool find_piece(const AttnArgs& a, int64_t item, Piece& p) {
    const int lane = threadIdx.x & 63;
    int64_t total = 0;
    for (int b = lane; b < a.requests; b += kWave) {
        const Request r = request(a, b);
        total += units_of(a, r) * tiles_of(r);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o);
    const int64_t least = min(max((total + kFewItems - 1) / kFewItems, static_cast<int64_t>(kSplitWaves)),
                              static_cast<int64_t>(kMinTiles));
    const int64_t cut = max(least, (total + kTargetItems - 1) / kTargetItems);
    p.tiles = static_cast<int>(min(cut, static_cast<int64_t>(0x7fffffff)));
    for (int b0 = 0; b0 < a.requests; b0 += kWave) {
        const int b = b0 + lane;
        int64_t n = 0;
        int splits = 0;
        if (b < a.requests) {
            const Request r = request(a, b);
            splits = static_cast<int>((tiles_of(r) + cut - 1) / cut);
            n = units_of(a, r) * splits;
        }
        const int64_t upto = wave_prefix(n, lane);
        const uint64_t hit = __ballot(item < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int64_t local = item - (__shfl(upto, l) - __shfl(n, l));
            p.b = __builtin_amdgcn_readfirstlane(b0 + l);
            p.splits = __builtin_amdgcn_readfirstlane(__shfl(splits, l));
            p.unit = __builtin_amdgcn_readfirstlane(static_cast<int>(local / p.splits));
            p.split = __builtin_amdgcn_readfirstlane(static_cast<int>(local - static_cast<int64_t>(p.unit) * p.splits));
            return true;
        }
        item -= __shfl(upto, 63);
    }
    return false;
}

// 8 codes -> the fp16 operand: byte u = code + 128 under 0x64 is the fp16 1024 + u.
__device__ __forceinline__ f16x8_t codes8(uint32_t a, uint32_t b) {
    const uint32_t x[2] = {a ^ 0x80808080u, b ^ 0x80808080u};
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        w[2 * i] = __builtin_amdgcn_perm(0x64646464u, x[i], 0x04010400u);
        w[2 * i + 1] = __builtin_amdgcn_perm(0x64646464u, x[i], 0x04030402u);
    }
    f16x8_t r;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const f16x2_t h = __builtin_bit_cast(f16x2_t, w[i]) - f16x2_t{(_Float16)1152.0f, (_Float16)1152.0f};
        r[2 * i] = h[0];
        r[2 * i + 1] = h[1];
    }
    return r;
}

__device__ __forceinline__ float max_over_lk(float v) {
    v = fmaxf(v, __shfl_xor(v, 16));
    return fmaxf(v, __shfl_xor(v, 32));
}

// The fp32 product behind a value that is then split in two fp16 parts: kept from being fused into the conversion
// (v_fma_mixlo_f16 rounds once where the other part's subtraction has rounded twice, and the parts miss by an fp16 ulp
// of one weight in some thousands).
__device__ __forceinline__ float rounded(float v) {
    asm("" : "+v"(v));
    return v;
}
// The value scale that the exponentials' reference counts with (0 where nothing of the octet is seen).
constexpr float kZerosScale = 0x1p-40f;
__device__ __forceinline__ float reference_scale(float sv) { return sv > kKv8Floor ? sv : kZerosScale; }

__device__ __forceinline__ float low_part(float v) { return v - static_cast<float>(static_cast<_Float16>(v)); }

// Where the octet of tokens that starts at token t lies: the page's first code (of one head) and the two scales. Tokens
// from `seen` on are not looked up (page 0, scales 0: their weights are 0); a page id outside the cache has scale NaN.
struct Octet {
    size_t base;   // (page, head) index
    bool live, bad;
};
__device__ __forceinline__ Octet octet(const AttnArgs& a, int b, int h, int t, int seen) {
    Octet o{static_cast<size_t>(h), t < seen, false};
    if (!o.live) return o;
    const int j = t >> a.page_shift;
    const int id = j < a.max_pages ? a.table[static_cast<size_t>(b) * a.max_pages + j] : -1;
    o.bad = id < 0 || id >= a.c.pages;
    if (!o.bad) o.base = static_cast<size_t>(id) * a.c.heads + h;
    return o;
}

// ------------------------------------------------------------------ few rows
template <int D>
__global__ __launch_bounds__(kSplitBlock, 2) void split_kernel(const AttnArgs a) {
    constexpr int NJ = D / 64, ND = D / 32, LD = D + 2;
    __shared__ float sums[kSplitWaves][kRows * LD];
    __shared__ float stat[kSplitWaves][kRows][2];
    __shared__ __align__(16) _Float16 qs[2 * kRows][D + 8];   // the queries' parts; 16 bytes more, and 16 rows meet no bank twice
    __shared__ float factors[kRows];
    Piece pc;
    if (!find_piece(a, blockIdx.x, pc)) return;   // the whole workgroup
    const Request r = request(a, pc.b);
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
    const size_t block = static_cast<size_t>(P) * D;

    struct Where {
        const int8_t* k;
        const int8_t* v;
        const float* ks;
        const float* vs;
        bool live, bad;
    };
    auto where = [&](int tile) {   // this lane's addresses: key rows of octet lr / 4, values and scales of octet lk
        const int t0 = tile * kTile;
        const int tk = t0 + 8 * (lr >> 2), tv = t0 + 8 * lk;
        const Octet ok = octet(a, pc.b, h, tk, seen), ov = octet(a, pc.b, h, tv, seen);
        Where w;
        w.k = a.c.k + ok.base * block + static_cast<size_t>((tk & (P - 1)) + (lr & 3)) * D + 16 * lk;
        w.v = a.c.v + ov.base * block + (static_cast<size_t>((tv & (P - 1)) >> 3) * D + 2 * lr) * 8;
        w.ks = a.c.ks + ov.base;
        w.vs = a.c.vs + ov.base;
        w.live = ov.live;
        w.bad = ov.bad;
        return w;
    };
    uint4 K[2][NJ], V[ND];
    float ksc, vsc;
    auto load_k = [&](const Where& w) {
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int j = 0; j < NJ; ++j) K[half][j] = ld16(w.k + 4 * half * D + 64 * j);
    };
    auto load_v = [&](const Where& w) {
#pragma unroll
        for (int m = 0; m < ND; ++m) V[m] = ld16(w.v + 32 * 8 * m);
        ksc = *w.ks;
        vsc = *w.vs;
        if (!w.live) ksc = vsc = 0.f;
        if (w.bad) ksc = __builtin_nanf("");
    };
    // The rows' queries, scaled by 2^e so that a row's largest magnitude is in [2^14, 2^15), as two fp16 parts: 2 rows a wave,
    // requested before the first tile. (Every wave on its own for all 8 rows: half of the vector work of a short piece.)
    const int qr = 2 * wv + (lane >> 5), qp = min(rb * kRows + qr, pairs - 1), qt = qp / G;
    const float* qrow = a.q + (static_cast<size_t>(r.first + qt) * a.heads + h * G + (qp - qt * G)) * D + (lane & 31) * (D / 32);
    float qf[D / 32];
    if constexpr (D >= 128) {
#pragma unroll
        for (int i = 0; i < D / 128; ++i) {
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
        for (int i = 0; i < D / 32; ++i) {
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
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const float v = ok ? ldexpf(qf[i], e) : 0.f;
            qs[2 * qr][(lane & 31) * (D / 32) + i] = static_cast<_Float16>(v);
            qs[2 * qr + 1][(lane & 31) * (D / 32) + i] = static_cast<_Float16>(low_part(v));
        }
        if ((lane & 31) == 0) factors[qr] = ok ? ldexpf(a.scale, -e) : __builtin_nanf("");   // products to log2 scores; NaN: a row
    }                                                                                        // with infinities or NaNs
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the tile's loads stay in flight
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    f16x8_t Q[2 * NJ];   // dims 64 j + 16 lk + 8 (d % 2) + 0..7 of depth d = 2 j + d % 2
#pragma unroll
    for (int d = 0; d < 2 * NJ; ++d)
        Q[d] = *reinterpret_cast<const f16x8_t*>(&qs[lr][64 * (d >> 1) + 16 * lk + 8 * (d & 1)]);
    const float factor = factors[lr >> 1];
    f32x4_t acc[ND][2];
#pragma unroll
    for (int m = 0; m < ND; ++m) acc[m][0] = acc[m][1] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    float mu = -FLT_MAX, l = 0.f;
    for (; t < t_end; t += kSplitWaves) {
        const bool more = t + kSplitWaves < t_end;
        f32x4_t S[2];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            S[half] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int j = 0; j < NJ; ++j) {
                const uint4 w = K[half][j];
                S[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w.x, w.y), Q[2 * j], S[half], 0, 0, 0);
                S[half] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w.z, w.w), Q[2 * j + 1], S[half], 0, 0, 0);
            }
        }
        if (more) load_k(next);
        const float f = factor * ksc;
        float sv = vsc;
        float s[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float v = S[i >> 2][i & 3];
            s[i] = (v + dpp_move<0xB1>(v)) * f;   // both fp16 parts of the query
        }
        if (t * kTile + kTile - 1 > first_limit) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (t * kTile + 8 * lk + i > limit) s[i] = -INFINITY;
            if (t * kTile + 8 * lk > limit) sv = 0.f;   // a page that the row does not see may be marked: no 0 * NaN
        }
        float top = s[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = fmaxf(top, s[i]);
        top += __builtin_amdgcn_logf(reference_scale(sv));   // log2
        if (__ballot(top > mu + kMoves)) {
            const float now = fmaxf(mu, max_over_lk(top));
            const float shrink = __builtin_amdgcn_exp2f(mu - now);
            mu = now;
            l *= shrink;
#pragma unroll
            for (int m = 0; m < ND; ++m)
#pragma unroll
                for (int e = 0; e < 2; ++e)
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[m][e][i] *= shrink;
        }
        f16x8_t W;
        const float up = sv * kWeightUp;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float p = __builtin_amdgcn_exp2f(s[i] - mu);
            l += p;
            const float w = rounded(p * up);
            W[i] = static_cast<_Float16>(part ? low_part(w) : w);
        }
#pragma unroll
        for (int m = 0; m < ND; ++m) {
            const uint4 w = V[m];
            acc[m][0] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w.x, w.y), W, acc[m][0], 0, 0, 0);
            acc[m][1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(w.z, w.w), W, acc[m][1], 0, 0, 0);
        }
        if (more) {
            load_v(next);
            if (t + 2 * kSplitWaves < t_end) next = where(t + 2 * kSplitWaves);
        }
    }
    // The waves' sums meet in LDS; the two parts of a row are neighbouring columns, each lane of a pair writes every
    // other dim of both.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    float* mine = sums[wv] + (lr >> 1) * LD;
#pragma unroll
    for (int m = 0; m < ND; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float e0 = acc[m][0][i] + dpp_move<0xB1>(acc[m][0][i]);
            const float e1 = acc[m][1][i] + dpp_move<0xB1>(acc[m][1][i]);
            mine[32 * m + 8 * lk + 2 * i + part] = part ? e1 : e0;
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
            float v = tot == 0.f ? 0.f : sum / kWeightUp / tot;
            if (a.gate) v *= sigmoid(a.gate[o]);
            a.out[o] = v;
        } else {
            a.part[(static_cast<size_t>(blockIdx.x) * kRows + row) * D + d] = sum;
            if (d == 0) a.stat[static_cast<size_t>(blockIdx.x) * kRows + row] = make_float2(m, tot);
        }
        if (d == 0 && pc.split == 0) a.info[o / D] = make_int2(static_cast<int>(blockIdx.x) * kRows + row, pc.splits);
    }
}

// ------------------------------------------------------------------ join
// Joins the pieces of (row, head) pairs. NW > 1: a workgroup of NW waves per pair, wave w takes pieces w, w + NW, ...; NW = 1:
// a wave per pair, and each wave looks at `per` pairs at once, because in a prompt's call most are there already (a
// workgroup per pair took 29 us at 5000 rows of 16 heads). Lanes hold the dims.
template <int D, int NW>
__global__ __launch_bounds__(NW == 1 ? 4 * kWave : NW * kWave) void combine_kernel(const AttnArgs a, int per) {
    constexpr int V = D / kWave;
    __shared__ float sums[NW][NW == 1 ? 1 : D], ls[NW], ms[NW];
    const int lane = threadIdx.x & 63, wv = NW == 1 ? 0 : wave_in_block();
    // Pairs of the requests' rows alone: only those have an entry of this call (the workspace may hold an earlier one's).
    const int from = min(max(a.row_start[0], 0), a.rows) * a.heads, live = min(max(a.row_start[a.requests], 0), a.rows) * a.heads;
    const int64_t pair0 = NW == 1 ? (static_cast<int64_t>(blockIdx.x) * 4 + wave_in_block()) * per : blockIdx.x;
    int2 in = make_int2(0, 0);
    if (lane < (NW == 1 ? per : 1) && pair0 + lane >= from && pair0 + lane < live) in = a.info[pair0 + lane];
    const bool join = in.y > 1 && in.x >= 0 && in.y <= a.all_items - in.x / kRows;
    auto load = [](const float* p, float(&f)[V]) {
        if constexpr (V == 4) {
            const float4 x = ld4(p);
            f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i) f[i] = p[i];
        }
    };
    uint64_t todo = __ballot(join);   // the same in every wave of a pair
    while (todo) {
        const int k = __builtin_ctzll(todo);
        todo &= todo - 1;
        const int pieces = __builtin_amdgcn_readlane(in.y, k), where = __builtin_amdgcn_readlane(in.x, k);
        const int slot = where % kRows, first = where / kRows;
        float m = -FLT_MAX, l = 0.f, s[V], gt[V];
        const size_t o = static_cast<size_t>(pair0 + k) * D;
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = 0.f, gt[i] = 0.f;
        if (NW == 1 && a.gate) load(a.gate + o + V * lane, gt);
        auto at = [&](int p) { return static_cast<size_t>(first + p) * kRows + slot; };
        constexpr int U = 4;   // pieces in flight
        for (int p0 = wv; p0 < pieces; p0 += U * NW) {
            float2 st[U];
            float x[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const size_t q = at(min(p0 + u * NW, pieces - 1));
                st[u] = a.stat[q];
                load(a.part + q * D + V * lane, x[u]);
            }
            __builtin_amdgcn_sched_barrier(0);   // all U loads before the first use
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (p0 + u * NW >= pieces) break;
                const float now = fmaxf(m, st[u].x);
                const float was = __builtin_amdgcn_exp2f(m - now), f = __builtin_amdgcn_exp2f(st[u].x - now);
                m = now;
                l = l * was + st[u].y * f;
#pragma unroll
                for (int i = 0; i < V; ++i) s[i] = s[i] * was + x[u][i] * f;
            }
        }
        auto done = [&](float sum, float tot, float gate) {
            const float v = tot == 0.f ? 0.f : sum / kWeightUp / tot;
            return a.gate ? v * sigmoid(gate) : v;
        };
        if constexpr (NW == 1) {
#pragma unroll
            for (int i = 0; i < V; ++i) s[i] = done(s[i], l, gt[i]);
            if constexpr (V == 4) {
                st4(a.out + o + 4 * lane, make_float4(s[0], s[1], s[2], s[3]));
            } else {
#pragma unroll
                for (int i = 0; i < V; ++i) a.out[o + V * lane + i] = s[i];
            }
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
                a.out[o + d] = done(sum, tot, a.gate ? a.gate[o + d] : 0.f);
            }
        }
    }
}

// ------------------------------------------------------------------ many rows
// 4 waves, one a SIMD, of 32 rows each, on v_mfma_f32_32x32x16_f16: an operand of keys or values, 1 KB of LDS, feeds 2
// products (both parts of 32 rows), 64 cycles, so that the waves' reads take half of the LDS's rate; with 16 rows a wave they
// took all of it (5000 rows 690 us, now 480 to 550 with the card's clock). A wave holds its rows' query parts (128
// registers at D = 256, pinned in accumulation registers) and sums (128). Its vector work - softmax, turning codes to fp16 -
// is laid between its own products: while tile t + 1's scores are computed, tile t's are exponentiated; while tile t's
// values are summed, the codes of the next tiles go to LDS. All waves run all tiles of the workgroup, though a wave's own
// rows may end one earlier: with a branch around the products the compiler moves the sums between register files at each.
// The scores^T tile has token rho = 8 b + 4 g + j of the 32 in register 4 b + j of lane half g; key row rho stands for token
// 16 (b / 2) + 8 g + 4 (b % 2) + j, so that a lane's registers 8 s .. 8 s + 7 are octet 2 s + g, its share of the second
// product's depth s.
constexpr int kPromptWaves = 4;
constexpr int kPromptRows = 32 * kPromptWaves;
// A workgroup has its CU to itself at D = 256 (registers; at 128 and 64 two would fit). If a call has less than half as many
// of them as the card has CUs, each one's keys are cut into pieces of at least kPromptMinTiles tiles, up to one piece a CU
// (777 rows behind 1500 keys: 98 workgroups 125 us, 196 pieces 88 when this was built, 72 now; a call with 16 rows behind
// 2500 keys 39 us with pieces of 8 tiles, 35 of 4).
constexpr int kPromptFill = 256;
constexpr int kPromptMinTiles = 4;
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
__global__ __launch_bounds__(kPromptWaves* kWave, 1) void prompt_kernel(const AttnArgs a) {
    constexpr int ND = D / 16, DT = D / 32, NTH = kPromptWaves * kWave;
    constexpr int UK = D > 128 ? D / 128 : 1;   // a lane's 16-byte pieces of a tile's keys, and of its values
    __shared__ __align__(16) f16x8_t ks[2][ND][kWave];
    __shared__ __align__(16) f16x8_t vs[2][DT][2][kWave];
    __shared__ float scl[2][4][4];   // [key, value][tile % 4][octet]
    // which request, KV head and row tile: the last row tiles (the longest rows) first
    const int G = a.group, lane = threadIdx.x & 63, col = lane & 31, g = lane >> 5;
    auto tiles_here = [&](int b) -> int64_t {   // workgroups of a request, before they are cut
        if (b >= a.requests) return 0;
        const Request r = request(a, b);
        return takes_split(a, r) ? 0 : (static_cast<int64_t>(r.n) * G + kPromptRows - 1) / kPromptRows * a.c.heads;
    };
    int64_t total = 0;
    for (int b0 = 0; b0 < a.requests; b0 += kWave) total += tiles_here(b0 + lane);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) total += __shfl_xor(total, o);
    if (total == 0) return;   // the whole workgroup
    const int splits = total < kPromptFill ? static_cast<int>(kPromptFill / total) : 1;
    int b = -1;
    int64_t item = blockIdx.x / static_cast<unsigned>(splits);
    const int split = static_cast<int>(blockIdx.x % static_cast<unsigned>(splits));
    for (int b0 = 0; b0 < a.requests && b < 0; b0 += kWave) {
        const int64_t n = tiles_here(b0 + lane);
        const int64_t upto = wave_prefix(n, lane);
        const uint64_t hit = __ballot(item < upto);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            item -= __shfl(upto, l) - __shfl(n, l);
            b = __builtin_amdgcn_readfirstlane(b0 + l);
        } else {
            item -= __shfl(upto, 63);
        }
    }
    if (b < 0) return;   // the whole workgroup
    const Request r = request(a, b);
    const int pairs = r.n * G, tiles = (pairs + kPromptRows - 1) / kPromptRows;
    const int unit = __builtin_amdgcn_readfirstlane(static_cast<int>(item));
    const int h = unit % a.c.heads, rt = tiles - 1 - unit / a.c.heads;
    const int wv = wave_in_block(), tid = threadIdx.x;
    const int row0 = rt * kPromptRows + 32 * wv;             // the wave's first pair
    const int rr = min(row0 + col, pairs - 1);
    const int ti = rr / G, head = h * G + (rr - ti * G);
    const int limit = r.len - r.n + ti;
    const int wave_first = r.len - r.n + min(row0, pairs - 1) / G;
    const int seen = max(r.len - r.n + min(rt * kPromptRows + kPromptRows - 1, pairs - 1) / G + 1, 0);
    const int all_steps = (seen + 31) / 32, pieces = min(splits, max(all_steps / kPromptMinTiles, 1));
    if (split >= pieces) return;   // the whole workgroup
    const int per = (all_steps + pieces - 1) / pieces;
    const int first_tile = split * per, steps = max(min(per, all_steps - first_tile), 0);   // this piece's tiles
    const int block_shift = a.page_shift + (D == 64 ? 6 : D == 128 ? 7 : 8);   // of a page and head, as a power of two

    // A wave brings one octet of tokens of each tile: page, offset and scales are the same for its lanes. A lane's pieces:
    // keys (token lane % 8, 16 dims), values (pair of dims 2 lane); at D = 64 half of the lanes have one. Octets past the
    // last are loaded from page 0 and never read from LDS. Page ids are read a tile ahead of the codes they lead to.
    uint4 kr[UK], vr[UK];
    float ksr = 0.f, vsr = 0.f;   // the octet's two scales
    bool sdead = false, sbad = false;
    const bool some = D > 64 || lane < 32;
    const uint32_t ko = static_cast<uint32_t>((lane & 7) * D + 16 * (some ? lane >> 3 : 0)), vo = 16 * (some ? lane : 0);
    int id = 0;
    size_t off[3];   // of the octet in tiles st + 1, st + 2, st + 3
    auto next_id = [&](int st) {   // the table's entry for the octet (any in-bounds entry past the row's end)
        id = a.table[static_cast<size_t>(b) * a.max_pages + min((32 * (first_tile + st) + 8 * wv) >> a.page_shift, a.max_pages - 1)];
    };
    auto k_load = [&](int st) {
        const int tok = 32 * (first_tile + st) + 8 * wv, page = __builtin_amdgcn_readfirstlane(id);
        sdead = tok >= seen;
        sbad = !sdead && (page < 0 || page >= a.c.pages);
        const size_t base = static_cast<size_t>(static_cast<uint32_t>(sdead || sbad ? 0 : page)) * a.c.heads + h;
        off[0] = off[1];
        off[1] = off[2];
        off[2] = (base << block_shift) + static_cast<uint32_t>((tok & (a.c.page - 1)) * D);
        const int8_t* p = a.c.k + off[2];
#pragma unroll
        for (int i = 0; i < UK; ++i) kr[i] = ld16(p + ko + 128 * i);
        ksr = a.c.ks[base];
        vsr = a.c.vs[base];
    };
    auto v_load = [&](int n) {   // n: how many tiles behind the keys
        const int8_t* p = a.c.v + off[2 - n];
#pragma unroll
        for (int i = 0; i < UK; ++i) vr[i] = ld16(p + vo + 1024 * i);
    };
    // piece 2 i + half of the keys / of the values to LDS; dim 64 m + 2 r + e is row r of value tile 2 m + e
    constexpr int PIECES = 2 * UK;
    const int ktok = 8 * wv + (lane & 7), rho = (ktok & 16) + 8 * ((ktok >> 2) & 1) + 4 * ((ktok >> 3) & 1) + (ktok & 3);
    auto k_put = [&](int st, int piece) {
        const int i = piece >> 1;
        const f16x8_t x = piece & 1 ? codes8(kr[i].z, kr[i].w) : codes8(kr[i].x, kr[i].y);
        if (some) ks[st & 1][(lane >> 3) + 8 * i][32 * (piece & 1) + rho] = x;
    };
    auto v_put = [&](int st, int piece) {
        const int i = piece >> 1;
        const f16x8_t x = piece & 1 ? codes8(vr[i].z, vr[i].w) : codes8(vr[i].x, vr[i].y);
        if (some) vs[st & 1][2 * (lane >> 5) + 4 * i + (piece & 1)][wv >> 1][32 * (wv & 1) + (lane & 31)] = x;
    };
    auto s_put = [&](int st) {   // (the same values from every lane)
        scl[0][st & 3][wv] = sbad ? __builtin_nanf("") : sdead ? 0.f : ksr;
        scl[1][st & 3][wv] = sdead ? 0.f : vsr;
    };
    auto k_store = [&](int st) {
#pragma unroll
        for (int i = 0; i < PIECES; ++i) k_put(st, i);
        s_put(st);
    };
    auto barrier = []() {   // LDS is written and read; the loads stay in flight
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    if (steps > 0) {
        next_id(0);
        off[1] = off[2] = 0;
        k_load(0);
        next_id(1);
        v_load(0);
    }
    // the row's query, times 2^e, in two parts: dims 16 d + 8 g + 0..7 of depth d
    f16x8_t Qh[ND], Ql[ND];
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
        float m = 0.f;
        bool bad = false;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                m = fmaxf(m, fabsf(f[d][i]));
                bad |= !(fabsf(f[d][i]) <= FLT_MAX);
            }
        if (bad) m = INFINITY;
        m = fmaxf(m, __shfl_xor(m, 32));
        const bool ok = m <= FLT_MAX;
        int e = 0;
        if (m > 0.f && ok) {
            int em;
            frexpf(m, &em);
            e = 15 - em;
        }
#pragma unroll
        for (int d = 0; d < ND; ++d) {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float v = ok ? ldexpf(f[d][i], e) : 0.f;
                Qh[d][i] = static_cast<_Float16>(v);
                Ql[d][i] = static_cast<_Float16>(low_part(v));
            }
        }
        factor = ok ? ldexpf(a.scale, -e) : __builtin_nanf("");
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
    float mu = -FLT_MAX, l = 0.f;
    f32x16_t S, N;          // a tile's scores, scaled; the next tile's
    f16x8_t Wh[2], Wl[2];   // weights of the last tile
    // The operands of a step's products are one sequence, the last tile's values (2 DT of them), then the next tile's keys
    // (ND = 2 DT); each is requested AP products' pairs ahead, into the register that the one before it has left. fill(i) goes
    // between the two products of an operand and after them.
    constexpr int AP = 4;
    f16x8_t A[AP];
    auto value_at = [&](int slot, int k) { return vs[slot][k >> 1][k & 1][lane]; };
    auto key_at = [&](int slot, int d) { return ks[slot][d][lane]; };
    // ahead(d): what to request when operand d has been taken
    auto scores = [&](auto&& ahead, auto&& fill) {
        static_for<ND>([&](auto dI) {
            constexpr int d = decltype(dI)::value;
            const f16x8_t x = A[d % AP];
            if constexpr (d == 0) {
                f32x16_t z;
#pragma unroll
                for (int i = 0; i < 16; ++i) z[i] = 0.f;
                N = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Qh[d], z, 0, 0, 0);
            } else {
                N = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Qh[d], N, 0, 0, 0);
            }
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
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Wh[s], acc[d], 0, 0, 0);
            fill(IC<2 * k>{});
            __builtin_amdgcn_sched_barrier(0);
            acc[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, Wl[s], acc[d], 0, 0, 0);
            ahead(kI);
            fill(IC<2 * k + 1>{});
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    for (int i = tid; i < DT * 2 * kWave; i += NTH) (&vs[1][0][0][0])[i] = f16x8_t{};   // the values before the first tile
#pragma unroll
    for (int s = 0; s < 2; ++s) Wh[s] = Wl[s] = f16x8_t{};
    if (steps > 0) {
        k_store(0);
        k_load(1);
        next_id(2);
        barrier();
        static_for<AP>([&](auto dI) { A[decltype(dI)::value] = key_at(0, decltype(dI)::value); });
        scores([&](auto dI) {
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
    // Step st: the scores of tile st are in S. Its values and the keys of st + 2 go to LDS (slots whose last readers passed
    // the barrier before); the values of st - 1 are summed beside that and beside the scaling and maximum of the scores, the
    // scores of st + 1 beside the exponentials. One step more than tiles; before the first the weights are zero.
    float f[2], sv[2], top[2], w0 = 0.f;
    auto scale_max = [&](int i) {
        S[i] = N[i] * f[i >> 3];
        top[i >> 3] = (i & 7) ? fmaxf(top[i >> 3], S[i]) : S[i];
        asm volatile("" : "+v"(S[i]), "+v"(top[i >> 3]));   // here, not where they are used
    };
    auto weight = [&](int i) {
        const float p = __builtin_amdgcn_exp2f(S[i] - mu);
        l += p;
        const float w = rounded(p * (sv[i >> 3] * kWeightUp));
        if (i & 1) {
            Wh[i >> 3][(i & 7) - 1] = static_cast<_Float16>(w0);
            Wh[i >> 3][i & 7] = static_cast<_Float16>(w);
            Wl[i >> 3][(i & 7) - 1] = static_cast<_Float16>(low_part(w0));
            Wl[i >> 3][i & 7] = static_cast<_Float16>(low_part(w));
        }
        w0 = w;
    };
    for (int st = 0; steps > 0 && st <= steps; ++st) {
        {
#pragma unroll
            for (int s = 0; s < 2; ++s) f[s] = factor * scl[0][st & 3][2 * s + g];
            constexpr int SLOTS = 4 * DT, PER = 32 / SLOTS;   // places between products; scores at a place of the second half
            values([&](auto kI) {
                constexpr int k = decltype(kI)::value;
                A[k % AP] = k + AP < ND ? value_at((st + 1) & 1, k + AP) : key_at((st + 1) & 1, k + AP - ND);
            }, [&](auto kI) {
                constexpr int k = decltype(kI)::value;
                constexpr int EVERY = SLOTS / (4 * PIECES);   // a piece to LDS at every so many places of the first half
                if constexpr (k < SLOTS / 2 && k % EVERY == 0) {
                    if constexpr ((k / EVERY) & 1)
                        k_put(st + 2, (k / EVERY) >> 1);
                    else
                        v_put(st, (k / EVERY) >> 1);
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
                    for (int i = (k - SLOTS / 2) * PER; i < (k - SLOTS / 2 + 1) * PER; ++i) scale_max(i);
                }
            });
        }
        {
            const int t0 = 32 * (first_tile + st);
#pragma unroll
            for (int s = 0; s < 2; ++s) sv[s] = scl[1][st & 3][2 * s + g];
            if (t0 + 31 > wave_first || st == steps) {   // past the piece's last tile nothing is seen
                const int last = st == steps ? -1 : limit;
#pragma unroll
                for (int s = 0; s < 2; ++s) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if (t0 + 16 * s + 8 * g + i > last) S[8 * s + i] = -INFINITY;
                        top[s] = i ? fmaxf(top[s], S[8 * s + i]) : S[8 * s];
                    }
                    if (t0 + 16 * s + 8 * g > last) sv[s] = 0.f;   // a page that the row does not see may be marked
                }
            }
#pragma unroll
            for (int s = 0; s < 2; ++s) top[s] += __builtin_amdgcn_logf(reference_scale(sv[s]));
            const float hi = fmaxf(top[0], top[1]);
            if (__ballot(hi > mu + kMoves)) {
                const float now = fmaxf(mu, fmaxf(hi, __shfl_xor(hi, 32)));
                const float shrink = __builtin_amdgcn_exp2f(mu - now);
                mu = now;
                l *= shrink;
#pragma unroll
                for (int d = 0; d < DT; ++d)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[d][i] *= shrink;
            }
            // (past the wave's last tile these scores are of an old one, and unused)
            scores([&](auto dI) {
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
                for (int i = k * 16 / PLACES; i < (k + 1) * 16 / PLACES; ++i) weight(i);
            });
        }
    }
    l += __shfl_xor(l, 32);
    if (row0 + col >= pairs) return;
    if (r.bad) l = __builtin_nanf("");
    const size_t o = (static_cast<size_t>(r.first + ti) * a.heads + head) * D;
    if (pieces > 1) {   // row k of the tile is slot k % kRows of item first + k / kRows * splits + piece, as combine_kernel reads
        const int k = 32 * wv + col;
        const int unit_items = static_cast<int>(blockIdx.x) / splits * (kPromptRows / kRows);
        const int item0 = a.items + (unit_items + k / kRows) * splits;
        const size_t row = static_cast<size_t>(item0 + split) * kRows + k % kRows;
#pragma unroll
        for (int m = 0; m < DT / 2; ++m)
#pragma unroll
            for (int n = 0; n < 8; ++n) {
                const int q = 4 * (n >> 1) + 2 * (n & 1);
                st4(a.part + row * D + 64 * m + 8 * g + 16 * (n >> 1) + 4 * (n & 1),
                    make_float4(acc[2 * m][q], acc[2 * m + 1][q], acc[2 * m][q + 1], acc[2 * m + 1][q + 1]));
            }
        if (g == 0) {
            a.stat[row] = make_float2(mu, l);
            if (split == 0) a.info[o / D] = make_int2(item0 * kRows + k % kRows, pieces);
        }
        return;
    }
    // (l is about 1 / value scale a key: from 2^-60 with the largest scales that the header allows to 2^108 a key at the
    // smallest, where values below 2^-93 come out as 0 once 64 l overflows. 2^-24 more beside the sums' roundings.)
    const float inv = 1.f / (kWeightUp * l);
    // A lane's registers 4 b .. 4 b + 3 of value tiles 2 m and 2 m + 1 are dims 64 m + 16 b + 8 g + 0..7 of its row. (One row's
    // gates after another's, each load waited for, were a third of the kernel's time.)
#pragma unroll
    for (int m = 0; m < DT / 2; ++m) {
        const size_t at = o + 64 * m + 8 * g;
        float4 gt[4][2];
        if (a.gate) {
#pragma unroll
            for (int n = 0; n < 8; ++n) gt[n >> 1][n & 1] = ld4(a.gate + at + 16 * (n >> 1) + 4 * (n & 1));
        }
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            float v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float x = acc[2 * m + (i & 1)][4 * (n >> 1) + 2 * (n & 1) + (i >> 1)];
                v[i] = l == 0.f ? 0.f : x * inv;
            }
            if (a.gate) {
                const float4 x = gt[n >> 1][n & 1];
                v[0] *= sigmoid(x.x);
                v[1] *= sigmoid(x.y);
                v[2] *= sigmoid(x.z);
                v[3] *= sigmoid(x.w);
            }
            st4(a.out + at + 16 * (n >> 1) + 4 * (n & 1), make_float4(v[0], v[1], v[2], v[3]));
        }
    }
    if (g == 0) a.info[o / D] = make_int2(0, 1);
}

// ------------------------------------------------------------------ host
// Whether a call can have requests for prompt_kernel; if not, split_kernel takes them all. A call with no more rows than
// requests is taken for a batch of single tokens, up to kSplitOnly (row, head) pairs of a KV head, and spared the launch
// (us: 64 tokens at 500 keys 21.1 -> 19.3, 128 31.6 -> 29.9, before the queries' parts were shared; 17.5 and 28.7 with
// that). Should one request have all the rows, split_kernel answers it too (64 rows at 2500 keys among 64 requests: 39, with
// prompt_kernel 44), if at long contexts not as fast (33 rows at 30000 keys 138, 67).
bool may_prompt(int rows, int requests, int group) {
    const int64_t pairs = static_cast<int64_t>(rows) * group;
    return rows > 1 && pairs > kSplitMax && (rows > requests || pairs > kSplitOnly);
}
// split_kernel's pieces are at most kTargetItems plus one per unit; units at most one per 8 pairs plus one per request that
// has rows, and, where larger requests go to prompt_kernel, at most one per 8 of the pairs with which one does not (plus one,
// so that the bound does not fall where the first request goes there).
int64_t unit_bound(int rows, int requests, int heads, int kv_heads) {
    const int group = heads / kv_heads;
    const int64_t pairs = static_cast<int64_t>(rows) * group, busy = std::min(rows, requests);
    int64_t units = pairs / kRows + busy;
    if (may_prompt(rows, requests, group)) units = std::min(units, busy * (blocks_for(std::max(kSplitMax, group), kRows) + 1));
    return units * kv_heads;
}
size_t align_up(size_t b) { return (b + 255) & ~size_t{255}; }

struct Layout {
    int64_t items, all;   // pieces of 8 rows: of split_kernel, and with those of prompt_kernel
    size_t stat, info, bytes;
};
Layout layout(int rows, int requests, int heads, int kv_heads, int dim) {
    Layout l;
    l.items = kTargetItems + unit_bound(rows, requests, heads, kv_heads);
    l.all = l.items;
    // Room for cut prompts by the rows alone, though a call with no more rows than requests has none: a workspace for some
    // rows and requests has to serve fewer of either.
    if (rows > 1 && static_cast<int64_t>(rows) * (heads / kv_heads) > kSplitMax) l.all += kPromptFill * (kPromptRows / kRows);
    l.stat = align_up(static_cast<size_t>(l.all) * kRows * dim * 4);
    l.info = l.stat + align_up(static_cast<size_t>(l.all) * kRows * 8);
    l.bytes = l.info + align_up(static_cast<size_t>(rows) * heads * 8);
    return l;
}

template <int D>
void launch(const AttnArgs& a, hipStream_t s) {
    split_kernel<D><<<static_cast<unsigned>(a.items), kSplitBlock, 0, s>>>(a);
    if (!a.split_all) {
        const int64_t pairs = static_cast<int64_t>(a.rows) * a.group;
        const int64_t tiles = (pairs / kPromptRows + std::min<int64_t>(a.requests, pairs / kSplitMax + 1)) * a.c.heads;
        prompt_kernel<D><<<static_cast<unsigned>(std::max<int64_t>(tiles, kPromptFill)), kPromptWaves * kWave, 0, s>>>(a);
    }
    const unsigned pairs = static_cast<unsigned>(a.rows) * static_cast<unsigned>(a.heads);
    if (pairs <= 128)   // few rows: many pieces each
        combine_kernel<D, 16><<<pairs, 16 * kWave, 0, s>>>(a, 1);
    else if (pairs <= 2048)
        combine_kernel<D, 4><<<pairs, 4 * kWave, 0, s>>>(a, 1);
    else if (pairs <= kPromptFill / 2 * kPromptRows)   // a cut prompt's pairs may all have pieces
        combine_kernel<D, 1><<<blocks_for(pairs, 4), 4 * kWave, 0, s>>>(a, 1);
    else
        combine_kernel<D, 1><<<blocks_for(pairs, 16), 4 * kWave, 0, s>>>(a, 4);
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qwen_attn_kv8_workspace_bytes(int rows, int requests, int heads, int kv_heads, int dim) {
    if (rows <= 0 || requests <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dim <= 0) return 0;
    return layout(rows, requests, heads, kv_heads, dim).bytes;
}

int qwen_attn_kv8_rows(const float* q, const int8_t* k_codes, const int8_t* v_codes, const float* k_scale,
                       const float* v_scale, int pages, int page_size, const int32_t* block_table, int max_pages,
                       const int32_t* row_start, const int32_t* kv_len, int requests, const float* gate, float* out, int rows,
                       int heads, int kv_heads, int dim, void* workspace, size_t workspace_bytes, void* stream) {
    const Kv8Cache c{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes), const_cast<float*>(k_scale),
                     const_cast<float*>(v_scale), pages, page_size, kv_heads, dim};
    if (const int rc = kv8_check("attn_kv8_rows", c)) return rc;
    QK_REQUIRE(heads > 0 && heads % kv_heads == 0, "attn_kv8_rows: %d query heads over %d KV heads", heads, kv_heads);
    QK_REQUIRE(rows >= 0 && requests >= 0 && max_pages >= 0, "attn_kv8_rows: negative size");
    QK_REQUIRE(requests <= kKv8MaxRequests, "attn_kv8_rows: %d requests (at most %d)", requests, kKv8MaxRequests);
    // (tokens a few tiles past a row's end are computed in 32 bits too)
    QK_REQUIRE(static_cast<int64_t>(max_pages) * page_size <= (1 << 30), "attn_kv8_rows: table rows of %d pages", max_pages);
    if (rows == 0 || requests == 0) return ok();
    QK_REQUIRE(q && out && row_start && kv_len && (block_table || max_pages == 0), "attn_kv8_rows: null pointer");
    QK_REQUIRE(static_cast<int64_t>(rows) * heads <= (int64_t{1} << 24), "attn_kv8_rows: %d rows of %d heads exceed one call",
               rows, heads);
    QK_REQUIRE(aligned16(q) && aligned16(out) && (!gate || aligned16(gate)),
               "attn_kv8_rows: q, gate and out must be 16-byte aligned");
    const size_t row_bytes = static_cast<size_t>(rows) * heads * dim * 4;
    QK_REQUIRE(apart(out, row_bytes, q, row_bytes), "attn_kv8_rows: out is q or overlaps it");
    QK_REQUIRE(!gate || gate == out || apart(out, row_bytes, gate, row_bytes), "attn_kv8_rows: out overlaps gate out of place");
    const Layout l = layout(rows, requests, heads, kv_heads, dim);
    QK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= l.bytes,
               "attn_kv8_rows: workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, l.bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    AttnArgs a;
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
    a.split_all = !may_prompt(rows, requests, a.group);
    a.part = reinterpret_cast<float*>(ws);
    a.stat = reinterpret_cast<float2*>(ws + l.stat);
    a.info = reinterpret_cast<int2*>(ws + l.info);
    a.items = static_cast<int>(l.items);
    a.all_items = static_cast<int>(l.all);
    a.scale = static_cast<float>(1.4426950408889634 / std::sqrt(static_cast<double>(dim)));
    const hipStream_t s = as_stream(stream);
    if (dim == 64)
        launch<64>(a, s);
    else if (dim == 128)
        launch<128>(a, s);
    else
        launch<256>(a, s);
    return check_launch("attn_kv8_rows");
}

}  // extern "C"
