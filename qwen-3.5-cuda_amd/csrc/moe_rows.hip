// The routed experts of many tokens on gfx950: (token, pick) pairs grouped by expert, then
//   hidden[p] = SiLU(Wg_e x_t) * (Wu_e x_t),  out[t] = sum_j w[t][j] Wd_e hidden[t k + j],   p = t k + j, e = idx[p]
// with K-quant weights of n_experts matrices each. The reference runs the experts of one token one after the other
// (src/layer_moe.cpp:127-142), five launches each; here every expert's rows go through it together.
//
// The products are gemm.hip's: x as two fp16 parts per row, weights as exact small integers in fp16, block scales in fp32
// (the mathematics stands there). What differs is the shape of the work: 256 products with a few to a few hundred rows
// each. A tile is up to 16 WT pairs of one expert, a table of tiles is written by the first launch from the experts'
// starts, and a workgroup takes a tile and a slice of the expert's rows. Rows of x are gathered by pair: their fp16 parts
// lie row by row, 128 bytes per depth of 32 elements, so a gathered operand is still whole cache lines. The hidden rows
// are kept in the order of the groups, so the down products read neighbouring rows and only the last step scatters.
#include <algorithm>
#include <cfloat>
#include <type_traits>

#include "capi_common.hpp"
#include "device_common.hpp"
#include "gemm_common.hpp"
#include "ggml_common.hpp"

namespace qk {
namespace {

constexpr int kMaxExperts = 1024;
constexpr int kGroupBlock = 1024;

// ------------------------------------------------------------------ grouping
// A stable counting sort in one launch: workgroup w places pairs [1024 w, 1024 w + 1024), one to a thread. Each counts
// all pairs' experts itself (LDS counters: integer sums, the same in any order), and those of the pairs before its own, so no
// workgroup waits for another; ranks among its own pairs come from ballots on the bits of the id (lanes of the wave with
// the same expert) and per-wave counts. Ids outside [0, n) go behind the last group.
__global__ __launch_bounds__(kGroupBlock) void group_kernel(const int32_t* __restrict__ idx, int pairs, int n,
                                                            int32_t* __restrict__ order, int32_t* __restrict__ starts) {
    __shared__ int all[kMaxExperts + 1], before[kMaxExperts + 1];
    __shared__ uint16_t mine[kGroupBlock / kWave][kMaxExperts + 2];
    __shared__ int part[kGroupBlock / kWave];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int first = blockIdx.x * kGroupBlock;
    for (int e = tid; e <= n; e += kGroupBlock) all[e] = before[e] = 0;
    for (int e = lane; e <= n; e += kWave) mine[wv][e] = 0;
    __syncthreads();
    auto bucket = [&](int i) {
        const int e = idx[i];
        return e >= 0 && e < n ? e : n;
    };
    constexpr int AHEAD = 8;   // ids requested before the first is counted
    for (int i0 = tid; i0 < pairs; i0 += AHEAD * kGroupBlock) {
        int e[AHEAD];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) e[j] = bucket(min(i0 + j * kGroupBlock, pairs - 1));
#pragma unroll
        for (int j = 0; j < AHEAD; ++j) {
            const int i = i0 + j * kGroupBlock;
            if (i < pairs) atomicAdd(i < first ? &before[e[j]] : &all[e[j]], 1);
        }
    }
    const int p = first + tid;
    const bool in = p < pairs;
    const int e = in ? bucket(p) : n + 1;   // n + 1: no pair
    uint64_t same = ~0ull;
    for (int bit = 0; (1 << bit) <= n + 1; ++bit) {
        const uint64_t set = __ballot((e >> bit) & 1);
        same &= (e >> bit) & 1 ? set : ~set;
    }
    const int rank = __popcll(same & ((1ull << lane) - 1));
    if (in && rank == 0) mine[wv][e] = static_cast<uint16_t>(__popcll(same));
    __syncthreads();
    // exclusive prefix of all[0 .. n], a bucket to a thread (n <= 1024; bucket n needs only the sum before it)
    const int c = tid < n ? all[tid] + before[tid] : 0;   // (the pairs before this workgroup's were counted apart)
    int inc = c;
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) {
        const int up = __shfl_up(inc, o);
        if (lane >= o) inc += up;
    }
    if (lane == 63) part[wv] = inc;
    __syncthreads();
    int base = 0, total = 0;
    for (int w = 0; w < kGroupBlock / kWave; ++w) {
        if (w < wv) base += part[w];
        total += part[w];
    }
    if (tid < n) all[tid] = base + inc - c;
    if (tid == 0) all[n] = total;
    __syncthreads();
    if (blockIdx.x == 0)
        for (int i = tid; i <= n; i += kGroupBlock) starts[i] = all[i];
    if (!in) return;
    int at = all[e] + before[e] + rank;
    for (int w = 0; w < wv; ++w) at += mine[w][e];
    order[at] = p;
}

// ------------------------------------------------------------------ tiles, x in two fp16 parts
struct Tile {
    int expert, first, n;   // pairs order[first .. first + n)
};

// Tiles of up to `size` pairs, expert by expert; the count in tiles[-1].expert. One workgroup of 256 threads, an expert to
// each (one wave took 4 us for 256 experts).
__device__ void write_tiles(const int32_t* __restrict__ starts, int experts, int pairs, int size, Tile* __restrict__ tiles,
                            int most) {
    __shared__ int part[2][4];
    const int lane = threadIdx.x & 63, wv = wave_in_block();
    int at = 0;
    for (int e0 = 0, turn = 0; e0 < experts; e0 += 256, turn ^= 1) {
        const int e = e0 + static_cast<int>(threadIdx.x);
        int s = 0, n = 0;
        if (e < experts) {
            const int from = starts[e], to = starts[e + 1];
            s = min(max(from, 0), pairs);
            n = min(max(to, s), pairs) - s;
        }
        // of several tiles of 16 pairs each: even ones, whole sixteens
        const int even = (n + size - 1) / size, one = size <= 16 || n == 0 ? size : ((n + even - 1) / even + 15) / 16 * 16;
        const int k = (n + one - 1) / one;
        int inc = k;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const int up = __shfl_up(inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 63) part[turn][wv] = inc;
        __syncthreads();   // (two sets of sums: the next turn's are written while a slow wave still reads these)
        for (int w = 0; w < 4; ++w) {
            if (w == wv) inc += at;
            at += part[turn][w];
        }
        for (int i = 0; i < k; ++i) {
            const int slot = inc - k + i;
            if (slot < most) tiles[slot] = Tile{e, s + i * one, min(one, n - i * one)};
        }
    }
    if (threadIdx.x == 0) tiles[-1] = Tile{min(at, most), 0, 0};
}

// Pair at a place of the order, inside the call's pairs whatever the array holds.
__device__ __forceinline__ int pair_at(const int32_t* __restrict__ order, int pos, int pairs) {
    return min(max(order[pos], 0), pairs - 1);
}

// A wave per row: exponent, group sums and parts, [row][depth of 32][part][lk][8 elements] (gemm.hip's order of the
// elements in a block). The last workgroup of the first launch (x) writes the table of tiles, the one of the second
// launch (hidden rows) marks the tokens that have a pair behind the last group: their output is NaN.
struct Grouping {
    const int32_t* order;
    const int32_t* starts;
    Tile* tiles;
    int* lost;   // per token
    int experts, pairs, top, size, most;
};
template <bool FIRST>
__global__ __launch_bounds__(256) void rows_prep(const float* __restrict__ x, int rows, int K, int* __restrict__ ex,
                                                 float* __restrict__ sx, uint8_t* __restrict__ xp, const Grouping gr) {
    const int wv = wave_in_block(), lane = threadIdx.x & 63;
    if (blockIdx.x == gridDim.x - 1) {
        if constexpr (FIRST) {
            write_tiles(gr.starts, gr.experts, gr.pairs, gr.size, gr.tiles, gr.most);
        } else {
            for (int q = max(gr.starts[gr.experts], 0) + static_cast<int>(threadIdx.x); q < gr.pairs; q += 256)
                gr.lost[pair_at(gr.order, q, gr.pairs) / gr.top] = 1;
        }
        return;
    }
    const int r = blockIdx.x * 4 + wv;
    if (r >= rows) return;
    if (FIRST && lane == 0) gr.lost[r] = 0;
    const float* row = x + static_cast<size_t>(r) * K;
    float m = 0.f;
#pragma unroll 4
    for (int k = 8 * lane; k < K; k += 512) m = max_abs4(max_abs4(m, ld4(row + k)), ld4(row + k + 4));
    const int e = prep_exponent(wave_max_abs(m)), es = e == kRowNonFinite ? 0 : e;
    if (lane == 0) ex[r] = e;
    const int c = lane & 31;   // chunk of 8 in the block: 16 (lk / 2) + 4 u + 2 (lk % 2) + j, depth 2 u + j
    const int depth = 2 * ((c >> 2) & 3) + (c & 1), lk = 2 * (c >> 4) + ((c >> 1) & 1);
    uint8_t* out = xp + static_cast<size_t>(r) * K * 4 + 128 * depth + 16 * lk;
#pragma unroll 4
    for (int k = 8 * lane; k < K; k += 512) {
        uint32_t h[4], l[4];
        float s = split8(ld4(row + k), ld4(row + k + 4), es, h, l);
        uint8_t* o = out + 1024 * (k >> 8);
        st16(o, make_uint4(h[0], h[1], h[2], h[3]));
        st16(o + 64, make_uint4(l[0], l[1], l[2], l[3]));
        s += __shfl_xor(s, 1);
        s += __shfl_xor(s, 2);
        if ((lane & 3) == 0) sx[static_cast<size_t>(r) * (K >> 5) + (k >> 5)] = s;
    }
}

// ------------------------------------------------------------------ the products
// v[rt][i] = f, rt and i not known at compile time (a register array).
__device__ __forceinline__ void replace(f32x4_t (&v)[2], int rt, int i, float f) {
#pragma unroll
    for (int q = 0; q < 8; ++q)
        if (q == 4 * rt + i) v[q >> 2][q & 3] = f;
}

// A block of a weight row between memory and the lanes that use it: the 16-byte pieces that it lies in, and a lane's share
// (WBlock, as load() would bring it) from a copy of them in LDS. Q6_K blocks begin at any even byte.
template <int TYPE>
struct Staged;
template <>
struct Staged<kQ4_K> {
    static constexpr int pieces = 9;
    static __device__ __forceinline__ void take(WBlock<kQ4_K>& w, const uint4* row, uint32_t, int lk) {
        const uint4* p = row + 1 + 4 * (lk >> 1) + (lk & 1);
        w.hd = row[0];
        w.q[0] = p[0];
        w.q[1] = p[2];
    }
};
template <>
struct Staged<kQ6_K> {
    static constexpr int pieces = 14;   // up to 14 bytes before a block's 210
    static __device__ __forceinline__ void take(WBlock<kQ6_K>& w, const uint4* row, uint32_t skew, int lk) {
        const uint32_t h = lk >> 1, l = lk & 1;
        auto words = [&](uint32_t byte, auto n, uint32_t* d) {   // n words from a byte that is 0 or 2 past a word
            constexpr int N = decltype(n)::value;
            const uint32_t* p = reinterpret_cast<const uint32_t*>(row) + ((byte + skew) >> 2);
            uint32_t v[N + 1];
#pragma unroll
            for (int i = 0; i <= N; ++i) v[i] = p[i];
#pragma unroll
            for (int i = 0; i < N; ++i) d[i] = __builtin_amdgcn_alignbyte(v[i + 1], v[i], skew & 2u);
        };
        uint32_t d[4];
        words(64u * h + 16u * l, IC<4>{}, d);
        w.q[0] = make_uint4(d[0], d[1], d[2], d[3]);
        words(64u * h + 16u * l + 32u, IC<4>{}, d);
        w.q[1] = make_uint4(d[0], d[1], d[2], d[3]);
        words(128u + 32u * h + 16u * l, IC<4>{}, d);
        w.qh = make_uint4(d[0], d[1], d[2], d[3]);
        words(192u + 8u * h, IC<2>{}, d);
        w.sc = make_uint2(d[0], d[1]);
        w.d = reinterpret_cast<const uint16_t*>(row)[(208u + skew) >> 1];
    }
};

struct RowsArgs {
    const uint8_t* w[2];   // gate and up, or down
    const Tile* tiles;     // tiles[-1].expert: how many
    const int32_t* order;
    const int* ex;
    const float* sx;
    const uint8_t* xp;
    const float* x;        // the rows in fp32, for those with an infinity
    float* y;
    int M, K, top, pairs, column_blocks;   // M: rows of an expert's matrix; top: pairs per row of x (gate and up)
};

// 4 waves; a wave owns the tile's 16 WT pairs x 32 weight rows: 16 gate and the same 16 up rows (SWIGLU), or 32 down rows,
// over the whole of K. Operands, pipeline and fold as gemm_kquant's (gemm.hip), but:
// A tile has one to kMaxTokenTiles sixteens of pairs and takes the code for its number of them (a group of 24 pairs in the
// code for 64 spent two thirds of its products on nothing).
// Loads ask for 64 neighbouring bytes with 4 neighbouring lanes. With the lanes in the operand's order, 16 rows apart from
// each other, every lane was an access of its own to the first cache, which was then busy 84% of the time (100 accesses a load
// at Q6_K's odd addresses). So x is laid into LDS by rows, with the 4 pieces of a row turned by its number, because a read
// takes 16 lanes at once, 8 of two neighbouring lane groups each; and a wave's weights pass through LDS too, where each lane
// finds its share; nobody else reads them, so that takes no barrier.
// Two workgroups share a CU, one's start and end beside the other's steps: they are a third of a workgroup's time at K = 512.
// Together (us, gate and up / down): 777 tokens Q6_K 355 / 237 -> 216 / 135, 4096 tokens Q4_K 585 / 364 -> 477 / 307.
constexpr int kRowsWaves = 4;
constexpr int kMaxTokenTiles = 4;   // of 16 pairs, in a tile (5 and 6 do not fit the registers)

template <int WT, bool SWIGLU>
struct RowsShape {
    static constexpr int FR = WT * 4, XF = FR / kRowsWaves, cols = (SWIGLU ? 16 : 32) * kRowsWaves;   // cols divides M
    static constexpr size_t ring = size_t{3} * FR * 1024;
};

template <int TYPE, int WT, bool SWIGLU>
__device__ __forceinline__ void rows_tile(const RowsArgs& a, const Tile& tl, int cb, uint8_t* smem, int* ends) {
    using G = RowsShape<WT, SWIGLU>;
    constexpr int BB = TYPE == kQ4_K ? 144 : 210, NB = TYPE == kQ4_K ? 1 : 2, WR = 2;
    uint4* xs = reinterpret_cast<uint4*>(smem);
    const int M = a.M, K = a.K, n = tl.n;
    const int lane = threadIdx.x & 63, lr = lane & 15, lk = lane >> 4;
    const int wv = wave_in_block();
    const int nb = K >> 8, steps = 4 * nb, nst = K >> 5;
    const int c0 = cb * G::cols, r0 = c0 + (SWIGLU ? 16 : 32) * wv;   // the workgroup's and the wave's first row
    const uint64_t eb = (static_cast<uint64_t>(tl.expert) * M + c0) * nb;
    const uint8_t* wbase[WR];
#pragma unroll
    for (int rt = 0; rt < WR; ++rt) wbase[rt] = a.w[SWIGLU ? rt : 0] + eb * BB;
    auto xrow = [&](int i) {   // row of x of the tile's pair i (the last one again past the end)
        const int pos = tl.first + min(i, n - 1);
        return SWIGLU ? pair_at(a.order, pos, a.pairs) / a.top : pos;
    };
    uint32_t xo[G::XF];   // this wave's fragments of a step: fragment id -> (slice, tile, (depth, part))
#pragma unroll
    for (int i = 0; i < G::XF; ++i) {
        const int id = wv * G::XF + i;
        const int ti = id / 4;
        // in pieces of 16 bytes
        xo[i] = static_cast<uint32_t>(xrow(16 * ti + (lane >> 2))) * static_cast<uint32_t>(K / 4) + 4 * (id % 4) +
                ((lane & 3) ^ (-(lane >> 4) & 3));
    }
    uint4 xr[1][G::XF];
    auto x_load = [&](uint4 (&d)[G::XF], int st) {
#pragma unroll
        for (int i = 0; i < G::XF; ++i) d[i] = ld16(a.xp + static_cast<size_t>(xo[i]) * 16 + 256u * static_cast<uint32_t>(min(st, steps - 1)));
    };
    auto x_store = [&](const uint4 (&d)[G::XF], int slot) {
#pragma unroll
        for (int i = 0; i < G::XF; ++i) xs[(slot * G::FR + wv * G::XF + i) * 64 + lane] = d[i];
    };
    const uint4* as = xs + 4 * lr + (lk ^ (-(lr >> 2) & 3));
    constexpr int PT = WT < 2 ? WT : 2;
    f16x8_t An[PT][2];
    auto a_load = [&](f16x8_t (&d)[PT][2], int slot, int j, int t0) {
#pragma unroll
        for (int i = 0; i < PT; ++i)
#pragma unroll
            for (int p = 0; p < 2; ++p)
                d[i][p] = *reinterpret_cast<const f16x8_t*>(&as[(slot * G::FR + 4 * min(t0 + i, WT - 1) + 2 * j + p) * 64]);
    };
    auto barrier = []() {
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    uint32_t so[WT];
#pragma unroll
    for (int tt = 0; tt < WT; ++tt) so[tt] = static_cast<uint32_t>(xrow(16 * tt + lr)) * static_cast<uint32_t>(nst) + 2 * lk;

    f32x4_t acc[WT][WR], C[WT][WR];
#pragma unroll
    for (int tt = 0; tt < WT; ++tt)
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) acc[tt][rt] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    uint32_t k64 = 0x64006400u;
    asm volatile("" : "+v"(k64));
    using W = Staged<TYPE>;
    constexpr int WP = 32 * W::pieces, WI = (WP + 63) / 64;   // 16-byte pieces of the wave's 32 rows of a block
    uint4 wr[WI];
    uint32_t wo[WI];
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int id = min(64 * i + lane, WP - 1), row = id / W::pieces;
        wo[i] = static_cast<uint32_t>(r0 - c0 + (SWIGLU ? row & 15 : row)) * static_cast<uint32_t>(nb) * BB;
    }
    const uint32_t skew = static_cast<uint32_t>(eb * BB) & 15u;   // of the first row's block in its 16 bytes
    uint4* wl = reinterpret_cast<uint4*>(smem + G::ring) + wv * WP;
    WBlock<TYPE> wc[WR];
    WScale<TYPE> sc[WR];
    f16x8_t B[2][WR][NB];
    auto w_load = [&](int b) {   // block b of the wave's rows, as it lies in memory
        const uint32_t at = static_cast<uint32_t>(min(b, nb - 1)) * BB;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int id = min(64 * i + lane, WP - 1);
            const uint8_t* base = SWIGLU && id >= WP / 2 ? wbase[1] : wbase[0];
            wr[i] = ld16(base - skew + ((wo[i] + at + skew) & ~15u) + 16 * (id % W::pieces));
        }
    };
    auto w_store = [&]() {
#pragma unroll
        for (int i = 0; i < WI; ++i) wl[min(64 * i + lane, WP - 1)] = wr[i];
    };
    auto w_take = [&](int b) {   // a lane's share of it
        const uint32_t at = static_cast<uint32_t>(min(b, nb - 1)) * BB;
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) {
            const uint32_t row = static_cast<uint32_t>(r0 - c0 + (SWIGLU ? 0 : 16 * rt) + lr) * (static_cast<uint32_t>(nb) * BB);
            W::take(wc[rt], wl + (16 * rt + lr) * W::pieces, (row + at + skew) & 15u, lk);
        }
    };
    auto b_make = [&](auto dI) {
        constexpr int D = decltype(dI)::value;
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) {
            if constexpr ((D & 1) == 0) sc[rt].template set<(D >> 1)>(wc[rt], lk);
            decode<(D >> 1), (D & 1)>(wc[rt], sc[rt], k64, B[D & 1][rt]);
        }
    };
    w_load(0);
    x_load(xr[0], 0);
    w_store();
    w_load(1);
    w_take(0);
    x_store(xr[0], 0);
    x_load(xr[0], 1);
    x_store(xr[0], 1);
    x_load(xr[0], 2);
    b_make(IC<0>{});
    if (static_cast<int>(threadIdx.x) < 16 * WT) {   // for the epilogue
        ends[threadIdx.x] = a.ex[xrow(threadIdx.x)];
        const int pos = tl.first + min(static_cast<int>(threadIdx.x), n - 1);
        ends[16 * kMaxTokenTiles + threadIdx.x] = SWIGLU ? 0 : pair_at(a.order, pos, a.pairs);
    }
    barrier();
    a_load(An, 0, 0, 0);
    int s0 = 0, s1 = 1, s2 = 2;   // the ring's slots of steps st, st + 1, st + 2
    for (int b = 0; b < nb; ++b) {
        f16x4_t Bm[WR];
        float dsc[WR], dmn[WR];
        float2 sg[WT];
        if constexpr (TYPE == kQ4_K) {
#pragma unroll
            for (int rt = 0; rt < WR; ++rt) {
                Bm[rt] = min_weights(wc[rt].hd, lk);
                dsc[rt] = opaque(half_bits(wc[rt].hd.x & 0xffffu));
                dmn[rt] = opaque(-32.0f * half_bits(wc[rt].hd.x >> 16));
            }
#pragma unroll
            for (int tt = 0; tt < WT; ++tt) sg[tt] = *reinterpret_cast<const float2*>(a.sx + static_cast<size_t>(so[tt]) + 8 * b);
        } else {
#pragma unroll
            for (int rt = 0; rt < WR; ++rt) dsc[rt] = opaque(half_bits(wc[rt].d));
        }
        static_for<8>([&](auto dI) {
            constexpr int D = decltype(dI)::value, U = D >> 1, J = D & 1;
            const int st = 4 * b + U;
            if constexpr (D == 5) {   // the last block's share has been read
                w_store();
                w_load(b + 2);
            }
            if constexpr (J == 0) {
                x_store(xr[0], s2);
                x_load(xr[0], st + 3);
            }
            __builtin_amdgcn_sched_barrier(0);
            b_make(IC<(D + 1) & 7>{});
            static_for<(WT + 1) / 2>([&](auto pI) {
                constexpr int P0 = 2 * decltype(pI)::value, PN = P0 + 2 <= WT ? 2 : 1;
                f16x8_t A[2][2];
#pragma unroll
                for (int i = 0; i < PN; ++i) {
#pragma unroll
                    for (int p = 0; p < 2; ++p) A[i][p] = An[i][p];
                }
                if constexpr (P0 + 2 < WT)
                    a_load(An, s0, J, P0 + 2);
                else
                    a_load(An, J == 0 ? s0 : s1, J ^ 1, 0);
#pragma unroll
                for (int i = 0; i < PN; ++i)
#pragma unroll
                    for (int rt = 0; rt < WR; ++rt)
                        C[P0 + i][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(
                            A[i][0], B[J][rt][0], D == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : C[P0 + i][rt], 0, 0, 0);
#pragma unroll
                for (int i = 0; i < PN; ++i)
#pragma unroll
                    for (int rt = 0; rt < WR; ++rt)
                        C[P0 + i][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[i][1], B[J][rt][0], C[P0 + i][rt], 0, 0, 0);
                if constexpr (NB == 2) {
#pragma unroll
                    for (int i = 0; i < PN; ++i)
#pragma unroll
                        for (int rt = 0; rt < WR; ++rt)
                            C[P0 + i][rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[i][0], B[J][rt][NB - 1], C[P0 + i][rt], 0, 0, 0);
                }
#pragma unroll
                for (int tt = P0; D == 7 && tt < P0 + PN; ++tt) {
                    f16x4_t As;
                    if constexpr (TYPE == kQ4_K) As = min_operand(sg[tt]);
#pragma unroll
                    for (int rt = 0; rt < WR; ++rt) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) acc[tt][rt][i] = __builtin_fmaf(dsc[rt], C[tt][rt][i], acc[tt][rt][i]);
                        if constexpr (TYPE == kQ4_K) {
                            const f32x4_t pm =
                                __builtin_amdgcn_mfma_f32_16x16x16f16(As, Bm[rt], f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                            for (int i = 0; i < 4; ++i) acc[tt][rt][i] = __builtin_fmaf(dmn[rt], pm[i], acc[tt][rt][i]);
                        }
                    }
                }
                __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (D == 6) w_take(b + 1);
            if constexpr (J == 1) {
                barrier();
                const int s = s0;
                s0 = s1;
                s1 = s2;
                s2 = s;
            }
        });
    }

    // lane: pairs 4 lk + i of token tile tt, row lr of each row tile
    auto put = [&](int tt, f32x4_t (&v)[WR]) {
        int bad = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = ends[16 * tt + 4 * lk + i];
            bad |= (e == kRowNonFinite) << i;
#pragma unroll
            for (int rt = 0; rt < WR; ++rt) v[rt][i] = ldexpf(v[rt][i], e == kRowNonFinite ? 0 : -e);
        }
        if (__ballot(bad != 0)) {   // a row of x with an infinity: its outputs element by element
#pragma unroll 1
            for (int q = 0; q < 4 * WR; ++q) {
                const int i = q & 3, rt = q >> 2, row = r0 + (SWIGLU ? 0 : 16 * rt) + lr;
                if (!((bad >> i) & 1) || row >= M) continue;
                replace(v, rt, i, row_dot_per_element(a.w[SWIGLU ? rt : 0], TYPE, (static_cast<uint64_t>(tl.expert) * M + row) * K,
                                                      a.x + static_cast<size_t>(xrow(16 * tt + 4 * lk + i)) * K, K));
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int t = 16 * tt + 4 * lk + i;
            if (t >= n) continue;
            if constexpr (SWIGLU) {
                const int pos = tl.first + t;
                if (r0 + lr < M) a.y[static_cast<size_t>(pos) * M + r0 + lr] = silu(v[0][i]) * v[1][i];
            } else {
                float* y = a.y + static_cast<size_t>(ends[16 * (kMaxTokenTiles + tt) + 4 * lk + i]) * M;
#pragma unroll
                for (int rt = 0; rt < WR; ++rt)
                    if (r0 + 16 * rt + lr < M) y[r0 + 16 * rt + lr] = v[rt][i];
            }
        }
    };
#pragma unroll
    for (int tt = 0; tt < WT; ++tt) put(tt, acc[tt]);
}

// A workgroup takes a tile and a slice of the expert's rows. Consecutive items go to one XCD (workgroups are handed to the
// 8 XCDs in turn), so that the slices of a tile find its rows of x, and the tiles of an expert its weights, in one L2.
template <int TYPE, bool SWIGLU>
__global__ __launch_bounds__(kRowsWaves* kWave) __attribute__((amdgpu_waves_per_eu(2, 2))) void rows_kernel(const RowsArgs a) {
    constexpr size_t staged = size_t{kRowsWaves} * 32 * Staged<TYPE>::pieces * 16;
    __shared__ __align__(16) uint8_t smem[RowsShape<kMaxTokenTiles, SWIGLU>::ring + staged];
    __shared__ int ends[2 * 16 * kMaxTokenTiles];   // exponents, pairs
    const int items = a.tiles[-1].expert * a.column_blocks, per = (items + 7) / 8;
    const int turn = static_cast<int>(blockIdx.x >> 3), item = static_cast<int>(blockIdx.x & 7) * per + turn;
    if (turn >= per || item >= items) return;   // the whole workgroup
    const int tile = item / a.column_blocks, cb = item - tile * a.column_blocks;
    const Tile tl = a.tiles[tile];
    const int wt = (tl.n + 15) >> 4;
    bool done = false;
    static_for<kMaxTokenTiles>([&](auto i) {
        constexpr int WT = decltype(i)::value + 1;
        if (!done && (wt == WT || WT == kMaxTokenTiles)) {
            rows_tile<TYPE, WT, SWIGLU>(a, tl, cb, smem, ends);
            done = true;
        }
    });
}

// ------------------------------------------------------------------ small groups
// Tiles of up to 8 or 16 pairs, rows of up to 8 blocks (K <= 2048): bound by the weights, each expert's read about once. A
// workgroup's waves split the blocks of a row, KW waves a block each, so that they read a row tile whole, 16 rows of
// neighbouring memory, at one time, and a wave keeps its block's operands of x in registers for all row tiles of a tile of
// pairs. (Waves that went through 32 rows a block at a time, 144 bytes here and there, took 100 us for the gate and up
// products of 77 tokens, of which 67 were the weight loads by themselves and 30 the repeated loads of x.) 8 / KW row groups;
// a turn is one row tile of each - 16 gate and the same 16 up rows, or 32 down rows - whose blocks' sums meet in LDS, two
// turns' worth, one barrier a turn; the waves of a group take turns in adding them up and writing.
// The grid is one workgroup a CU, and each has an equal part of all tiles' turns: its weights are requested AHEAD turns
// ahead, over the border of a tile too, where only the operands of x are loaded anew. (A workgroup per tile and share of its
// rows: two rounds of some 45 us at 77 tokens. Two workgroups a CU of 128 registers, two turns ahead: 92 us against 65.)
// Of up to 8 pairs both fp16 parts enter one operand, rows 0-7 the high ones and 8-15 the low ones: half the products, and
// a sum of two lanes at the end (5 tokens 20.5 and 12.4 us for the two products, 22.2 and 13.6 with tiles of 16).
// A block's rows come as the 16-byte pieces that they lie in, neighbours to neighbouring lanes, and go to the lanes that use
// them through LDS, the next turn's before the barrier (each lane its own pieces from memory, us in all: 64 tokens 118 -> 114,
// Q6_K, whose blocks begin at odd places, 186 -> 171, one token of 8 picks 50 -> 36). 77 tokens: 64 us for 202 MB; 8 are the
// start, and the products and the decode of a turn, counted, are three quarters of the rest.
template <int TYPE, int TP, int KW, bool SWIGLU>
__global__ __launch_bounds__(512, 2) void strip_kernel(const RowsArgs a) {
    constexpr int BB = TYPE == kQ4_K ? 144 : 210, NB = TYPE == kQ4_K ? 1 : 2, WR = 2, RW = 8 / KW;
    constexpr int RT = SWIGLU ? 16 : 32;              // rows of a row tile
    constexpr int NP = TP == 8 ? 1 : 2;               // operands of x per depth
    constexpr int AHEAD = TYPE == kQ4_K ? 4 : 3;   // turns of weights in flight, as the registers allow
    using W = Staged<TYPE>;
    constexpr int WP = 32 * W::pieces, WI = (WP + 63) / 64;   // 16-byte pieces of a wave's 32 rows of its block
    __shared__ uint4 staged[8][WP];
    __shared__ f32x4_t part[2][8][WR][kWave];
    __shared__ int exps[2][TP];                       // of the rows of this tile and the one before
    const int M = a.M, K = a.K, nb = K >> 8;
    const int lane = threadIdx.x & 63, lr = lane & 15, lk = lane >> 4;
    const int wv = wave_in_block(), kw = wv % KW, rw = wv / KW;
    const int row_tiles = (M + RT - 1) / RT, groups = (row_tiles + RW - 1) / RW;   // turns of a tile
    const int tiles = a.tiles[-1].expert;
    const int64_t total = static_cast<int64_t>(tiles) * groups;
    const int64_t from = total * blockIdx.x / gridDim.x;
    const int count = static_cast<int>(total * (blockIdx.x + 1) / gridDim.x - from);
    if (count <= 0) return;                           // the whole workgroup
    const int kb = min(kw, nb - 1);                   // a wave past the row's blocks repeats the last one, and adds nothing
    const bool active = kw < nb;
    int tile = static_cast<int>(from / groups), group = static_cast<int>(from - static_cast<int64_t>(tile) * groups);
    // the weights' cursor
    int lt = tile, lg = group, ln = 0;
    const uint8_t* wexp[WR];
    auto w_expert = [&]() {
        const int e = a.tiles[lt].expert;
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) wexp[rt] = a.w[SWIGLU ? rt : 0] + (static_cast<uint64_t>(e) * M * nb + kb) * BB;
    };
    uint32_t wo[WI];
#pragma unroll
    for (int i = 0; i < WI; ++i) {
        const int id = min(64 * i + lane, WP - 1), row = id / W::pieces;
        wo[i] = static_cast<uint32_t>(SWIGLU ? row & 15 : row) * nb * BB + 16 * (id - row * W::pieces);
    }
    auto row_offset = [&](int g) { return static_cast<uint32_t>(min(g * RW + rw, row_tiles - 1) * RT) * nb * BB; };
    auto w_load = [&](uint4 (&d)[WI]) {               // past the end the last one again: nothing waits for it
        const uint32_t skew = TYPE == kQ4_K ? 0 : static_cast<uint32_t>(reinterpret_cast<uintptr_t>(wexp[0])) & 15u;
        const uint32_t at = row_offset(lg) + skew;
#pragma unroll
        for (int i = 0; i < WI; ++i) {
            const int id = min(64 * i + lane, WP - 1);
            d[i] = ld16((SWIGLU && id >= WP / 2 ? wexp[1] : wexp[0]) - skew + ((at + wo[i]) & ~15u));
        }
        if (++ln < count && ++lg == groups) {
            lg = 0;
            ++lt;
            w_expert();
        }
    };
    // the weights of the turn that is taken next: where its first row lies in its 16 bytes
    int tt = tile, tg = group, tn = 0;
    WBlock<TYPE> wc[WR];
    auto w_take = [&](const uint4 (&d)[WI]) {
        uint4* wl = staged[wv];
#pragma unroll
        for (int i = 0; i < WI; ++i) wl[min(64 * i + lane, WP - 1)] = d[i];
        uint32_t base = 0;
        if constexpr (TYPE != kQ4_K)
            base = static_cast<uint32_t>((static_cast<uint64_t>(a.tiles[tt].expert) * M * nb + kb) * BB) + row_offset(tg);
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) {
            const uint32_t row = static_cast<uint32_t>((SWIGLU ? 0 : 16 * rt) + lr) * nb * BB;
            W::take(wc[rt], wl + (16 * rt + lr) * W::pieces, (base + row) & 15u, lk);
        }
        if (++tn < count && ++tg == groups) {
            tg = 0;
            ++tt;
        }
    };
    uint4 w[AHEAD][WI];
    w_expert();
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
        w_load(w[i]);
        __builtin_amdgcn_sched_barrier(0);   // in this order, which the waits of the loop below count on
    }
    uint32_t k64 = 0x64006400u;
    asm volatile("" : "+v"(k64));
    Tile tl{};
    f16x8_t A[8][NP];
    f16x4_t As;
    auto row_of = [&](const Tile& q, int i) {   // row of x of a tile's pair i (the last one again past the end)
        const int pos = q.first + min(i, q.n - 1);
        return SWIGLU ? pair_at(a.order, pos, a.pairs) / a.top : pos;
    };
    int next_row = row_of(a.tiles[tile], lr % TP);
    auto x_load = [&]() {   // the operands of tile `tile`
        tl = a.tiles[tile];
        const size_t mine = static_cast<size_t>(next_row);
        const uint8_t* x0 = a.xp + mine * K * 4 + 1024 * kb + 16 * lk + (TP == 8 ? 64 * (lr >> 3) : 0);
#pragma unroll
        for (int d = 0; d < 8; ++d)
#pragma unroll
            for (int p = 0; p < NP; ++p) A[d][p] = *reinterpret_cast<const f16x8_t*>(x0 + 128 * d + 64 * p);
        if constexpr (TYPE == kQ4_K) {   // the minima's terms enter with the high part
            const float2 s = *reinterpret_cast<const float2*>(a.sx + mine * (K >> 5) + 8 * kb + 2 * lk);
            As = min_operand(TP == 16 || lr < 8 ? s : make_float2(0.f, 0.f));
        }
        if (wv == 0 && lane < TP) exps[tile & 1][lane] = a.ex[mine];
        next_row = row_of(a.tiles[min(tile + 1, tiles - 1)], lr % TP);   // known when the next tile's turn comes
    };
    const int p0 = TP == 8 ? 4 * (lk & 1) : 4 * lk;   // the lane's first pair in the sums
    auto finish = [&](int turn) {
        const int row_tile = group * RW + rw, r0 = row_tile * RT;
        f32x4_t v[WR];
        int bad = 0;
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) {
            v[rt] = part[turn & 1][rw * KW][rt][lane];
#pragma unroll
            for (int s = 1; s < KW; ++s) v[rt] += part[turn & 1][rw * KW + s][rt][lane];
            if constexpr (TP == 8) {
#pragma unroll
                for (int i = 0; i < 4; ++i) v[rt][i] += __shfl_xor(v[rt][i], 32);
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int e = exps[tile & 1][p0 + i];
            bad |= (e == kRowNonFinite) << i;
#pragma unroll
            for (int rt = 0; rt < WR; ++rt) v[rt][i] = ldexpf(v[rt][i], e == kRowNonFinite ? 0 : -e);
        }
        if (__ballot(bad != 0)) {   // a row of x with an infinity: its outputs element by element
#pragma unroll 1
            for (int q = 0; q < 4 * WR; ++q) {
                const int i = q & 3, rt = q >> 2, row = r0 + (SWIGLU ? 0 : 16 * rt) + lr;
                if (!((bad >> i) & 1) || row >= M) continue;
                replace(v, rt, i, row_dot_per_element(a.w[SWIGLU ? rt : 0], TYPE, (static_cast<uint64_t>(tl.expert) * M + row) * K,
                                                      a.x + static_cast<size_t>(row_of(tl, p0 + i)) * K, K));
            }
        }
        if ((TP == 8 && lk >= 2) || row_tile >= row_tiles) return;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (p0 + i >= tl.n) continue;
            const int pos = tl.first + p0 + i;
            if constexpr (SWIGLU) {
                if (r0 + lr < M) a.y[static_cast<size_t>(pos) * M + r0 + lr] = silu(v[0][i]) * v[1][i];
            } else {
                float* y = a.y + static_cast<size_t>(pair_at(a.order, pos, a.pairs)) * M;
#pragma unroll
                for (int rt = 0; rt < WR; ++rt)
                    if (r0 + 16 * rt + lr < M) y[r0 + 16 * rt + lr] = v[rt][i];
            }
        }
    };
    x_load();
    w_take(w[0]);
    w_load(w[0]);
    auto step = [&](uint4 (&next)[WI], int turn) {   // next: the weights of the turn after this one
        f32x4_t C[WR];
        WScale<TYPE> sc[WR];
        static_for<8>([&](auto dI) {
            constexpr int D = decltype(dI)::value, U = D >> 1, J = D & 1;
#pragma unroll
            for (int rt = 0; rt < WR; ++rt) {
                if constexpr (J == 0) sc[rt].template set<U>(wc[rt], lk);
                f16x8_t B[NB];
                decode<U, J>(wc[rt], sc[rt], k64, B);
                C[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[D][0], B[0], D == 0 ? f32x4_t{0.f, 0.f, 0.f, 0.f} : C[rt], 0, 0, 0);
                if constexpr (NP == 2) C[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[D][1], B[0], C[rt], 0, 0, 0);
                if constexpr (NB == 2) C[rt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(A[D][0], B[NB - 1], C[rt], 0, 0, 0);
            }
        });
#pragma unroll
        for (int rt = 0; rt < WR; ++rt) {
            f32x4_t s;
            if constexpr (TYPE == kQ4_K) {
                const float d = opaque(half_bits(wc[rt].hd.x & 0xffffu)), dmin = opaque(-32.0f * half_bits(wc[rt].hd.x >> 16));
                const f32x4_t pm =
                    __builtin_amdgcn_mfma_f32_16x16x16f16(As, min_weights(wc[rt].hd, lk), f32x4_t{0.f, 0.f, 0.f, 0.f}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = __builtin_fmaf(dmin, pm[i], d * C[rt][i]);
            } else {
                const float d = opaque(half_bits(wc[rt].d));
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = d * C[rt][i];
            }
            part[turn & 1][wv][rt][lane] = active ? s : f32x4_t{0.f, 0.f, 0.f, 0.f};
        }
        w_take(next);
        w_load(next);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the sums are in LDS (the loads of weights stay in flight)
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        if (turn % KW == kw) finish(turn);
        if (++group == groups) {
            group = 0;
            ++tile;
            if (turn + 1 < count) x_load();
        }
    };
    // Left from the middle, not skipped over: so that on every way back to the first step the other buffers' loads have been
    // issued after its own, and it waits for its own alone.
    for (int u = 0;;) {
        step(w[1 % AHEAD], u);
        if (++u == count) break;
        step(w[2 % AHEAD], u);
        if (++u == count) break;
        step(w[3 % AHEAD], u);
        if (++u == count) break;
        if constexpr (AHEAD == 4) {
            step(w[0], u);
            if (++u == count) break;
        }
    }
}

// out[t] = sum_j w[t][j] y[t k + j], j in order; NaN for a token one of whose pairs has no expert (y has no row of it).
__global__ __launch_bounds__(256) void rows_combine(const float* __restrict__ y, const float* __restrict__ w,
                                                    const int* __restrict__ lost, int rows, int k, int dim4,
                                                    float* __restrict__ out) {
    const int per = (dim4 + 255) / 256;   // workgroups of a row
    for (int64_t b = blockIdx.x; b < static_cast<int64_t>(rows) * per; b += gridDim.x) {
        const int t = static_cast<int>(b / per), d4 = static_cast<int>(b - static_cast<int64_t>(t) * per) * 256 + static_cast<int>(threadIdx.x);
        if (d4 >= dim4) continue;
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        const float* yt = y + (static_cast<size_t>(t) * k * dim4 + d4) * 4;
        for (int j = 0; j < k; ++j) {
            const float4 v = ld4(yt + static_cast<size_t>(j) * dim4 * 4);
            const float a = w[static_cast<size_t>(t) * k + j];
            o.x = __builtin_fmaf(a, v.x, o.x);
            o.y = __builtin_fmaf(a, v.y, o.y);
            o.z = __builtin_fmaf(a, v.z, o.z);
            o.w = __builtin_fmaf(a, v.w, o.w);
        }
        if (lost[t]) o = make_float4(__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""));
        st4(out + (static_cast<size_t>(t) * dim4 + d4) * 4, o);
    }
}

// ------------------------------------------------------------------ host
size_t align_up(size_t b) { return (b + 255) & ~size_t{255}; }

// Pairs of a tile, and with them the kernel, by the mean size of the groups (those of a routing over all experts):
// strip_kernel with tiles of 8 or 16 pairs, rows_kernel with up to 64. (All launches of a call, us, strip / rows: 128 tokens
// of 8 picks among 256 experts Q4_K 142 / 161, Q6_K 208 / 222; 256 tokens 175 / 184 and 251 / 255; 512, before the strips'
// loads by pieces, 240 / 231 and 365 / 303.)
int tile_pairs(int64_t pairs, int experts, int width, int inter) {
    const double mean = static_cast<double>(pairs) / std::min<int64_t>(pairs, experts);
    if (mean <= 8 && std::max(width, inter) <= 2048) return mean <= 1.5 ? 8 : 16;
    return 16 * kMaxTokenTiles;
}
int64_t tile_bound(int64_t pairs, int experts, int size) { return pairs / size + std::min<int64_t>(pairs, experts); }

struct Layout {
    int64_t tiles;
    size_t table, lost, ex, sx, xp, hidden, hex, hsx, hxp, y, bytes;
};
Layout layout(int rows, int top, int experts, int width, int inter) {
    const size_t pairs = static_cast<size_t>(rows) * top;
    Layout l;
    l.tiles = tile_bound(pairs, experts, tile_pairs(pairs, experts, width, inter));
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += align_up(n);
        return here;
    };
    l.table = take(sizeof(Tile) * (l.tiles + 1));
    l.lost = take(4 * static_cast<size_t>(rows));
    l.ex = take(4 * static_cast<size_t>(rows));
    l.sx = take(static_cast<size_t>(rows) * (width / 32) * 4);
    l.xp = take(static_cast<size_t>(rows) * width * 4);
    l.hidden = take(pairs * inter * 4);
    l.hex = take(4 * pairs);
    l.hsx = take(pairs * (inter / 32) * 4);
    l.hxp = take(pairs * inter * 4);
    l.y = take(pairs * width * 4);
    l.bytes = at;
    return l;
}

// The sizes that a call takes; the message names the first that it does not.
int check_sizes(int rows, int top, int n_experts, int width, int inter) {
    QK_REQUIRE(width > 0 && inter > 0 && width % 256 == 0 && inter % 256 == 0,
               "moe_experts_rows: widths %d and %d are not multiples of 256", width, inter);
    QK_REQUIRE(width <= (1 << 20) && inter <= (1 << 20), "moe_experts_rows: widths %d and %d exceed 2^20", width, inter);
    QK_REQUIRE(n_experts > 0 && n_experts <= kMaxExperts, "moe_experts_rows: %d experts (1 to %d)", n_experts, kMaxExperts);
    QK_REQUIRE(rows >= 0 && top > 0 && static_cast<int64_t>(rows) * top <= (1 << 24), "moe_experts_rows: %d rows of %d picks",
               rows, top);
    QK_REQUIRE(static_cast<int64_t>(rows) * std::max<int64_t>(width, static_cast<int64_t>(top) * inter) < (int64_t{1} << 34),
               "moe_experts_rows: %d rows exceed one call", rows);
    return QWEN_STATUS_OK;
}

template <int TYPE, bool SWIGLU>
void launch_rows(RowsArgs a, int64_t tiles, hipStream_t s) {
    a.column_blocks = static_cast<int>(blocks_for(a.M, RowsShape<1, SWIGLU>::cols));
    const unsigned grid = static_cast<unsigned>((tiles * a.column_blocks + 7) / 8 * 8);
    rows_kernel<TYPE, SWIGLU><<<grid, kRowsWaves * kWave, 0, s>>>(a);
}

template <int TYPE, int TP, int KW, bool SWIGLU>
void launch_strip(const RowsArgs& a, hipStream_t s) {
    strip_kernel<TYPE, TP, KW, SWIGLU><<<256, 512, 0, s>>>(a);   // one a CU
}

template <int TYPE, int TP, bool SWIGLU>
void launch_small(const RowsArgs& a, hipStream_t s) {
    const int nb = a.K / 256;   // at most 8
    if (nb > 4)
        launch_strip<TYPE, TP, 8, SWIGLU>(a, s);
    else if (nb > 2)
        launch_strip<TYPE, TP, 4, SWIGLU>(a, s);
    else
        launch_strip<TYPE, TP, 2, SWIGLU>(a, s);
}

template <int TYPE, bool SWIGLU>
void launch_type(const RowsArgs& a, int size, int64_t tiles, hipStream_t s) {
    if (size == 8) {
        launch_small<TYPE, 8, SWIGLU>(a, s);
    } else if (size == 16) {
        launch_small<TYPE, 16, SWIGLU>(a, s);
    } else {
        launch_rows<TYPE, SWIGLU>(a, tiles, s);
    }
}

template <bool SWIGLU>
void launch_product(int type, const RowsArgs& a, int size, int64_t tiles, hipStream_t s) {
    if (type == kQ4_K)
        launch_type<kQ4_K, SWIGLU>(a, size, tiles, s);
    else
        launch_type<kQ6_K, SWIGLU>(a, size, tiles, s);
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qwen_moe_group_rows(const int32_t* idx, int pairs, int n_experts, int32_t* order, int32_t* starts, void* stream) {
    QK_REQUIRE(pairs >= 0 && pairs <= (1 << 24), "moe_group_rows: %d pairs", pairs);
    QK_REQUIRE(n_experts > 0 && n_experts <= kMaxExperts, "moe_group_rows: %d experts (1 to %d)", n_experts, kMaxExperts);
    QK_REQUIRE(starts && (pairs == 0 || (idx && order)), "moe_group_rows: null pointer");
    // every workgroup reads all ids: one written over by another's pairs would be counted as another expert's
    const size_t ids = static_cast<size_t>(pairs) * 4, offsets = static_cast<size_t>(n_experts + 1) * 4;
    QK_REQUIRE(apart(idx, ids, order, ids) && apart(idx, ids, starts, offsets) && apart(order, ids, starts, offsets),
               "moe_group_rows: idx, order and starts overlap");
    group_kernel<<<std::max(blocks_for(pairs, kGroupBlock), 1u), kGroupBlock, 0, as_stream(stream)>>>(idx, pairs, n_experts,
                                                                                                   order, starts);
    return check_launch("moe_group_rows");
}

size_t qwen_moe_experts_rows_workspace_bytes(int rows, int top, int n_experts, int width, int inter) {
    if (rows == 0 || check_sizes(rows, top, n_experts, width, inter)) return 0;
    return layout(rows, top, n_experts, width, inter).bytes;
}

int qwen_moe_experts_rows(const void* w_gate, const void* w_up, int type, const void* w_down, int down_type, int n_experts,
                          const int32_t* order, const int32_t* starts, const float* weights, int top, const float* x, int rows,
                          int width, int inter, float* out, void* workspace, size_t workspace_bytes, void* stream) {
    QK_REQUIRE(w_gate && w_up && w_down, "moe_experts_rows: tensor is not loaded");
    if ((type != kQ4_K && type != kQ6_K) || (down_type != kQ4_K && down_type != kQ6_K))
        return fail(QWEN_STATUS_UNSUPPORTED_TYPE, "moe_experts_rows: GGML types %d, %d (Q4_K and Q6_K)", type, down_type);
    if (const int rc = check_sizes(rows, top, n_experts, width, inter)) return rc;
    if (rows == 0) return ok();
    QK_REQUIRE(order && starts && weights && x && out, "moe_experts_rows: null pointer");
    QK_REQUIRE(aligned16(w_gate) && aligned16(w_up) && aligned16(w_down) && aligned16(x) && aligned16(out),
               "moe_experts_rows: tensors must be 16-byte aligned");
    QK_REQUIRE(out != x, "moe_experts_rows: out is x");
    const Layout l = layout(rows, top, n_experts, width, inter);
    QK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= l.bytes,
               "moe_experts_rows: workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, l.bytes);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    const hipStream_t s = as_stream(stream);
    const int pairs = rows * top, size = tile_pairs(pairs, n_experts, width, inter);
    Tile* tiles = reinterpret_cast<Tile*>(ws + l.table) + 1;
    int* lost = reinterpret_cast<int*>(ws + l.lost);
    const Grouping gr{order, starts, tiles, lost, n_experts, pairs, top, size, static_cast<int>(l.tiles)};
    int *ex = reinterpret_cast<int*>(ws + l.ex), *hex = reinterpret_cast<int*>(ws + l.hex);
    float *sx = reinterpret_cast<float*>(ws + l.sx), *hsx = reinterpret_cast<float*>(ws + l.hsx);
    float *hidden = reinterpret_cast<float*>(ws + l.hidden), *y = reinterpret_cast<float*>(ws + l.y);
    rows_prep<true><<<blocks_for(rows, 4) + 1, 256, 0, s>>>(x, rows, width, ex, sx, ws + l.xp, gr);
    RowsArgs a{};
    a.w[0] = static_cast<const uint8_t*>(w_gate);
    a.w[1] = static_cast<const uint8_t*>(w_up);
    a.tiles = tiles;
    a.order = order;
    a.ex = ex;
    a.sx = sx;
    a.xp = ws + l.xp;
    a.x = x;
    a.y = hidden;
    a.M = inter;
    a.K = width;
    a.top = top;
    a.pairs = pairs;
    launch_product<true>(type, a, size, l.tiles, s);
    rows_prep<false><<<blocks_for(pairs, 4) + 1, 256, 0, s>>>(hidden, pairs, inter, hex, hsx, ws + l.hxp, gr);
    a.w[0] = static_cast<const uint8_t*>(w_down);
    a.w[1] = nullptr;
    a.ex = hex;
    a.sx = hsx;
    a.xp = ws + l.hxp;
    a.x = hidden;
    a.y = y;
    a.M = width;
    a.K = inter;
    launch_product<false>(down_type, a, size, l.tiles, s);
    const int64_t strips = static_cast<int64_t>(rows) * blocks_for(width / 4, 256);
    rows_combine<<<static_cast<unsigned>(std::min<int64_t>(strips, 1 << 16)), 256, 0, s>>>(
        y, weights, lost, rows, top, width / 4, out);
    return check_launch("moe_experts_rows");
}

}  // extern "C"
