// The paged 8-bit key / value cache on gfx950: page bookkeeping of a step of several requests, storing fresh keys and
// values, reading slots back. Layout and quantization: kv8_common.hpp. The attention that reads it: kv8_attn.hip.
//
// The reference keeps one sequence's keys and values in fp32 rows of a fixed array (src/layer_attn.cpp:44-46, copied to
// row pos at :99-100); these entry points have no counterpart there.
#include <algorithm>

#include "capi_common.hpp"
#include "kv8_common.hpp"

namespace qk {
namespace {

// ------------------------------------------------------------------ page bookkeeping
// Two prefix sums over the requests (fresh rows, pages needed) and what follows from them. Every workgroup runs the
// scans of all requests itself (4096 at most, 4 per thread: shuffles, one LDS exchange), so one launch with no
// dependence between workgroups does everything: workgroup w then writes the slots and positions of rows
// [1024 w, 1024 w + 1024), each found by a binary search in the row starts in LDS; workgroup 0 writes the rest. A slot in
// a fresh page is taken from the free list, not from the table entry that workgroup 0 writes.
// Bound by latency: two dependent loads, the scans and 12 steps of the search.
constexpr int kPlanBlock = 1024;

__device__ __forceinline__ int clamp0(int v) { return v > 0 ? v : 0; }

__global__ __launch_bounds__(kPlanBlock) void kv8_plan_kernel(
    const int32_t* __restrict__ cached, const int32_t* __restrict__ fresh, int requests, int32_t* table, int max_pages,
    const int32_t* __restrict__ free_pages, int n_free, const int32_t* free_head, int32_t* free_head_out, int page, int rows,
    int32_t* __restrict__ row_start, int32_t* __restrict__ kv_len, int32_t* __restrict__ slots, int32_t* __restrict__ pos) {
    __shared__ int start[kKv8MaxRequests + 1], first_free[kKv8MaxRequests], base[kKv8MaxRequests];
    __shared__ long long part[2][kPlanBlock / kWave];
    __shared__ int head_used;
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int per = (requests + kPlanBlock - 1) / kPlanBlock;   // 1..4 neighbouring requests of this thread
    const int b0 = tid * per;
    const long long limit = static_cast<long long>(max_pages) * page;
    const int head0 = free_head[0], head = min(clamp0(head0), n_free);
    if (tid == 0) head_used = head0;

    int c[4], n[4];
    long long sum_n = 0, sum_need = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool in = i < per && b0 + i < requests;
        c[i] = in ? clamp0(cached[b0 + i]) : 0;
        n[i] = in ? clamp0(fresh[b0 + i]) : 0;
        sum_n += n[i];
    }
    // exclusive prefix of `v` over the workgroup's threads; slot: which LDS line carries it
    auto prefix = [&](long long v, int slot) {
        long long inc = v;
#pragma unroll
        for (int o = 1; o < kWave; o <<= 1) {
            const long long up = __shfl_up(inc, o);
            if (lane >= o) inc += up;
        }
        if (lane == 63) part[slot][wv] = inc;
        __syncthreads();
        long long before = 0;
        for (int w = 0; w < wv; ++w) before += part[slot][w];
        return before + inc - v;
    };
    long long row = prefix(sum_n, 0);
    int need[4], have[4];
    bool room[4];
    {
        long long r = row;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long total = static_cast<long long>(c[i]) + n[i];
            room[i] = total <= limit && r + n[i] <= rows;
            have[i] = static_cast<int>((static_cast<long long>(c[i]) + page - 1) / page);
            need[i] = n[i] > 0 && room[i] ? static_cast<int>((total + page - 1) / page) - have[i] : 0;
            sum_need += need[i];
            r += n[i];
        }
    }
    long long want = prefix(sum_need, 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int b = b0 + i;
        if (i >= per || b >= requests) break;
        const bool granted = room[i] && (need[i] == 0 || want + need[i] <= n_free - head);
        const int begin = static_cast<int>(row < 0x7fffffffLL ? row : 0x7fffffffLL);
        start[b] = begin;
        base[b] = granted ? c[i] : -1 - c[i];            // cached tokens; marked where nothing is granted
        first_free[b] = granted ? static_cast<int>(head + want) - have[i] : 0;   // + page index: place in the free list
        row += n[i];
        if (b == requests - 1) start[requests] = static_cast<int>(row < 0x7fffffffLL ? row : 0x7fffffffLL);
        if (blockIdx.x == 0) {
            row_start[b] = begin;
            if (b == requests - 1) row_start[requests] = start[requests];
            kv_len[b] = granted ? c[i] + n[i] : 0;
            if (granted && need[i] > 0) {
                for (int j = 0; j < need[i]; ++j)
                    table[static_cast<size_t>(b) * max_pages + have[i] + j] = free_pages[head + want + j];
                atomicMax(&head_used, static_cast<int>(head + want + need[i]));   // a maximum: the order does not matter
            }
        }
        want += need[i];
    }
    if (requests == 0 && tid == 0) {
        start[0] = 0;
        if (blockIdx.x == 0) row_start[0] = 0;
    }
    __syncthreads();
    if (blockIdx.x == 0 && tid == 0) free_head_out[0] = head_used;
    const int filled = start[requests];
    for (int r = blockIdx.x * kPlanBlock + tid; r < rows; r += gridDim.x * kPlanBlock) {
        int slot = -1, p = 0;
        if (r < filled) {
            int lo = 0, hi = requests;   // the last request with start <= r: start[lo] <= r < start[hi]
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (start[mid] <= r)
                    lo = mid;
                else
                    hi = mid;
            }
            const bool granted = base[lo] >= 0;
            const int was = granted ? base[lo] : -1 - base[lo];
            p = static_cast<int>(static_cast<uint32_t>(was) + static_cast<uint32_t>(r - start[lo]));
            if (granted) {
                const int j = p / page, have_pages = (was + page - 1) / page;
                const int id = j < have_pages ? table[static_cast<size_t>(lo) * max_pages + j] : free_pages[first_free[lo] + j];
                const long long s = static_cast<long long>(id) * page + (p - j * page);
                slot = s >= 0 && s <= 0x7fffffffLL ? static_cast<int>(s) : -1;
            }
        }
        slots[r] = slot;
        pos[r] = p;
    }
}

// ------------------------------------------------------------------ store
// A workgroup takes the runs that start in its share of the rows (a run: neighbouring rows with neighbouring slots of
// one page), for one head and for keys or values: it alone writes that page's codes and scale, so no order of workgroups
// shows in the result. A thread's item is an octet of tokens x 4 dims: 16-byte loads, kept in registers between the
// largest magnitude and the codes (what does not fit, past 64 tokens of 256, is read again), 4-byte stores of keys, 32
// bytes in a row of values. Bound by latency: one round of loads, one reduction, the stores.
constexpr int kStoreBlock = 512;

template <bool ALIGNED>
__device__ __forceinline__ float4 row4(const float* p) {
    if constexpr (ALIGNED) return ld4(p);
    return make_float4(p[0], p[1], p[2], p[3]);
}

__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return (static_cast<uint32_t>(static_cast<int>(a)) & 0xffu) | ((static_cast<uint32_t>(static_cast<int>(b)) & 0xffu) << 8) |
           ((static_cast<uint32_t>(static_cast<int>(c)) & 0xffu) << 16) | (static_cast<uint32_t>(static_cast<int>(d)) << 24);
}
__device__ __forceinline__ float code_of(uint32_t w, int i) { return static_cast<float>(static_cast<int8_t>((w >> (8 * i)) & 0xffu)); }

__device__ __forceinline__ uint32_t rescale4(uint32_t w, float ratio) {
    return pack4(kv8_rescale(code_of(w, 0), ratio), kv8_rescale(code_of(w, 1), ratio), kv8_rescale(code_of(w, 2), ratio),
                 kv8_rescale(code_of(w, 3), ratio));
}

template <int BLOCK, bool ALIGNED, bool VALUES>
__device__ void store_run(const float* __restrict__ x, int64_t stride, int n, int8_t* __restrict__ codes, float* scale,
                          int off, int dim, uint32_t* red) {
    const int tid = threadIdx.x, d_shift = __builtin_ctz(dim) - 2, d4s = 1 << d_shift;   // dim 64, 128 or 256
    const int end = off + n, o0 = off >> 3, items = (((end + 7) >> 3) - o0) << d_shift;
    const int first_o = o0 + (tid >> d_shift), d4 = tid & (d4s - 1), o_step = BLOCK >> d_shift;
    float4 f[8];
    auto load = [&](int o) {   // tokens of octet o that are not in the run come out 0
#pragma unroll
        for (int t = 0; t < 8; ++t) {
            const int at = 8 * o + t - off;
            f[t] = at >= 0 && at < n ? row4<ALIGNED>(x + at * stride + 4 * d4) : make_float4(0.f, 0.f, 0.f, 0.f);
        }
    };
    // the run's largest magnitude, as bits: infinities and NaNs come out above every finite value
    uint32_t m = 0;
    auto take = [&]() {
#pragma unroll
        for (int t = 0; t < 8; ++t)
            m = max(max(m, max(__float_as_uint(f[t].x) & 0x7fffffffu, __float_as_uint(f[t].y) & 0x7fffffffu)),
                    max(__float_as_uint(f[t].z) & 0x7fffffffu, __float_as_uint(f[t].w) & 0x7fffffffu));
    };
    const bool single = items <= BLOCK;
    if (single) {
        load(first_o);   // past the run's end: zeros
        take();
    } else {
        for (int i = tid, o = first_o; i < items; i += BLOCK, o += o_step) {
            load(o);
            take();
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), o)));
    const float was = off ? *scale : 0.0f;   // read before the barrier that the one write comes after
    if ((tid & 63) == 0) red[tid >> 6] = m;
    __syncthreads();
    m = red[0];
#pragma unroll
    for (int w = 1; w < BLOCK / kWave; ++w) m = max(m, red[w]);
    const bool bad = m >= 0x7f800000u || was != was;
    const float s = bad ? __builtin_nanf("") : fmaxf(fmaxf(was, __uint_as_float(m) / 127.0f), kKv8Floor);
    const float rs = 1.0f / s;
    const bool again = off > 0 && !bad && s > was;   // kept codes change
    const float ratio = was / s;
    auto code = [&](float v) { return static_cast<uint32_t>(static_cast<int>(kv8_code(v, s, rs))) & 0xffu; };
    for (int i = tid, o = first_o; i < items; i += BLOCK, o += o_step) {
        if (!single) load(o);
        if constexpr (VALUES) {
            uint4* p = reinterpret_cast<uint4*>(codes + (static_cast<size_t>(o) * dim + 4 * d4) * 8);
            uint32_t w[8] = {};   // [dim][tokens 0-3, 4-7]
            if (8 * o < off) {
                const uint4 a = p[0], b = p[1];
                const uint32_t old[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
                for (int k = 0; k < 8; ++k) w[k] = again ? rescale4(old[k], ratio) : old[k];
            }
#pragma unroll
            for (int t = 0; t < 8; ++t) {
                if (8 * o + t < off || 8 * o + t >= end) continue;
                const float v[4] = {f[t].x, f[t].y, f[t].z, f[t].w};
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const int sh = 8 * (t & 3);
                    w[2 * k + (t >> 2)] = (w[2 * k + (t >> 2)] & ~(0xffu << sh)) | ((bad ? 0u : code(v[k])) << sh);
                }
            }
            p[0] = make_uint4(w[0], w[1], w[2], w[3]);
            p[1] = make_uint4(w[4], w[5], w[6], w[7]);
        } else {
            uint32_t* p = reinterpret_cast<uint32_t*>(codes) + (static_cast<size_t>(8 * o) << d_shift) + d4;
#pragma unroll
            for (int t = 0; t < 8; ++t)
                if (8 * o + t >= off && 8 * o + t < end)
                    p[t << d_shift] = bad ? 0u : code(f[t].x) | (code(f[t].y) << 8) | (code(f[t].z) << 16) | (code(f[t].w) << 24);
        }
    }
    if (again) {   // the page's tokens before the run (values: its octets; a shared octet has been written above)
        uint32_t* p = reinterpret_cast<uint32_t*>(codes);
        const int words = VALUES ? (o0 << d_shift) * 8 : off << d_shift;
        for (int i = tid; i < words; i += BLOCK) p[i] = rescale4(p[i], ratio);
    }
    if (tid == 0) *scale = s;
    __syncthreads();   // red is used again by the next run
}

// Grid: x = shares of `share` rows (at most 64), y = head, z = keys, values.
template <int BLOCK, bool ALIGNED>
__global__ __launch_bounds__(BLOCK) void kv8_store_kernel(const float* __restrict__ k, const float* __restrict__ v,
                                                                int64_t k_stride, int64_t v_stride,
                                                                const int32_t* __restrict__ slots, int rows, int share,
                                                                const Kv8Cache c) {
    __shared__ uint32_t red[BLOCK / kWave];
    const int lane = threadIdx.x & 63, h = blockIdx.y, P = c.page;
    const int total = c.pages * P;
    const int r0 = blockIdx.x * share;
    const int r = r0 + lane;
    bool starts = false;
    if (lane < share && r < rows) {
        const int s = slots[r], before = r > 0 ? slots[r - 1] : -1;
        starts = s >= 0 && s < total && (s % P == 0 || before != s - 1);
    }
    uint64_t todo = __ballot(starts);   // the same in every wave
    while (todo) {
        const int first = r0 + __builtin_ctzll(todo);
        todo &= todo - 1;
        const int s0 = slots[first], off = s0 % P, pg = s0 / P;
        int n = 0;
        for (;;) {   // 64 rows at a time; ends at the page's end at the latest
            const int i = n + lane;
            const bool in = off + i < P && first + i < rows && slots[first + i] == s0 + i;
            const uint64_t miss = ~__ballot(in);
            if (miss) {
                n += __builtin_ctzll(miss);
                break;
            }
            n += 64;
        }
        const size_t at = static_cast<size_t>(pg) * c.heads + h, block = static_cast<size_t>(P) * c.dim;
        if (blockIdx.z == 0)
            store_run<BLOCK, ALIGNED, false>(k + first * k_stride + h * c.dim, k_stride, n, c.k + at * block, c.ks + at, off, c.dim, red);
        else
            store_run<BLOCK, ALIGNED, true>(v + first * v_stride + h * c.dim, v_stride, n, c.v + at * block, c.vs + at, off, c.dim, red);
    }
}

// ------------------------------------------------------------------ read
// Slots back as fp32 rows: a thread takes 4 dims of a row's head; a negative slot gives zeros, one past the cache NaN.
// Write-bound (8 bytes out per byte of key or value); the value codes' 8-byte groups are read once per token of the
// group, from L1 where the tokens are neighbours.
__global__ __launch_bounds__(256) void kv8_read_kernel(const Kv8Cache c, const int32_t* __restrict__ slots, int rows,
                                                       float* __restrict__ k, float* __restrict__ v) {
    const int d_shift = __builtin_ctz(c.dim) - 2, p_shift = __builtin_ctz(c.page);
    const uint32_t per_row = static_cast<uint32_t>(c.heads) << d_shift, n = static_cast<uint32_t>(rows) * per_row;   // below 2^31
    for (uint32_t i = blockIdx.x * 256 + threadIdx.x; i < n; i += gridDim.x * 256) {
        const uint32_t r = i / per_row, rest = i - r * per_row;
        const int h = static_cast<int>(rest >> d_shift), d4 = static_cast<int>(rest) & ((1 << d_shift) - 1);
        const int s = slots[r];
        float4 a = make_float4(0.f, 0.f, 0.f, 0.f), b = a;
        if (s >= c.pages * c.page) {
            const float nan = __builtin_nanf("");
            a = b = make_float4(nan, nan, nan, nan);
        } else if (s >= 0) {
            const int pg = s >> p_shift, t = s & (c.page - 1);
            const size_t at = static_cast<size_t>(pg) * c.heads + h;
            const int8_t* kc = c.k + (at * c.page + t) * c.dim + 4 * d4;
            const int8_t* vc = c.v + at * c.page * c.dim + (static_cast<size_t>(t >> 3) * c.dim + 4 * d4) * 8 + (t & 7);
            const uint32_t w = *reinterpret_cast<const uint32_t*>(kc);
            const float ks = c.ks[at], vs = c.vs[at];
            a = make_float4(code_of(w, 0) * ks, code_of(w, 1) * ks, code_of(w, 2) * ks, code_of(w, 3) * ks);
            b = make_float4(static_cast<float>(vc[0]) * vs, static_cast<float>(vc[8]) * vs, static_cast<float>(vc[16]) * vs,
                            static_cast<float>(vc[24]) * vs);
        }
        st4(k + 4 * static_cast<size_t>(i), a);
        st4(v + 4 * static_cast<size_t>(i), b);
    }
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

int qwen_kv8_plan(const int32_t* cached, const int32_t* fresh, int requests, int32_t* block_table, int max_pages,
                  const int32_t* free_pages, int n_free, const int32_t* free_head, int32_t* free_head_out, int page_size,
                  int rows, int32_t* row_start, int32_t* kv_len, int32_t* slots, int32_t* pos, void* stream) {
    QK_REQUIRE(requests >= 0 && requests <= kKv8MaxRequests, "kv8_plan: %d requests (at most %d)", requests, kKv8MaxRequests);
    QK_REQUIRE(max_pages >= 0 && n_free >= 0 && rows >= 0, "kv8_plan: negative size");
    QK_REQUIRE(kv8_page_ok(page_size), "kv8_plan: page size %d is not a power of two from 8 to %d", page_size, kKv8MaxPage);
    QK_REQUIRE(static_cast<int64_t>(max_pages) * page_size <= 0x7fffffff, "kv8_plan: table rows of %d pages", max_pages);
    QK_REQUIRE(free_head && free_head_out && row_start, "kv8_plan: null pointer");
    QK_REQUIRE(requests == 0 || (cached && fresh && kv_len && (block_table || max_pages == 0)), "kv8_plan: null pointer");
    QK_REQUIRE(n_free == 0 || free_pages, "kv8_plan: null free list");
    QK_REQUIRE(rows == 0 || (slots && pos), "kv8_plan: null slots or pos");
    // every workgroup reads the inputs, at any time beside the outputs' writes
    const size_t b = static_cast<size_t>(requests) * 4, r = static_cast<size_t>(rows) * 4;
    const struct {
        const void* p;
        size_t n;
    } in[] = {{cached, b}, {fresh, b}, {free_pages, static_cast<size_t>(n_free) * 4}, {free_head, 4}},
      out[] = {{block_table, b * static_cast<size_t>(max_pages)}, {row_start, b + 4}, {kv_len, b}, {slots, r}, {pos, r}, {free_head_out, 4}};
    for (const auto& o : out)
        for (const auto& i : in)
            QK_REQUIRE(apart(o.p, o.n, i.p, i.n) || (o.p == free_head_out && free_head_out == free_head && i.p == free_head),
                       "kv8_plan: an output overlaps an input");
    // one workgroup where the head is updated in place: no other may read it after the write
    const unsigned grid = free_head_out == free_head ? 1u : std::min(std::max(blocks_for(rows, kPlanBlock), 1u), 256u);
    kv8_plan_kernel<<<grid, kPlanBlock, 0, as_stream(stream)>>>(cached, fresh, requests, block_table, max_pages, free_pages,
                                                                n_free, free_head, free_head_out, page_size, rows, row_start,
                                                                kv_len, slots, pos);
    return check_launch("kv8_plan");
}

int qwen_kv8_store_rows(const float* k, const float* v, int64_t k_stride, int64_t v_stride, const int32_t* slots, int rows,
                        int8_t* k_codes, int8_t* v_codes, float* k_scale, float* v_scale, int pages, int page_size,
                        int kv_heads, int dim, void* stream) {
    const Kv8Cache c{k_codes, v_codes, k_scale, v_scale, pages, page_size, kv_heads, dim};
    if (const int rc = kv8_check("kv8_store_rows", c)) return rc;
    QK_REQUIRE(rows >= 0, "kv8_store_rows: negative rows %d", rows);
    if (rows == 0) return ok();
    QK_REQUIRE(k && v && slots, "kv8_store_rows: null pointer");
    const int64_t width = static_cast<int64_t>(kv_heads) * dim;
    QK_REQUIRE(rows == 1 || (k_stride >= width && v_stride >= width), "kv8_store_rows: row strides below kv_heads x dim");
    // Steps of single tokens: every row starts a run, a workgroup each. Longer ones: 16 rows to a workgroup, of which a
    // page's first row lies in one.
    const int share = rows <= 512 ? 1 : 16;
    const dim3 grid(blocks_for(rows, share), static_cast<unsigned>(kv_heads), 2);
    const hipStream_t s = as_stream(stream);
    const bool vec = aligned16(k) && aligned16(v) && k_stride % 4 == 0 && v_stride % 4 == 0;
    const auto launch = vec ? kv8_store_kernel<kStoreBlock, true> : kv8_store_kernel<kStoreBlock, false>;
    launch<<<grid, kStoreBlock, 0, s>>>(k, v, k_stride, v_stride, slots, rows, share, c);
    return check_launch("kv8_store_rows");
}

int qwen_kv8_read_rows(const int8_t* k_codes, const int8_t* v_codes, const float* k_scale, const float* v_scale, int pages,
                       int page_size, int kv_heads, int dim, const int32_t* slots, int rows, float* k, float* v, void* stream) {
    const Kv8Cache c{const_cast<int8_t*>(k_codes), const_cast<int8_t*>(v_codes), const_cast<float*>(k_scale),
                     const_cast<float*>(v_scale), pages, page_size, kv_heads, dim};
    if (const int rc = kv8_check("kv8_read_rows", c)) return rc;
    QK_REQUIRE(rows >= 0, "kv8_read_rows: negative rows %d", rows);
    if (rows == 0) return ok();
    QK_REQUIRE(slots && k && v, "kv8_read_rows: null pointer");
    QK_REQUIRE(aligned16(k) && aligned16(v), "kv8_read_rows: outputs must be 16-byte aligned");
    const int64_t items = static_cast<int64_t>(rows) * kv_heads * (dim / 4);
    QK_REQUIRE(items <= 0x7fffffff, "kv8_read_rows: %d rows exceed one call", rows);
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>((items + 255) / 256, 8192));
    kv8_read_kernel<<<grid, 256, 0, as_stream(stream)>>>(c, slots, rows, k, v);
    return check_launch("kv8_read_rows");
}

}  // extern "C"
