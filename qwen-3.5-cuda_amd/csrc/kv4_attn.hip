// Attention over the paged 4-bit cache (kv4_common.hpp) on gfx950: the rows of several requests in one call, single tokens
// and prompts mixed. Row i of a request with n rows and kv_len keys stands at position kv_len - n + i and sees keys
// 0 .. position:
//   score_t = (sum_g scale_tg (q . code_t)_g + min_tg sum(q)_g) / sqrt(D) over the groups g of 64 dims,
//   out = (sum_t p_t scale_t code_t + sum_t p_t min_t) / sum_t p_t, p = exp(score - max)  (x sigmoid(gate)),
// zeros where no key is seen. The reference has the one-token form over an fp32 cache (src/cuda/attn_kernels.cu:72-195,
// src/layer_attn.cpp:103-108).
#include <algorithm>
#include <cfloat>
#include <cmath>

#include "capi_common.hpp"
#include "device_common.hpp"
#include "kv4_common.hpp"

namespace qk {
namespace {

struct Attn4Args {
    const float* q;
    const float* gate;   // or null
    float* out;
    Kv4Cache c;
    const int32_t* table;
    const int32_t* row_start;
    const int32_t* kv_len;
    int max_pages, page_shift, requests, rows, heads, group;
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

// One wave per row and head, 64 tokens at a time: a lane scores one token, then sums D / 64 dims.
template <int D>
__global__ __launch_bounds__(kWave) void attn4_kernel(const Attn4Args a) {
    constexpr int NG = D / 64, ND = D / 64;
    __shared__ float qs[D], ps[kWave], qsum[NG];
    const int lane = threadIdx.x, row = static_cast<int>(blockIdx.x) / a.heads, head = static_cast<int>(blockIdx.x) % a.heads;
    const int h = head / a.group;
    int b = -1;
    for (int b0 = 0; b0 < a.requests; b0 += kWave) {
        const int at = b0 + lane;
        bool mine = false;
        if (at < a.requests) {
            const Request4 r = request(a, at);
            mine = row >= r.first && row < r.first + r.n;
        }
        const uint64_t hit = __ballot(mine);
        if (hit) b = b0 + __builtin_ctzll(hit);
    }
    if (b < 0) return;   // the whole workgroup
    const Request4 r = request(a, b);
    const int seen = max(r.len - r.n + row - r.first + 1, 0);
    const size_t o = (static_cast<size_t>(row) * a.heads + head) * D;
    for (int d = lane; d < D; d += kWave) qs[d] = a.q[o + d];
    __syncthreads();
    if (lane < NG) {
        float s = 0.f;
        for (int i = 0; i < 64; ++i) s += qs[64 * lane + i];
        qsum[lane] = s;
    }
    __syncthreads();
    float m = -FLT_MAX, l = 0.f, low = 0.f, acc[ND];
    for (int i = 0; i < ND; ++i) acc[i] = 0.f;
    for (int t0 = 0; t0 < seen; t0 += kWave) {
        const int t = t0 + lane, off = t & (a.c.page - 1);
        int id = 0;
        bool bad = false;
        if (t < seen) {
            id = a.table[static_cast<size_t>(b) * a.max_pages + (t >> a.page_shift)];
            bad = id < 0 || id >= a.c.pages;
            if (bad) id = 0;
        }
        const size_t at = (static_cast<size_t>(id) * a.c.heads + h) << a.page_shift, tok = at + off;
        float s = 0.f;
        const uint32_t* kw = reinterpret_cast<const uint32_t*>(a.c.k) + tok * (D / 8);
        for (int g = 0; g < NG; ++g) {
            float dot = 0.f;
            for (int x = 0; x < 8; ++x) {
                const uint32_t w = kw[(x >> 1) * 2 * NG + 2 * g + (x & 1)];
                for (int j = 0; j < 8; ++j) dot = __builtin_fmaf(qs[64 * g + 8 * x + j], static_cast<float>((w >> kv4_shift(j)) & 15u), dot);
            }
            const float ks = bf16_value(a.c.ks[(at + (off & ~7)) * NG + g * 8 + (off & 7)]), km = bf16_value(a.c.km[tok * NG + g]);
            s += ks * dot + km * qsum[g];
        }
        s *= a.scale;
        if (bad) s = __builtin_nanf("");
        if (t >= seen) s = -INFINITY;
        float top = s;
        bool nan = s != s;
        for (int x = 32; x >= 1; x >>= 1) top = fmaxf(top, __shfl_xor(top, x));
        const float now = __ballot(nan) ? __builtin_nanf("") : fmaxf(m, top);
        const float shrink = __builtin_amdgcn_exp2f(m - now);
        m = now;
        l *= shrink;
        low *= shrink;
        for (int i = 0; i < ND; ++i) acc[i] *= shrink;
        const float p = t < seen ? __builtin_amdgcn_exp2f(s - m) : 0.f;
        l += group_sum<kWave>(p);
        low += group_sum<kWave>(t < seen ? p * bf16_value(a.c.vm[tok]) : 0.f);
        ps[lane] = t < seen ? p * bf16_value(a.c.vs[tok]) : 0.f;
        __syncthreads();
        for (int j = 0; j < kWave && t0 + j < seen; ++j) {
            const size_t page_at = __shfl(static_cast<long long>(at), j);
            const int oj = (t0 + j) & (a.c.page - 1);
            const uint32_t* vw = reinterpret_cast<const uint32_t*>(a.c.v) + ((page_at + (oj & ~7)) >> 3) * D;
            for (int i = 0; i < ND; ++i)
                acc[i] = __builtin_fmaf(ps[j], static_cast<float>((vw[64 * i + lane] >> kv4_shift(oj & 7)) & 15u), acc[i]);
        }
        __syncthreads();
    }
    if (r.bad) l = __builtin_nanf("");
    for (int i = 0; i < ND; ++i) {
        const size_t x = o + 64 * i + lane;
        float v = l == 0.f ? 0.f : (acc[i] + low) / l;
        if (a.gate) v *= sigmoid(a.gate[x]);
        a.out[x] = v;
    }
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" {

size_t qwen_attn_kv4_workspace_bytes(int rows, int requests, int heads, int kv_heads, int dim) {
    if (rows <= 0 || requests <= 0 || kv_heads <= 0 || heads <= 0 || heads % kv_heads || dim <= 0) return 0;
    return 16;
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
    const size_t need = qwen_attn_kv4_workspace_bytes(rows, requests, heads, kv_heads, dim);
    QK_REQUIRE(workspace && aligned16(workspace) && workspace_bytes >= need,
               "attn_kv4_rows: workspace of %zu bytes, need %zu (16-byte aligned)", workspace_bytes, need);
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
    const hipStream_t s = as_stream(stream);
    const unsigned grid = static_cast<unsigned>(rows) * static_cast<unsigned>(heads);
    if (dim == 64)
        attn4_kernel<64><<<grid, kWave, 0, s>>>(a);
    else if (dim == 128)
        attn4_kernel<128><<<grid, kWave, 0, s>>>(a);
    else
        attn4_kernel<256><<<grid, kWave, 0, s>>>(a);
    return check_launch("attn_kv4_rows");
}

}  // extern "C"
