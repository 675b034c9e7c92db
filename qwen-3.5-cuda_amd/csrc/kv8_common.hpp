// The paged 8-bit key / value cache: layout, and how codes are made from values.
//
// A page holds `page` tokens (a power of two from 8 up) of every KV head. Per page and head: P x D key codes [token][dim],
// P x D value codes [token / 8][dim][8] (the order in which a matrix-core operand of values is read: 8 tokens of one
// dim), and one fp32 scale each for keys and values. A slot is page * P + token in page.
//   value = code * scale,  code in -127..127
//   scale = max(RN(largest |value| / 127), 2^-100) when a page's first tokens are stored; it only grows while later
//   tokens join, and the codes that are there are then re-rounded: rne(code * RN(old / new)).
// Codes are rne(x / scale) of the exact quotient, so they do not depend on how the quotient is evaluated.
#pragma once

#include "capi_common.hpp"
#include "device_common.hpp"

namespace qk {
namespace {

constexpr float kKv8Floor = 0x1p-100f;   // smallest scale: every quotient and reciprocal below stays a normal number
constexpr int kKv8MaxPage = 1024;
constexpr int kKv8MaxRequests = 4096;

struct Kv8Cache {
    int8_t* k;
    int8_t* v;
    float* ks;
    float* vs;
    int pages, page, heads, dim;
};

inline bool kv8_page_ok(int page) { return page >= 8 && page <= kKv8MaxPage && (page & (page - 1)) == 0; }

inline int kv8_check(const char* what, const Kv8Cache& c) {
    QK_REQUIRE(c.k && c.v && c.ks && c.vs, "%s: null cache pointer", what);
    QK_REQUIRE(aligned16(c.k) && aligned16(c.v), "%s: cache codes must be 16-byte aligned", what);
    QK_REQUIRE(c.heads > 0 && c.heads <= 65535, "%s: %d KV heads", what, c.heads);
    QK_REQUIRE(c.dim == 64 || c.dim == 128 || c.dim == 256, "%s: head dim %d is not 64, 128 or 256", what, c.dim);
    QK_REQUIRE(kv8_page_ok(c.page), "%s: page size %d is not a power of two from 8 to %d", what, c.page, kKv8MaxPage);
    QK_REQUIRE(c.pages > 0 && static_cast<int64_t>(c.pages) * c.page <= 0x7fffffff, "%s: %d pages of %d tokens", what,
               c.pages, c.page);
    return QWEN_STATUS_OK;
}

// rne(x / s) of the exact quotient for |x / s| < 2^7 and s >= 2^-100. q is within one of it; r = x - q s has at most 25
// bits where |r| is near s / 2 (both terms are multiples of the smaller ulp, and cancel), so the comparisons are exact.
__device__ __forceinline__ float kv8_code(float x, float s, float rs) {
    float q = rintf(x * rs);
    const float r = __builtin_fmaf(-q, s, x), h = 0.5f * s;
    const bool odd = static_cast<int>(q) & 1;
    if (r > h || (r == h && odd)) q += 1.0f;
    if (r < -h || (r == -h && odd)) q -= 1.0f;
    return fminf(fmaxf(q, -127.0f), 127.0f);
}

// rne(q ratio) of the exact product, q an integer of up to 7 bits: the fp32 product can only go wrong by landing on a
// tie, and its rounding error says on which side of the tie the exact one is.
__device__ __forceinline__ float kv8_rescale(float q, float ratio) {
    const float t = q * ratio, e = __builtin_fmaf(q, ratio, -t);
    float r = rintf(t);
    if (t - r == 0.5f && e > 0.0f) r += 1.0f;
    if (t - r == -0.5f && e < 0.0f) r -= 1.0f;
    return r;
}

}  // namespace
}  // namespace qk
