// The paged 4-bit key / value cache: layout, and how codes are made from values.
//
// A page holds `page` tokens (a power of two from 8 up) of every KV head. A value is min + scale * code, code 0..15, with
// bf16 scale and min of each group of values: of keys 64 dims of a token and head, of values all dims of a token and head.
// Keys are the ones whose errors are exponentiated, and 64 of their dims share a depth of the first product; a value's
// scale rides on its token's softmax weight, where one for the whole head costs one conversion of the weight.
//   min = the group's smallest value, rounded down; scale = the smallest bf16 that is at least (largest - min) / 15 and
//   2^-100; code = rne((x - min) / scale) of the 64-bit quotient, 0 to 15.
// Every token is quantized by itself: no store changes what another one has left.
//
// Per page and head, D = dim, NG = D / 64. 8 codes are a word; its elements 0, 2, 4, 6 lie in nibbles 0..3 and 1, 3, 5, 7 in
// nibbles 4..7, so that a mask of 0x000f000f (the word as it is, and shifted by 4, 8, 12) leaves two neighbours in the
// halves of a register.
//   k        [page][4][NG][2] words of a token: word (lk, g, h) has dims 64 g + 16 lk + 8 h + 0..7. Of depth 64 g .. of a matrix
//            product on 16x16x32 operands, lane group lk takes words (lk, g, 0) and (lk, g, 1); its words are neighbours.
//   v        [page / 8][D] words of 8 tokens of a dim, as the second product's operand wants them
//   k_scale  [page / 8][NG][8], k_min [page][NG], v_scale, v_min [page]
// A slot is page * P + token in page.
#pragma once

#include <cfloat>

#include "capi_common.hpp"
#include "device_common.hpp"

namespace qk {
namespace {

constexpr float kKv4Floor = 0x1p-100f;   // smallest scale: every quotient and reciprocal below stays a normal number
constexpr int kKv4MaxPage = 1024;
constexpr int kKv4MaxRequests = 4096;

struct Kv4Cache {
    uint8_t* k;
    uint8_t* v;
    uint16_t* ks;
    uint16_t* km;
    uint16_t* vs;
    uint16_t* vm;
    int pages, page, heads, dim;
};

inline bool kv4_page_ok(int page) { return page >= 8 && page <= kKv4MaxPage && (page & (page - 1)) == 0; }

inline int kv4_check(const char* what, const Kv4Cache& c) {
    QK_REQUIRE(c.k && c.v && c.ks && c.km && c.vs && c.vm, "%s: null cache pointer", what);
    QK_REQUIRE(aligned16(c.k) && aligned16(c.v) && aligned16(c.ks) && aligned16(c.km) && aligned16(c.vs) && aligned16(c.vm),
               "%s: cache arrays must be 16-byte aligned", what);
    QK_REQUIRE(c.heads > 0 && c.heads <= 65535, "%s: %d KV heads", what, c.heads);
    QK_REQUIRE(c.dim == 64 || c.dim == 128 || c.dim == 256, "%s: head dim %d is not 64, 128 or 256", what, c.dim);
    QK_REQUIRE(kv4_page_ok(c.page), "%s: page size %d is not a power of two from 8 to %d", what, c.page, kKv4MaxPage);
    QK_REQUIRE(c.pages > 0 && static_cast<int64_t>(c.pages) * c.page <= 0x7fffffff, "%s: %d pages of %d tokens", what,
               c.pages, c.page);
    return QWEN_STATUS_OK;
}

__device__ __forceinline__ float bf16_value(uint16_t h) { return __uint_as_float(static_cast<uint32_t>(h) << 16); }

// What a group is held with, from its smallest and largest value.
struct Kv4Group {
    float scale, low, inverse;
};
__device__ __forceinline__ Kv4Group kv4_group(float smallest, float largest, bool bad) {
    uint32_t m = __float_as_uint(smallest);
    if ((m >> 31) && (m & 0xffffu)) m += 0x10000u;   // away from zero: down
    const float low = __uint_as_float(m & 0xffff0000u) + 0.0f;   // of zeros of either sign +0
    const double step = fmax((static_cast<double>(largest) - static_cast<double>(low)) / 15.0, static_cast<double>(kKv4Floor));
    uint32_t s = (__float_as_uint(static_cast<float>(step)) + 0xffffu) & 0xffff0000u;
    if (static_cast<double>(__uint_as_float(s)) < step) s += 0x10000u;   // the fp32 number was rounded down to a bf16 one
    if (bad || !(fabsf(low) <= FLT_MAX)) return Kv4Group{__builtin_nanf(""), 0.f, 0.f};
    return Kv4Group{__uint_as_float(s), low, 1.0f / __uint_as_float(s)};
}

// rne((x - low) / scale) of the 64-bit quotient, in fp32 where that cannot differ: (x - low) * inverse is off by less than
// 2^-18, and the 64-bit form only runs within 2^-13 of a tie (or where the difference overflows).
__device__ __forceinline__ uint32_t kv4_code(float x, const Kv4Group& g) {
    const float y = (x - g.low) * g.inverse;
    float q = rintf(y);
    if (!(fabsf(y - q) < 0.4999f))
        q = static_cast<float>(rint((static_cast<double>(x) - static_cast<double>(g.low)) / static_cast<double>(g.scale)));
    return static_cast<uint32_t>(fminf(fmaxf(q, 0.0f), 15.0f));
}

// Bits of element j's nibble in its word.
__device__ __forceinline__ int kv4_shift(int j) { return 4 * ((j >> 1) + 4 * (j & 1)); }

}  // namespace
}  // namespace qk
