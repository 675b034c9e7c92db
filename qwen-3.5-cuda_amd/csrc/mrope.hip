// Attention front end for positions with several axes (time, height, width of image and video tokens) on gfx950: per-head
// RMSNorm fused with the split-half partial RoPE whose pairs take their angle from one axis each, Q and K in place.
//   angle(t, i) = pos[axis(i)][t] * theta^(-2 i / rope_dim),  x = x * (r * w), then (a, b) -> (a c - b s, b c + a s)
// The reference has the form with one position (src/layer_attn.cpp:91-96; attn.hip).
//
// Angles: the product with 1 / (2 pi theta^(2 i / rope_dim)) is taken in 64 bits, in revolutions, and only what is left of
// it after the nearest whole one goes to 32 bits (2^-25 of a revolution). In 32 bits a position of 40000 times a frequency
// near 1 is off by 2e-3 radians.
//
// Bound by bytes (8 an element), at a few tokens by latency. A wave takes J float4 rows of 64 / LPH heads of one token (LPH
// lanes a head), all of them requested before the first angle; the token's pairs are evaluated once per wave, one a lane,
// and handed out by ds_bpermute.
#include <cmath>

#include "capi_common.hpp"
#include "device_common.hpp"

namespace qk {
namespace {

constexpr int kMropeBlock = 256;
constexpr int kMropeMaxPairs = 128;
constexpr int kMropeMaxAxes = 4;

struct MropeTable {
    double rev[kMropeMaxPairs];   // revolutions per position
    uint8_t axis[kMropeMaxPairs];
};

struct MropeArgs {
    float* q;
    float* k;
    const float* qw;
    const float* kw;
    const int32_t* pos;   // [axes][rows]
    int rows, q_heads, k_heads, head_dim, half;
    float eps;
};

__device__ __forceinline__ void angle_of(const MropeArgs& a, const MropeTable& tab, int t, int i, float& s, float& c) {
    const int p = a.pos[static_cast<size_t>(tab.axis[i]) * a.rows + t];
    const double turns = static_cast<double>(p) * tab.rev[i];
    sincospif(2.0f * static_cast<float>(turns - rint(turns)), &s, &c);
}

template <int LPH, int J>
__global__ __launch_bounds__(kMropeBlock) void mrope_vec(const MropeArgs a, const MropeTable tab) {
    constexpr int HPV = kWave / LPH, HD = 4 * LPH;   // heads of a float4 row of the wave
    const int lane = threadIdx.x & 63, lg = lane % LPH, gbase = lane - lg;
    const int hpr = a.q_heads + a.k_heads, groups = (hpr + HPV * J - 1) / (HPV * J);
    const uint32_t at = (blockIdx.y * gridDim.x + blockIdx.x) * (kMropeBlock / kWave) + wave_in_block();
    if (at >= static_cast<uint32_t>(a.rows) * static_cast<uint32_t>(groups)) return;   // the whole wave; the host checks rows * heads < 2^31
    const int wave = static_cast<int>(at);
    const int t = wave / groups, h0 = (wave - t * groups) * HPV * J + lane / LPH;
    float4 v[J];
    float* ptr[J];
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int h = min(h0 + j * HPV, hpr - 1);   // clamped: loads never branch
        ptr[j] = (h < a.q_heads ? a.q + (static_cast<size_t>(t) * a.q_heads + h) * HD
                                : a.k + (static_cast<size_t>(t) * a.k_heads + (h - a.q_heads)) * HD) + 4 * lg;
        v[j] = ld4_nt(ptr[j]);
    }
    // a tensor with no heads may come without weights: the other's are read
    const float4 wq = ld4((a.q_heads > 0 ? a.qw : a.kw) + 4 * lg), wk = ld4((a.k_heads > 0 ? a.kw : a.qw) + 4 * lg);
    const int half = a.half;
    float c0 = 1.f, s0 = 0.f, c1 = 1.f, s1 = 0.f;   // pairs lane and lane + 64
    if (lane < half) angle_of(a, tab, t, lane, s0, c0);
    if (LPH == 64 && lane + 64 < half) angle_of(a, tab, t, lane + 64, s1, c1);
    const int d0 = 4 * lg;
    const bool first = d0 < half, second = !first && d0 < 2 * half;
    const int src = gbase + (first ? lg + (half >> 2) : second ? lg - (half >> 2) : lg);
    const int i0 = first ? d0 : second ? d0 - half : 0;
    float cs[4], sn[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        cs[i] = lane_fetch(c0, (i0 + i) & 63);
        sn[i] = lane_fetch(s0, (i0 + i) & 63);
        if (LPH == 64 && half > 64) {
            const float c = lane_fetch(c1, (i0 + i) & 63), s = lane_fetch(s1, (i0 + i) & 63);
            if (i0 + i >= 64) cs[i] = c, sn[i] = s;
        }
        if (first) sn[i] = -sn[i];
        if (!first && !second) cs[i] = 1.f, sn[i] = 0.f;
    }
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int h = h0 + j * HPV;
        const float4 w = min(h, hpr - 1) < a.q_heads ? wq : wk;
        const float r = rsqrtf(group_sum<LPH>(sumsq4(v[j])) / static_cast<float>(HD) + a.eps);
        const float x[4] = {v[j].x * (r * w.x), v[j].y * (r * w.y), v[j].z * (r * w.z), v[j].w * (r * w.w)};
        float o[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float y = lane_fetch(x[i], src);
            o[i] = first || second ? x[i] * cs[i] + y * sn[i] : x[i];   // a c - b s; b c + a s
        }
        if (h < hpr) st4_nt(ptr[j], make_float4(o[0], o[1], o[2], o[3]));
    }
}

// Any head dim and alignment: a workgroup per row and head. A thread reads and writes its own pairs and dims alone.
__global__ __launch_bounds__(kMropeBlock) void mrope_any(const MropeArgs a, const MropeTable tab) {
    __shared__ float lds[kMropeBlock / kWave];
    const int hpr = a.q_heads + a.k_heads;
    const uint32_t at = blockIdx.y * gridDim.x + blockIdx.x;
    if (at >= static_cast<uint32_t>(a.rows) * static_cast<uint32_t>(hpr)) return;   // the whole workgroup
    const int t = static_cast<int>(at) / hpr, h = static_cast<int>(at) - t * hpr;
    const bool is_q = h < a.q_heads;
    float* p = is_q ? a.q + (static_cast<size_t>(t) * a.q_heads + h) * a.head_dim
                    : a.k + (static_cast<size_t>(t) * a.k_heads + (h - a.q_heads)) * a.head_dim;
    const float* w = is_q ? a.qw : a.kw;
    float ss = 0.f;
    for (int i = threadIdx.x; i < a.head_dim; i += kMropeBlock) ss += p[i] * p[i];
    ss = group_sum<kWave>(ss);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = ss;
    __syncthreads();
    ss = (lds[0] + lds[1]) + (lds[2] + lds[3]);
    const float r = rsqrtf(ss / static_cast<float>(a.head_dim) + a.eps);
    const int half = a.half;
    for (int i = threadIdx.x; i < a.head_dim - half; i += kMropeBlock) {
        if (i < half) {
            float s, c;
            angle_of(a, tab, t, i, s, c);
            const float x = p[i] * (r * w[i]), y = p[i + half] * (r * w[i + half]);
            p[i] = x * c - y * s;
            p[i + half] = y * c + x * s;
        } else {
            p[i + half] = p[i + half] * (r * w[i + half]);
        }
    }
}

template <int LPH>
void launch_vec(const MropeArgs& a, const MropeTable& tab, hipStream_t s) {
    constexpr int J = LPH == 64 ? 3 : 2;
    const int per = kWave / LPH * J;
    const int64_t waves = static_cast<int64_t>(a.rows) * ((a.q_heads + a.k_heads + per - 1) / per);
    mrope_vec<LPH, J><<<grid_of(blocks_for(waves, kMropeBlock / kWave)), kMropeBlock, 0, s>>>(a, tab);
}

}  // namespace
}  // namespace qk

using namespace qk;

extern "C" int qwen_attn_qk_norm_mrope_rows(float* q, float* k, const float* q_weight, const float* k_weight,
                                            const int32_t* pos, const int32_t* sections, int axes, int interleaved, int rows,
                                            int q_heads, int k_heads, int head_dim, float theta, float eps, void* stream) {
    QK_REQUIRE(rows >= 0 && q_heads >= 0 && k_heads >= 0, "attn_qk_norm_mrope: negative size");
    QK_REQUIRE(head_dim > 0, "attn_qk_norm_mrope: head_dim %d must be positive", head_dim);
    QK_REQUIRE(axes >= 1 && axes <= kMropeMaxAxes && sections, "attn_qk_norm_mrope: %d axes (1 to %d)", axes, kMropeMaxAxes);
    QK_REQUIRE(theta > 0.0f && std::isfinite(theta), "attn_qk_norm_mrope: theta must be positive");
    int64_t pairs = 0;
    for (int x = 0; x < axes; ++x) {
        QK_REQUIRE(sections[x] >= 0, "attn_qk_norm_mrope: section %d is negative", x);
        pairs += sections[x];
    }
    QK_REQUIRE(pairs >= 1 && pairs <= kMropeMaxPairs && 2 * pairs <= head_dim,
               "attn_qk_norm_mrope: sections of %lld pairs in a head of %d (1 to %d pairs)", static_cast<long long>(pairs), head_dim,
               kMropeMaxPairs);
    QK_REQUIRE(static_cast<int64_t>(rows) * (static_cast<int64_t>(q_heads) + k_heads) < (int64_t{1} << 31),
               "attn_qk_norm_mrope: rows x heads exceeds 2^31");
    if (rows == 0 || q_heads + k_heads == 0) return ok();
    QK_REQUIRE(pos, "attn_qk_norm_mrope: null pos");
    QK_REQUIRE(q_heads == 0 || (q && q_weight), "attn_qk_norm_mrope: null q or q_weight");
    QK_REQUIRE(k_heads == 0 || (k && k_weight), "attn_qk_norm_mrope: null k or k_weight");
    const size_t head = static_cast<size_t>(head_dim) * 4;
    const size_t nq = static_cast<size_t>(rows) * q_heads * head, nk = static_cast<size_t>(rows) * k_heads * head;
    const size_t np = static_cast<size_t>(rows) * axes * 4;
    QK_REQUIRE(apart(q, nq, k, nk) && apart(q, nq, pos, np) && apart(k, nk, pos, np) && apart(q, nq, q_weight, head) &&
                   apart(q, nq, k_weight, head) && apart(k, nk, q_weight, head) && apart(k, nk, k_weight, head),
               "attn_qk_norm_mrope: q or k overlaps another argument");
    MropeArgs a{q, k, q_weight, k_weight, pos, rows, q_heads, k_heads, head_dim, static_cast<int>(pairs), eps};
    MropeTable tab{};
    int left[kMropeMaxAxes], turn = 0;
    for (int x = 0; x < axes; ++x) left[x] = sections[x];
    // Frequency by frequency: the product's error, i 2^-53, is of a frequency that has fallen by theta^(-i / half), so that no
    // angle is further off than the first ones (a power each took 1.3 us a call).
    const double ratio = std::pow(static_cast<double>(theta), -1.0 / a.half);
    double rev = 1.0 / 6.283185307179586;
    for (int i = 0; i < a.half; ++i, rev *= ratio) {
        while (left[turn] == 0) turn = (turn + 1) % axes;   // some axis has a pair left
        tab.axis[i] = static_cast<uint8_t>(turn);
        tab.rev[i] = rev;
        --left[turn];
        if (interleaved) turn = (turn + 1) % axes;
    }
    const hipStream_t s = as_stream(stream);
    const int lph = head_dim / 4;
    const bool vec = (head_dim == 64 || head_dim == 128 || head_dim == 256) && a.half % 4 == 0 &&
                     (q_heads == 0 || (aligned16(q) && aligned16(q_weight))) &&
                     (k_heads == 0 || (aligned16(k) && aligned16(k_weight)));
    if (!vec)
        mrope_any<<<grid_of(static_cast<int64_t>(rows) * (q_heads + k_heads)), kMropeBlock, 0, s>>>(a, tab);
    else if (lph == 64)
        launch_vec<64>(a, tab, s);
    else if (lph == 32)
        launch_vec<32>(a, tab, s);
    else
        launch_vec<16>(a, tab, s);
    return check_launch("attn_qk_norm_mrope");
}
