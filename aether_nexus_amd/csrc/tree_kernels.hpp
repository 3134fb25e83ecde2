// tree_kernels.hpp — gfx950 attention of trees of drafted tokens over pages: each node
// sees its sequence's tokens in pages, its ancestors and itself.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "engine_internal.hpp"
#include "weaver_kernels.hpp"

namespace aw {

struct TreeArgs {
    const uint16_t *q, *k, *v;  // rows [token][heads][HD], *_stride halves from token to token; v is k where K rows are the values
    const uint16_t *hk, *hv;    // pools [blocks][16][kv_heads][HD]
    const uint32_t *refs, *seq_held, *token_offsets, *mask;
    uint16_t* out;
    uint32_t* err;
    uint64_t q_stride, k_stride, v_stride, out_stride, blocks;
    uint32_t batch, tokens, q_heads, kv_heads, gqa, hot_count, refs_stride, mask_words;
    float scale_log2;
};

// The simplest form: a work-group a row and query head, its 4 waves every fourth token, a
// token's dims over the lanes.
template <int HD>
__global__ __launch_bounds__(256) void tree_row_kernel(TreeArgs a) {
    constexpr int E = HD / 64;
    __shared__ float s_m[4], s_l[4], s_o[4][HD];
    const uint32_t t = blockIdx.x, head = blockIdx.y, g = head / a.gqa;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t b = 0, first = 0, n = 0;
    if (a.token_offsets) {
        for (; b < a.batch; ++b) {
            if (a.token_offsets[b + 1] < a.token_offsets[b] && threadIdx.x == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
            if (a.token_offsets[b + 1] > t) break;
        }
        if (b >= a.batch) return;
        first = a.token_offsets[b];
        const uint32_t end = a.token_offsets[b + 1];
        if (first > t || end > a.tokens) {
            if (threadIdx.x == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
            return;
        }
        n = end - first;
    } else {
        n = a.tokens / a.batch;
        b = t / n;
        first = b * n;
    }
    if (a.mask && n > 32u * a.mask_words && threadIdx.x == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
    uint32_t held = a.seq_held ? a.seq_held[b] : 0u;
    if (held > a.hot_count * kBlockTokens) {
        held = a.hot_count * kBlockTokens;
        if (threadIdx.x == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
    }
    float q[E], o[E] = {}, m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) q[e] = h2f_bits(a.q[t * a.q_stride + (uint64_t)head * HD + 64 * e + lane]);
    for (uint32_t p = wave; p < held + n; p += 4u) {
        const uint16_t *kr, *vr;
        if (p < held) {
            const uint32_t ref = a.refs[(uint64_t)b * a.refs_stride + p / kBlockTokens] & kRefMask;
            if (ref >= a.blocks) {
                if (lane == 0) flag_error(a.err, kErrHotRef);
                continue;
            }
            const uint64_t at = (((uint64_t)ref * kBlockTokens + p % kBlockTokens) * a.kv_heads + g) * HD;
            kr = a.hk + at;
            vr = a.hv + at;
        } else {
            const uint32_t j = p - held;
            const bool see = a.mask ? j < 32u * a.mask_words && (a.mask[(uint64_t)t * a.mask_words + j / 32u] >> (j % 32u) & 1u) : j <= t - first;
            if (!see) continue;
            kr = a.k + (first + j) * a.k_stride + (uint64_t)g * HD;
            vr = a.v + (first + j) * a.v_stride + (uint64_t)g * HD;
        }
        float s = 0.0f;
        for (int e = 0; e < E; ++e) s += q[e] * h2f_bits(kr[64 * e + lane]);
        s = wave_sum(s) * a.scale_log2;
        const float mn = fmaxf(m, s), f = mn == -INFINITY ? 1.0f : fast_exp2(m - mn), w = mn == -INFINITY ? 0.0f : fast_exp2(s - mn);
        l = l * f + w;
        m = mn;
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * h2f_bits(vr[64 * e + lane]);
    }
    if (lane == 0) {
        s_m[wave] = m;
        s_l[wave] = l;
    }
    for (int e = 0; e < E; ++e) s_o[wave][64 * e + lane] = o[e];
    __syncthreads();
    if (wave) return;
    const float M = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
    float L = 0.0f, sum[E] = {};
    for (int w = 0; w < 4; ++w) {
        const float f = s_l[w] != 0.0f ? fast_exp2(s_m[w] - M) : 0.0f;
        L += f * s_l[w];
        if (s_l[w] != 0.0f)
            for (int e = 0; e < E; ++e) sum[e] += f * s_o[w][64 * e + lane];
    }
    for (int e = 0; e < E; ++e)
        a.out[t * a.out_stride + (uint64_t)head * HD + 64 * e + lane] =
            __builtin_bit_cast(uint16_t, (_Float16)(L == 0.0f ? 0.0f : sum[e] / L));
}

} // namespace aw
