// rotary_kernels.hpp — gfx950 kernels that turn q and k heads by their positions:
// alone, after an RMS norm of each head, or on the way into the pages of a paged cache.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ops_kernels.hpp"

#pragma clang fp contract(off)

namespace awo {

constexpr uint32_t kRotaryMaxDim = 1024;  // head_dim; half as many cosines and sines in LDS
constexpr uint32_t kPageTokens = 16;      // tokens per page (a hot block)
constexpr uint32_t kPageMask = 0x7FFFFFFFu;
constexpr uint32_t kErrPage = 1u;         // a page of an append (the hot block ref bit)
constexpr uint32_t kErrSeq = aw_engine_internal::kErrSeqBit;

struct RotaryArgs {
    const uint16_t *q, *k, *v;    // rows [token][heads][hd], `*_stride` halves from token to token
    uint16_t *q_out, *k_out;      // append: k_out and v_out are the pools [block][16][kv_heads][hd]
    uint16_t* v_out;              // append: null where K rows are the values too
    uint64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const uint16_t *q_norm, *k_norm; // [hd], or null: no norm
    const uint32_t* positions;    // [tokens], or null: start + (append: the token's place in its sequence, else its index)
    const double* inv_freq;       // [rotary_dim / 2] radians per position
    uint32_t tokens, q_heads, kv_heads, hd, rotary_dim, interleaved, start;
    float magnitude, eps;
    // append
    uint32_t batch, hot_count, refs_stride;
    uint64_t hot_blocks;
    const uint32_t *refs, *seq_hot, *token_offsets; // token_offsets null: tokens / batch each
    uint32_t* err;
};

// Where a token of an append goes.
struct Place {
    bool rows;     // the token belongs to a sequence: its q row is written
    bool page;     // ... and to a page of it: so are its k and v rows
    uint32_t at;   // its place in the sequence's pages
    uint64_t row;  // its row of the pools
};

// Token t of an append: the sequence whose tokens hold it, its place behind the tokens
// that the sequence had, the page of the block table.  Every lane of a wave asks for
// the same token; the offsets are read 64 at a time, so the search is one or two round
// trips to L2, not a chain of them.
__device__ inline Place find_place(const RotaryArgs& a, uint32_t t, uint32_t lane, bool report) {
    uint32_t b, first, end;
    if (a.token_offsets) {
        b = 0;
        for (uint32_t i = 0; i < a.batch; i += 64u) {
            const uint32_t at = i + lane;
            b += (uint32_t)__popcll(__ballot(at < a.batch && a.token_offsets[min(at, a.batch - 1u) + 1u] <= t));
        }
        if (b >= a.batch) return {false, false, 0, 0}; // behind the last sequence
        first = a.token_offsets[b];
        end = a.token_offsets[b + 1u];
    } else {
        const uint32_t each = a.tokens / a.batch;
        b = t / each;
        first = b * each;
        end = first + each;
    }
    const uint32_t held = a.seq_hot[b], n = end - first;
    if (t < first || t >= end || n > held) { // offsets that do not ascend, or more new tokens than the sequence has
        if (report && lane == 0) flag(a.err, kErrSeq);
        return {false, false, 0, 0};
    }
    const uint32_t at = held - n + (t - first), page = at / kPageTokens;
    const uint32_t ref = page < a.hot_count ? a.refs[(uint64_t)b * a.refs_stride + page] & kPageMask : kPageMask;
    const bool ok = page < a.hot_count && ref < a.hot_blocks;
    if (!ok && report && lane == 0) flag(a.err, kErrPage);
    return {true, ok, at, (uint64_t)ref * kPageTokens + at % kPageTokens};
}

// Cosine and sine (times the magnitude) of pair p at a position.  The angle is taken in
// 64 bits, as turns: a position of 10^6 times 2^-24 would be off by 0.06 radians in 32.
// What is left of it after whole turns is at most half a turn and fits 32 bits.
__device__ inline float2 turn_of(const RotaryArgs& a, uint32_t p, uint32_t position) {
    const double turns = (double)position * (a.inv_freq[p] * 0.15915494309189533577);
    float s, c;
    sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
    return make_float2(c * a.magnitude, s * a.magnitude);
}

// Any head_dim, rotary_dim, stride and alignment: work-group = one token, a wave per
// head in turn, lanes over the pairs and then over the dims that pass.
template <bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 s_turn[kRotaryMaxDim / 2];
    const uint32_t t = blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    Place place{true, true, t, 0};
    if constexpr (APPEND) place = find_place(a, t, lane, wave == 0);
    if (!place.rows) return; // the same in every wave
    const uint32_t half = a.rotary_dim / 2;
    const uint32_t position = a.positions ? a.positions[t] : a.start + place.at;
    for (uint32_t p = tid; p < half; p += 256u) s_turn[p] = turn_of(a, p, position);
    __syncthreads();
    const uint32_t heads = a.q_heads + a.kv_heads + (APPEND && a.v_out ? a.kv_heads : 0u);
    for (uint32_t h = wave; h < heads; h += 4u) {
        const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + a.kv_heads;
        const uint32_t g = is_q ? h : (is_v ? h - a.q_heads - a.kv_heads : h - a.q_heads);
        const uint16_t* x = (is_q ? a.q + t * a.q_stride : is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride) + (uint64_t)g * a.hd;
        uint16_t* y;
        if (is_q) {
            y = a.q_out + t * a.q_out_stride + (uint64_t)g * a.hd;
        } else if constexpr (APPEND) {
            if (!place.page) continue;
            y = (is_v ? a.v_out : a.k_out) + (place.row * a.kv_heads + g) * a.hd;
        } else {
            y = a.k_out + t * a.k_out_stride + (uint64_t)g * a.hd;
        }
        if (is_v) {
            for (uint32_t d = lane; d < a.hd; d += 64u) y[d] = x[d];
            continue;
        }
        const uint16_t* w = is_q ? a.q_norm : a.k_norm;
        float inv = 1.0f;
        if (w) {
            float sum = 0.0f;
            for (uint32_t d = lane; d < a.hd; d += 64u) sum += h2f(x[d]) * h2f(x[d]);
            for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
            inv = 1.0f / sqrtf(sum / (float)a.hd + a.eps);
        }
        auto value = [&](uint32_t d) { return w ? h2f(x[d]) * inv * h2f(w[d]) : h2f(x[d]); };
        for (uint32_t p = lane; p < half; p += 64u) {
            const uint32_t d0 = a.interleaved ? 2u * p : p, d1 = a.interleaved ? 2u * p + 1u : p + half;
            const float x0 = value(d0), x1 = value(d1);
            const float2 cs = s_turn[p];
            y[d0] = f2h(x0 * cs.x - x1 * cs.y);
            y[d1] = f2h(x0 * cs.y + x1 * cs.x);
        }
        for (uint32_t d = a.rotary_dim + lane; d < a.hd; d += 64u) y[d] = w ? f2h(value(d)) : x[d];
    }
}

} // namespace awo
