// tree_kernels.hpp — gfx950 attention of trees of drafted tokens over pages: each node
// sees its sequence's tokens in pages, its ancestors and itself.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "engine_internal.hpp"
#include "prefix_kernels.hpp"

namespace aw {

struct TreeArgs {
    const uint16_t *q, *k, *v;  // rows [token][heads][HD], *_stride halves from token to token; v is k where K rows are the values
    const uint16_t *hk, *hv;    // pools [blocks][16][kv_heads][HD]
    const uint32_t *refs, *seq_held, *token_offsets, *mask;
    uint16_t* out;
    float *part_m, *part_l;     // [2 work_groups][kPrefixRows]
    float* part_o;              // [2 work_groups][kPrefixRows][HD]
    uint32_t* cuts;             // [work_groups][kCutWords]
    uint32_t* err;
    uint64_t q_stride, k_stride, v_stride, out_stride, blocks;
    uint32_t batch, tokens, q_heads, kv_heads, gqa, hot_count, refs_stride, mask_words;
    uint32_t work_groups;       // a multiple of 8
    uint32_t q_and, q_xor;
    float scale_log2;           // > 0
};

// A sequence's share of the work: a unit is kPrefixRows query rows of a kv head, a step
// kPrefixTok tokens of it, first those in pages, then the nodes.
struct TreeSeq {
    uint32_t first, nodes, held; // its rows, its tokens in pages
    uint32_t tiles, paged, steps; // units of a kv head, steps of a unit
    __device__ uint64_t all(uint32_t kv_heads) const { return (uint64_t)kv_heads * tiles * steps; }
};
__device__ inline TreeSeq tree_seq(const TreeArgs& a, uint32_t b, bool report) {
    TreeSeq s;
    uint32_t end;
    if (a.token_offsets) {
        s.first = a.token_offsets[b];
        end = a.token_offsets[b + 1u];
    } else {
        s.first = b * (a.tokens / a.batch);
        end = s.first + a.tokens / a.batch;
    }
    s.held = a.seq_held ? a.seq_held[b] : 0u;
    const uint32_t most = a.hot_count * kBlockTokens;
    const bool rows = s.first <= end && end <= a.tokens;
    s.nodes = rows ? end - s.first : 0u;
    if (report && (!rows || s.held > most || (a.mask && s.nodes > 32u * a.mask_words))) flag_error(a.err, aw_engine_internal::kErrSeqBit);
    s.held = min(s.held, most);
    s.tiles = (s.nodes * a.gqa + kPrefixRows - 1u) / kPrefixRows;
    s.paged = (s.held + (uint32_t)kPrefixTok - 1u) / (uint32_t)kPrefixTok;
    s.steps = s.paged + (s.nodes + (uint32_t)kPrefixTok - 1u) / (uint32_t)kPrefixTok;
    return s;
}

// What a merge needs of a unit that is cut: its parts, its rows and where they go.
constexpr uint32_t kCutWords = 6; // parts (0: no unit begins and is cut here), rows, row0, first, kv head, unused

// The steps of all units, laid end to end (sequence, kv head, rows, tokens), are shared out
// equally: work-group w takes those from w / work_groups of them on, so lengths may differ as
// they like.  A unit that lies in one work-group is normed and stored; of one that is cut
// each part's sums go to the workspace, at most two of a work-group: slot 2 w + 1 for the
// unit that begins here and is cut, 2 w for one that began before.
template <int HD>
__global__ __launch_bounds__(kPrefixThreads) __attribute__((amdgpu_waves_per_eu(2))) void tree_kernel(TreeArgs a) {
    extern __shared__ __attribute__((aligned(16))) _Float16 prefix_lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    // Work-group b runs on XCD b % 8: neighbours in the line, which read the same pages for
    // several tiles of rows, run on one XCD.
    const uint32_t w = (blockIdx.x & 7u) * (a.work_groups >> 3) + (blockIdx.x >> 3);
    uint64_t* s_sum = (uint64_t*)prefix_lds; // [4] sums of waves, [2] the sequence found
    auto wave_sum64 = [](uint64_t x) {
#pragma unroll
        for (int o = 32; o; o /= 2) x += (uint64_t)__shfl_xor((uint32_t)(x >> 32), o) << 32 | __shfl_xor((uint32_t)x, o);
        return x;
    };
    // All steps, and this work-group's.
    uint64_t mine = 0;
    for (uint32_t b = tid; b < a.batch; b += 256u) mine += tree_seq(a, b, blockIdx.x == 0).all(a.kv_heads);
    const uint64_t part = wave_sum64(mine);
    if (lane == 0) s_sum[wave] = part;
    __syncthreads();
    const uint64_t total = s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3], each = (total + a.work_groups - 1u) / a.work_groups;
    __syncthreads();
    uint64_t pos = (uint64_t)w * each;
    const uint64_t end = pos + each < total ? pos + each : total;
    uint32_t* cut = a.cuts + (uint64_t)w * kCutWords;
    if (pos >= end) {
        if (tid == 0) cut[0] = 0;
        return;
    }
    // The sequence that holds the first of them: 256 at a time.
    uint64_t base = 0;
    uint32_t b = 0;
    for (uint32_t c0 = 0; c0 < a.batch; c0 += 256u) {
        const uint64_t x = c0 + tid < a.batch ? tree_seq(a, c0 + tid, false).all(a.kv_heads) : 0u;
        uint64_t sum = x;
#pragma unroll
        for (int o = 1; o < 64; o *= 2) {
            const uint64_t y = (uint64_t)__shfl_up((uint32_t)(sum >> 32), o) << 32 | __shfl_up((uint32_t)sum, o);
            if (lane >= (uint32_t)o) sum += y;
        }
        if (lane == 63u) s_sum[wave] = sum;
        __syncthreads();
        uint64_t before = base, all = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            if (i < wave) before += s_sum[i];
            all += s_sum[i];
        }
        sum += before;
        if (sum - x <= pos && pos < sum) { // one thread
            s_sum[4] = sum - x;
            s_sum[5] = c0 + tid;
        }
        const bool here = pos < base + all; // uniform
        __syncthreads();
        if (here) {
            base = s_sum[4];
            b = (uint32_t)s_sum[5];
            break;
        }
        base += all;
    }
    __syncthreads(); // the sums have been read
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    auto uniform64 = [&](uint64_t x) { return (uint64_t)uniform((uint32_t)(x >> 32)) << 32 | uniform((uint32_t)x); };
    b = uniform(b);
    pos = uniform64(pos);
    base = uniform64(base);
    const uint64_t stop = uniform64(end), share = uniform64(each);
    uint32_t parts = 0, cut_rows = 0, cut_row0 = 0, cut_first = 0, cut_g = 0;
    for (; pos < stop; ++b) {
        TreeSeq s = tree_seq(a, b, false);
        s.first = uniform(s.first);
        s.nodes = uniform(s.nodes);
        s.held = uniform(s.held);
        s.tiles = uniform(s.tiles);
        s.paged = uniform(s.paged);
        s.steps = uniform(s.steps);
        const uint64_t all = uniform64(s.all(a.kv_heads));
        while (pos < stop && pos - base < all) {
            const uint32_t unit = uniform((uint32_t)((pos - base) / s.steps)), s0 = uniform((uint32_t)((pos - base) - (uint64_t)unit * s.steps));
            const uint32_t s1 = uniform((uint32_t)min((uint64_t)s.steps, s0 + (stop - pos)));
            const uint32_t g = uniform(unit / s.tiles), row0 = (unit - g * s.tiles) * kPrefixRows;
            const bool whole = s0 == 0 && s1 == s.steps;
            const uint64_t slot = (2ull * w + (s0 == 0 ? 1u : 0u)) * kPrefixRows;
            const uint32_t t0 = min(s0 * (uint32_t)kPrefixTok, s.held), t1 = min(s1 * (uint32_t)kPrefixTok, s.held);
            TilePart p{};
            p.q = a.q + s.first * a.q_stride + (uint64_t)g * a.gqa * HD;
            p.k = a.hk + (uint64_t)g * HD;
            p.v = a.hv + (uint64_t)g * HD;
            p.table = a.refs + (uint64_t)b * a.refs_stride + s0 * (uint32_t)(kPrefixTok / 16);
            p.q_step = a.q_stride;
            p.blocks = a.blocks;
            p.rstride = a.kv_heads * (uint32_t)HD;
            p.gqa = a.gqa;
            p.rows = s.nodes * a.gqa;
            p.row0 = row0;
            p.tokens = t1 - t0;
            p.q_and = a.q_and;
            p.q_xor = a.q_xor;
            p.scale_log2 = a.scale_log2;
            p.m = a.part_m + slot - row0;
            p.l = a.part_l + slot - row0;
            p.o = a.part_o + (int64_t)(slot - row0) * HD;
            p.err = a.err;
            p.nk = a.k + s.first * a.k_stride + (uint64_t)g * HD;
            p.nv = a.v + s.first * a.v_stride + (uint64_t)g * HD;
            p.nk_step = a.k_stride;
            p.nv_step = a.v_stride;
            p.mask = a.mask ? a.mask + (uint64_t)s.first * a.mask_words : nullptr;
            p.mask_words = a.mask_words;
            p.node0 = s0 > s.paged ? (s0 - s.paged) * (uint32_t)kPrefixTok : 0u;
            p.nodes = s1 > s.paged ? min((s1 - s.paged) * (uint32_t)kPrefixTok, s.nodes) : p.node0;
            p.out = whole ? a.out + s.first * a.out_stride + (uint64_t)g * a.gqa * HD : nullptr;
            p.o_step = a.out_stride;
            p.turn = blockIdx.x >= a.work_groups / 2u ? 2u : 0u;
            PrefixTile<HD, true>::run(p, prefix_lds);
            __syncthreads(); // the tile's LDS has been read
            if (s0 == 0 && !whole) { // the last of this work-group
                cut_rows = min(kPrefixRows, p.rows - row0);
                cut_row0 = row0;
                cut_first = s.first;
                cut_g = g;
                parts = 1u + (uint32_t)((s.steps - s1 + share - 1u) / share);
            }
            pos += s1 - s0;
        }
        base += all;
    }
    if (tid == 0) {
        cut[0] = parts;
        cut[1] = cut_rows;
        cut[2] = cut_row0;
        cut[3] = cut_first;
        cut[4] = cut_g;
    }
}

// Joins the parts of the units that are cut, a wave a row: their largest maximum, each
// part's sums times 2^(its maximum - that), in the order of the parts; zeros where no part saw a
// token.  An inf or NaN in a part's sum stays, as in prefix_merge_kernel.
constexpr uint32_t kTreeMergeRows = 8; // of a work-group
template <int HD>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr int LP = HD / 4, PG = 64 / LP, U = 4; // lanes of a part's row, parts of one load, loads in flight
    const uint32_t w = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t* cut = a.cuts + (uint64_t)w * kCutWords;
    const uint32_t S = cut[0], rows = cut[1], row0 = cut[2], first = cut[3], g = cut[4];
    if (!S) return;
    const uint32_t sub = lane / LP, d = 4u * (lane % LP);
    for (uint32_t r = blockIdx.y * kTreeMergeRows + wave; r < min(rows, (blockIdx.y + 1u) * kTreeMergeRows); r += 4u) {
        auto slot = [&](uint32_t p) { return (p ? 2ull * (w + p) : 2ull * w + 1u) * kPrefixRows + r; };
        float M = -INFINITY;
        for (uint32_t p = lane; p < S; p += 64u)
            if (a.part_l[slot(p)] != 0.0f) M = fmaxf(M, a.part_m[slot(p)]);
        M = wave_max(M);
        float L = 0.0f;
        float4_t acc = (float4_t)0.0f;
        for (uint32_t p0 = 0; p0 < S; p0 += (uint32_t)(U * PG)) {
            float4_t v[U];
            float m[U], l[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const uint64_t at = slot(min(p0 + (uint32_t)(j * PG) + sub, S - 1u));
                v[j] = *(const float4_t*)(a.part_o + at * HD + d);
                m[j] = a.part_m[at];
                l[j] = a.part_l[at];
            }
#pragma unroll
            for (int j = 0; j < U; ++j)
                if (p0 + (uint32_t)(j * PG) + sub < S && l[j] != 0.0f) { // a part that saw nothing holds no sums
                    const float f = fast_exp2(m[j] - M);
                    L = fmaf(f, l[j], L);
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = fmaf(f, v[j][e], acc[e]);
                }
        }
#pragma unroll
        for (int o = LP; o < 64; o *= 2) {
            L += __shfl_xor(L, o);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
        }
        if (sub) continue;
        const uint32_t R = row0 + r;
        half4_t h;
#pragma unroll
        for (int e = 0; e < 4; ++e) h[e] = (_Float16)(L == 0.0f ? 0.0f : acc[e] / L);
        *(half4_t*)(a.out + (first + R / a.gqa) * a.out_stride + (g * a.gqa + R % a.gqa) * (uint64_t)HD + d) = h;
    }
}

} // namespace aw
