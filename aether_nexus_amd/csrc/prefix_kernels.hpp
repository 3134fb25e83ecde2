// prefix_kernels.hpp — gfx950 attention of a batch whose sequences share a prefix:
// the prefix' pages read once for all, each sequence's own pages beside them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "engine_internal.hpp"
#include "prefill_kernels.hpp"
#include "weaver_kernels.hpp"

namespace aw {

struct PrefixArgs {
    const uint16_t* q;          // [batch][queries][q_heads][HD]
    const uint16_t* k;          // pools [blocks][16][kv_heads][HD]
    const uint16_t* v;          // k where K rows are the values
    const uint32_t* prefix_refs;
    const uint32_t* refs;       // [batch][refs_stride]
    const uint32_t* seq_own;    // [batch], or null: own_max each
    uint16_t* out;
    float* part_m;              // [kv_heads][splits][rows]
    float* part_l;
    float* part_o;              // [kv_heads][splits][rows][HD]
    uint32_t* err;
    uint32_t batch, queries, q_heads, kv_heads, gqa, causal;
    uint32_t rows, own_rows;    // query rows per kv head: of all sequences, of one
    uint32_t prefix_tokens, own_max, refs_stride;
    uint32_t prefix_splits, own_splits, splits; // splits = prefix_splits + own_splits
    uint32_t prefix_span, own_span;             // tokens of a split, a multiple of 32
    uint32_t prefix_items, prefix_tiles, own_tiles;
    uint64_t blocks;
    float scale_log2;
};

// 16 query rows of one kv head x the tokens [t0, t1) of one table, one wave, as in the
// decode over hot blocks: S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32 MFMAs, 32
// tokens a step, V read back from LDS transposed.  A row's softmax keeps its running
// maximum and sum in fp32; weights are f16 operands of the second product (each off by
// 2^-12 of itself, independently: less than the f16 store of the output).
// Tokens past `end` and tokens of a bad ref load as zeros and score -inf.
template <int HD>
struct PrefixWave {
    static constexpr int KS = HD / 32, NB = HD / 16, P = HD + 16;
    half8_t qop[KS];
    float m_run, l_run;
    float4_t oacc[NB];
    bool bad;

    // SPLIT: the products take the values' finite part; tokens whose values hold an inf or
    // NaN are then added one by one, in fp32, to the rows that see them.
    template <bool SPLIT>
    __device__ __forceinline__ void pass(const PrefixArgs& a, const uint32_t* table, uint32_t g, uint32_t t0, uint32_t t1,
                                         uint32_t end, uint32_t lim, _Float16* lds, int lane) {
        const int li = lane & 15, lg = lane >> 4;
        m_run = -INFINITY;
        l_run = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) oacc[nb] = (float4_t)0.0f;
        uint32_t held = ~0u, refv = 0;
        for (uint32_t c0 = t0; c0 < t1; c0 += 32u) {
            uint4_t kr[2][KS], vr[2][KS];
            bool ok[2];
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                const uint32_t tok = c0 + 16u * tb, blk = tok / kBlockTokens;
                const bool in = tok < end; // wave-uniform
                if (in && blk / 64u != held) { // the refs of 64 blocks, one in each lane
                    held = blk / 64u;
                    const uint32_t i = min(held * 64u + (uint32_t)lane, (end - 1u) / kBlockTokens);
                    refv = table[i] & kRefMask;
                }
                const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)refv, (int)(blk & 63u));
                ok[tb] = in && ref < a.blocks;
                bad |= in && !ok[tb];
                const uint64_t at = (((uint64_t)(ok[tb] ? ref : 0u) * kBlockTokens + li) * a.kv_heads + g) * HD + 8 * lg;
                const bool row = ok[tb] && tok + (uint32_t)li < end;
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    kr[tb][j] = row ? *(const uint4_t*)(a.k + at + 32 * j) : (uint4_t)0u;
                    vr[tb][j] = row ? *(const uint4_t*)(a.v + at + 32 * j) : (uint4_t)0u;
                }
            }
            float4_t sacc[2];
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                sacc[tb] = (float4_t)0.0f;
#pragma unroll
                for (int j = 0; j < KS; ++j) sacc[tb] = mfma16x16x32(as_h8(kr[tb][j]), qop[j], sacc[tb]);
            }
            __syncthreads(); // one wave
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int j = 0; j < KS; ++j) *(uint4_t*)(lds + (16 * tb + li) * P + 32 * j + 8 * lg) = vr[tb][j];
            __syncthreads(); // one wave
            float pf[8], mx = -INFINITY;
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool see = ok[tb] && c0 + (uint32_t)(16 * tb + 4 * lg + e) < lim;
                    pf[4 * tb + e] = see ? sacc[tb][e] * a.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, pf[4 * tb + e]);
                }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mnew = fmaxf(m_run, mx), mref = mnew == -INFINITY ? 0.0f : mnew;
            const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m_run - mnew);
            half8_t pop;
            float psum = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                pf[e] = fast_exp2(pf[e] - mref);
                psum += pf[e];
                pop[e] = (_Float16)pf[e];
            }
            l_run = l_run * alpha + psum;
            m_run = mnew;
            const _Float16* vrow = lds + (4 * lg + (li >> 2)) * P + 4 * (li & 3);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                half8_t vop = __builtin_bit_cast(
                    half8_t, __builtin_shufflevector(lds_read_tr16(vrow + 16 * nb), lds_read_tr16(vrow + 16 * P + 16 * nb), 0,
                                                     1, 2, 3, 4, 5, 6, 7));
                if constexpr (SPLIT) vop = finite_part(vop);
                oacc[nb] = mfma16x16x32(vop, pop, oacc[nb] * alpha);
            }
            if constexpr (SPLIT) {
                bool any[2] = {false, false};
#pragma unroll
                for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                    for (int j = 0; j < KS; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e)
                            any[tb] |= (vr[tb][j][e] & 0x7C00u) == 0x7C00u || (vr[tb][j][e] & 0x7C000000u) == 0x7C000000u;
#pragma unroll
                for (int tb = 0; tb < 2; ++tb) {
                    uint64_t todo = __ballot(any[tb]); // lane li + 16 lg: token li
                    todo = (todo | todo >> 16 | todo >> 32 | todo >> 48) & 0xFFFFu;
#pragma unroll 1
                    for (; todo; todo &= todo - 1u) {
                        const int tok = __builtin_ctzll(todo);
                        float p = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = __shfl(pf[4 * tb + e], li + 16 * (tok >> 2));
                            if (e == (tok & 3)) p = x;
                        }
                        const bool see = c0 + (uint32_t)(16 * tb + tok) < lim;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const half4_t x = *(const half4_t*)(lds + (16 * tb + tok) * P + 16 * nb + 4 * lg);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float f = (float)x[e];
                                if (see && !(fabsf(f) < INFINITY)) oacc[nb][e] = fmaf(p, f, oacc[nb][e]);
                            }
                        }
                    }
                }
            }
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
    }

    __device__ __forceinline__ void run(const PrefixArgs& a, const uint32_t* table, uint32_t g, uint32_t row, bool valid,
                                        uint32_t t0, uint32_t t1, uint32_t end, uint32_t lim, uint32_t slot, _Float16* lds,
                                        int lane) {
        const int lg = lane >> 4;
        const uint32_t head = g * a.gqa + row % a.gqa;
        const uint16_t* p = a.q + ((uint64_t)(row / a.gqa) * a.q_heads + head) * HD;
#pragma unroll
        for (int j = 0; j < KS; ++j) qop[j] = as_h8(*(const uint4_t*)(p + 32 * j + 8 * lg));
        bad = false;
        pass<false>(a, table, g, t0, t1, end, lim, lds, lane);
        // An inf or NaN among the sums under finite weights comes from the values, and may
        // have reached rows that do not see it (0 * inf): once more, split.
        float chk = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) chk = fmaf(oacc[nb][e], 0.0f, chk);
        if (__any(chk != 0.0f && l_run * 0.0f == 0.0f)) pass<true>(a, table, g, t0, t1, end, lim, lds, lane);
        if (bad) flag_error(a.err, kErrHotRef);
        if (!valid) return;
        const uint64_t at = ((uint64_t)g * a.splits + slot) * a.rows + row;
        if (lg == 0) {
            a.part_m[at] = m_run;
            a.part_l[at] = l_run;
        }
        if (l_run == 0.0f) return; // nothing seen: the merge takes no value of it
        float* po = a.part_o + at * HD;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) *(float4_t*)(po + 16 * nb + 4 * lg) = oacc[nb];
    }
};

template <int HD>
__global__ __launch_bounds__(64) void prefix_kernel(PrefixArgs a) {
    __shared__ __attribute__((aligned(16))) _Float16 lds[32 * (HD + 16)];
    const int lane = threadIdx.x;
    const uint32_t li = (uint32_t)lane & 15u;
    PrefixWave<HD> w;
    uint32_t t = blockIdx.x;
    if (t < a.prefix_items) {
        const uint32_t s = t % a.prefix_splits;
        t /= a.prefix_splits;
        const uint32_t tile = t % a.prefix_tiles, g = t / a.prefix_tiles, r = tile * 16u + li;
        const uint32_t t0 = s * a.prefix_span, t1 = min(t0 + a.prefix_span, a.prefix_tokens);
        w.run(a, a.prefix_refs, g, min(r, a.rows - 1u), r < a.rows, t0, t1, a.prefix_tokens, a.prefix_tokens, s, lds, lane);
        return;
    }
    t -= a.prefix_items;
    const uint32_t s = t % a.own_splits;
    t /= a.own_splits;
    const uint32_t g = t % a.kv_heads;
    t /= a.kv_heads;
    const uint32_t tile = t % a.own_tiles, b = t / a.own_tiles, r = tile * 16u + li, rc = min(r, a.own_rows - 1u);
    uint32_t n = a.seq_own ? a.seq_own[b] : a.own_max;
    if (n > a.own_max) {
        n = a.own_max;
        if (lane == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
    }
    const uint32_t i = rc / a.gqa; // query of the row: it sees n - queries + 1 + i tokens
    const uint32_t lim = a.causal ? (n + 1u + i > a.queries ? n + 1u + i - a.queries : 0u) : n;
    const uint32_t t0 = s * a.own_span, t1 = min(t0 + a.own_span, n);
    w.run(a, a.refs + (uint64_t)b * a.refs_stride, g, b * a.own_rows + rc, r < a.own_rows, t0, t1, n, lim,
          a.prefix_splits + s, lds, lane);
}

// Joins a row's splits: the largest maximum, each split's sums times 2^(its maximum -
// that), in the order of the splits; zeros where no split saw a token.  An inf or NaN
// in a split's sum stays in the result.  Wave per row.
template <int HD>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a) {
    constexpr int V = HD / 64;
    const uint32_t lane = threadIdx.x & 63u;
    const uint64_t id = (uint64_t)blockIdx.x * 4u + (threadIdx.x >> 6);
    if (id >= (uint64_t)a.kv_heads * a.rows) return;
    const uint32_t g = (uint32_t)(id / a.rows), r = (uint32_t)(id % a.rows);
    const uint64_t at = (uint64_t)g * a.splits * a.rows + r;
    const bool in = lane < a.splits;
    const float l = in ? a.part_l[at + (uint64_t)lane * a.rows] : 0.0f;
    const float m = l != 0.0f ? a.part_m[at + (uint64_t)lane * a.rows] : -INFINITY;
    const float M = wave_max(m);
    const float f = l != 0.0f ? fast_exp2(m - M) : 0.0f;
    const float L = wave_sum(f * l);
    float acc[V] = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float fs = __shfl(f, (int)s);
        if (fs == 0.0f) continue; // uniform
        const float* po = a.part_o + (at + (uint64_t)s * a.rows) * HD + V * lane;
#pragma unroll
        for (int e = 0; e < V; ++e) acc[e] = fmaf(fs, po[e], acc[e]);
    }
    uint16_t* out = a.out + ((uint64_t)(r / a.gqa) * a.q_heads + g * a.gqa + r % a.gqa) * HD + V * lane;
#pragma unroll
    for (int e = 0; e < V; ++e) out[e] = __builtin_bit_cast(uint16_t, (_Float16)(L == 0.0f ? 0.0f : acc[e] / L));
}

} // namespace aw
