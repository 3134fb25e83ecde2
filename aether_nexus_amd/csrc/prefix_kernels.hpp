// prefix_kernels.hpp — gfx950 attention of a batch whose sequences share a prefix:
// the prefix' pages read once for all, each sequence's own pages beside them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "engine_internal.hpp"
#include "prefill_kernels.hpp"
#include "weaver_kernels.hpp"

namespace aw {

// lds_read_tr16 of data whose loads into LDS this kernel has waited for itself.  Without
// the restrict (any alias information does) the compiler puts a wait for every load into
// LDS before such a read.
__device__ __forceinline__ short4_t lds_read_tr16_waited(const _Float16* __restrict__ p) { return lds_read_tr16(p); }

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
    uint32_t prefix_splits, own_splits, splits; // splits = prefix_splits + own_splits, or 0: no parts to join
    uint32_t prefix_span, own_span;             // tokens of a split, a multiple of 64
    uint32_t prefix_wgs, work_groups;           // work-groups of PrefixTile parts, all
    uint32_t prefix_units, own_units;           // 16 rows x a part of a table, kv_heads work-groups each
    uint32_t prefix_tiles, own_tiles;
    uint64_t blocks;
    float scale_log2;           // > 0
    uint32_t q_and, q_xor;      // of two halves of q: the sign of the scale, or all zero for a scale of 0
};

// 8 halves of a query row, with the scale's sign.
__device__ __forceinline__ half8_t prefix_query(const uint16_t* p, uint32_t q_and, uint32_t q_xor) {
    uint4_t w = *(const uint4_t*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (w[e] & q_and) ^ q_xor;
    return as_h8(w);
}

// Few rows to a table (a sequence's own pages; a prefix that few rows see, or a short
// one): a work-group takes 16 query rows of one kv head x a run of pages, its 4 waves the
// pages in turn, each on its own until the waves' sums meet in LDS.  A page's K and V go
// from memory straight into LDS, 256 bytes (128 dims) of a row side by side, kPageBufs
// pages a wave.
//   S^T = K Q^T on v_mfma_f32_16x16x32_f16 (lane li + 16 lg): A = K (token li, dims 32 j
//     + 8 lg ..), B = Q^T from registers; a lane ends with tokens 4 lg .. + 3 of row li;
//   O^T += V^T P^T on v_mfma_f32_16x16x16_f16: B = P^T from the same registers, A = V^T
//     (dim 16 nb + li, tokens 4 lg ..) by transposing LDS reads.
// A row's softmax keeps its running maximum and sum in fp32; weights are f16 operands of
// the second product (each off by 2^-12 of itself on average, independently: less than
// the f16 store of the output).  Staged rows are HD / 8 16-byte chunks, chunk c of K row
// r at c ^ r, of V row r at c ^ vsw(r): no bank conflict at 128 dims.
// Bound: HBM, the pages' bytes (96 sequences of up to 1500 own tokens of 8 heads x 128,
// 290 MB: 4.2 to 4.4 TB/s); few pages: a chain of refs, pages, products, sums (2
// sequences behind 117 tokens 5 us, half of it the launch).
constexpr int kPageBufs = 2;
constexpr size_t pages_lds_bytes(int HD) {
    const size_t ring = (size_t)4 * kPageBufs * 2 * 16 * HD * 2, sums = (size_t)4 * 16 * (HD + 4) * 4 + 4 * 16 * 2 * 4;
    return ring > sums ? ring : sums;
}

// A stretch of one table for 16 rows: pages [p0, p1) of it, tokens below `end`, of which
// this lane's row sees those below `lim`.
struct PageRun {
    const uint32_t* table;
    uint32_t p0, p1, end, lim;
};

template <int HD>
struct PrefixPages {
    static constexpr int CH = HD / 8, KS = HD / 32, NB = HD / 16, P = HD + 4;
    static constexpr int LPP = CH / 4;                     // loads of a wave for a page of K (or V)
    static constexpr uint32_t OP = 16 * HD;                // halves of a staged page operand
    half8_t qop[KS];
    float m_run, l_run;
    float4_t oacc[NB];
    bool bad;

    static __device__ __forceinline__ uint32_t ksw(uint32_t row) { return row & (uint32_t)(CH - 1); }
    static __device__ __forceinline__ uint32_t vsw(uint32_t row) {
        return CH == 16 ? ((row & 3u) << 2) | ((row >> 2) & 3u) : ((row >> 1) & 1u) << 2;
    }

    // This wave's pages of the runs.  SPLIT: the products take the values' finite part;
    // tokens whose values hold an inf or NaN are then added one by one, in fp32, to the
    // rows that see them.
    template <bool SPLIT, int RUNS>
    __device__ __forceinline__ void pass(const PrefixArgs& a, const PageRun (&runs)[RUNS], uint32_t g, _Float16* lds, int lane, uint32_t wave) {
        const int li = lane & 15, lg = lane >> 4;
        m_run = -INFINITY;
        l_run = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) oacc[nb] = (float4_t)0.0f;
        const uint32_t n0 = runs[0].p1 - runs[0].p0, n = n0 + (RUNS > 1 ? runs[RUNS - 1].p1 - runs[RUNS - 1].p0 : 0u);
        if (wave >= n) return; // wave-uniform
        const uint32_t mine = (n - wave + 3u) / 4u; // pages wave, wave + 4, ..
        // Page i of this wave: its run and its place there.
        auto place = [&](uint32_t i, uint32_t& p) -> const PageRun& {
            p = wave + 4u * i;
            if (RUNS > 1 && p >= n0) {
                p = runs[RUNS - 1].p0 + (p - n0);
                return runs[RUNS - 1];
            }
            p += runs[0].p0;
            return runs[0];
        };
        // Refs of this wave's pages, 64 at a time, one in each lane, and of the next 64.
        auto refs_from = [&](uint32_t from) {
            uint32_t p;
            const uint32_t i = min(from + (uint32_t)lane, mine - 1u), q = wave + 4u * i;
            const bool second = RUNS > 1 && q >= n0;
            p = second ? runs[RUNS - 1].p0 + (q - n0) : runs[0].p0 + q;
            return (second ? runs[RUNS - 1].table : runs[0].table)[p] & kRefMask;
        };
        uint32_t held = 0, ref_cur = 0, ref_next = refs_from(0);
        uint64_t ok_cur = 0, ok_old = 0;
        auto take = [&] {
            const bool ok = ref_next < a.blocks;
            ref_cur = ok ? ref_next : 0u;
            ok_old = ok_cur;
            ok_cur = __ballot(ok);
            bad |= !ok;
        };
        take();
        ref_next = refs_from(64u);
        // Staging: load j of a page fills slots lane + 64 j (slot -> row, chunk).
        const uint32_t rstride = a.kv_heads * (uint32_t)HD;
        _Float16* ring = lds + wave * (uint32_t)(kPageBufs * 2) * OP;
        auto load = [&](uint32_t i) {
            if (i / 64u != held) {
                held = i / 64u;
                take();
                ref_next = refs_from((held + 1u) * 64u);
            }
            uint32_t p;
            const PageRun& r = place(i, p);
            const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)ref_cur, (int)(i & 63u));
            const uint32_t rows = min(16u, r.end - p * 16u); // rows past the end load the last one (and count for nothing)
            const uint64_t at = (uint64_t)ref * (16u * rstride) + (uint64_t)g * HD;
            _Float16* dst = ring + (i % (uint32_t)kPageBufs) * 2u * OP;
#pragma unroll
            for (int o = 0; o < 2; ++o)
#pragma unroll
                for (int j = 0; j < LPP; ++j) {
                    const uint32_t slot = (uint32_t)(lane + 64 * j), row = slot / CH, c = slot % CH;
                    const uint16_t* src = (o ? a.v : a.k) + at + min(row, rows - 1u) * rstride + 8u * (c ^ (o ? vsw(row) : ksw(row)));
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                                     (__attribute__((address_space(3))) void*)(dst + (uint32_t)o * OP + 512u * j), 16, 0, 0);
                }
        };
        auto wait = [](auto pages) {
            constexpr uint32_t vm = (uint32_t)decltype(pages)::value * 2u * (uint32_t)LPP;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt((short)((vm & 15u) | ((vm >> 4) << 14) | (7u << 4) | (15u << 8))); // vmcnt(vm)
            __asm__ volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (int i = 0; i < kPageBufs - 1; ++i)
            if ((uint32_t)i < mine) load((uint32_t)i);
        for (uint32_t i = 0; i < mine; ++i) {
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); // the page before has been read
            if (i + (uint32_t)kPageBufs - 1u < mine) {
                load(i + (uint32_t)kPageBufs - 1u);
                wait(std::integral_constant<int, kPageBufs - 1>{});
            } else {
                wait(std::integral_constant<int, 0>{});
            }
            uint32_t p;
            const PageRun& r = place(i, p);
            const bool ok = ((i / 64u == held ? ok_cur : ok_old) >> (i & 63u)) & 1u;
            const _Float16 *sk = ring + (i % (uint32_t)kPageBufs) * 2u * OP, *sv = sk + OP;
            float4_t sacc = (float4_t)0.0f;
#pragma unroll
            for (int j = 0; j < KS; ++j)
                sacc = mfma16x16x32(*(const half8_t*)(sk + li * HD + 8 * ((4 * j + lg) ^ (int)ksw((uint32_t)li))), qop[j], sacc);
            const uint32_t rlim = ok ? min(r.lim, r.end) : 0u;
            float pf[4], mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pf[e] = p * 16u + (uint32_t)(4 * lg + e) < rlim ? sacc[e] * a.scale_log2 : -INFINITY;
                mx = fmaxf(mx, pf[e]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mnew = fmaxf(m_run, mx), mref = mnew == -INFINITY ? 0.0f : mnew;
            const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m_run - mnew);
            half4_t pop;
            float psum = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                pf[e] = fast_exp2(pf[e] - mref);
                psum += pf[e];
                pop[e] = (_Float16)pf[e];
            }
            l_run = l_run * alpha + psum;
            m_run = mnew;
            const uint32_t vr = 4u * (uint32_t)lg + ((uint32_t)li >> 2), vc = ((uint32_t)li & 3u) >> 1, vlo = 4u * ((uint32_t)li & 1u);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                half4_t v = __builtin_bit_cast(half4_t, lds_read_tr16_waited(sv + vr * HD + 8u * ((2u * nb + vc) ^ vsw(vr)) + vlo));
                if constexpr (SPLIT) v = finite_part4(v);
                oacc[nb] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, pop, oacc[nb] * alpha, 0, 0, 0);
            }
            if constexpr (SPLIT) {
                bool any = false; // token li, a quarter of its chunks
#pragma unroll
                for (int j = 0; j < LPP; ++j) {
                    const uint4_t w = *(const uint4_t*)(sv + li * HD + 8 * (LPP * lg + j));
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t x = w[e];
                        any |= (x & 0x7C00u) == 0x7C00u || (x & 0x7C000000u) == 0x7C000000u;
                    }
                }
                uint64_t todo = __ballot(any);
                todo = (todo | todo >> 16 | todo >> 32 | todo >> 48) & 0xFFFFu;
#pragma unroll 1
                for (; todo; todo &= todo - 1u) {
                    const int tok = __builtin_ctzll(todo);
                    float w = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float x = __shfl(pf[e], li + 16 * (tok >> 2));
                        if (e == (tok & 3)) w = x;
                    }
                    const bool see = p * 16u + (uint32_t)tok < rlim;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        const half4_t x = *(const half4_t*)(sv + tok * HD + 8 * ((2 * nb + (lg >> 1)) ^ (int)vsw((uint32_t)tok)) + 4 * (lg & 1));
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float f = (float)x[e];
                            if (see && !(fabsf(f) < INFINITY)) oacc[nb][e] = fmaf(w, f, oacc[nb][e]);
                        }
                    }
                }
            }
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
    }

    // x with its infinities and NaNs replaced by zeros.
    static __device__ __forceinline__ half4_t finite_part4(half4_t x) {
        uint2_t w = __builtin_bit_cast(uint2_t, x);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint32_t v = w[e];
            w[e] = ((v & 0x7C00u) == 0x7C00u ? 0u : v & 0xFFFFu) | ((v & 0x7C000000u) == 0x7C000000u ? 0u : v & 0xFFFF0000u);
        }
        return __builtin_bit_cast(half4_t, w);
    }

    // `row` of all rows is this lane's (clamped), row0 + i < row_end the work-group's.
    template <int RUNS>
    __device__ __forceinline__ void run(const PrefixArgs& a, const PageRun (&runs)[RUNS], uint32_t g, uint32_t row, uint32_t row0,
                                        uint32_t row_end, uint32_t slot, _Float16* lds, int lane, uint32_t wave) {
        const int li = lane & 15, lg = lane >> 4;
        const uint32_t head = g * a.gqa + row % a.gqa;
        const uint16_t* p = a.q + ((uint64_t)(row / a.gqa) * a.q_heads + head) * HD;
#pragma unroll
        for (int j = 0; j < KS; ++j) qop[j] = prefix_query(p + 32 * j + 8 * lg, a.q_and, a.q_xor);
        bad = false;
        pass<false>(a, runs, g, lds, lane, wave);
        // An inf or NaN among the sums under finite weights comes from the values, and may
        // have reached rows that do not see it (0 * inf): once more, split.
        float chk = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4; ++e) chk = fmaf(oacc[nb][e], 0.0f, chk);
        if (__any(chk != 0.0f && l_run * 0.0f == 0.0f)) pass<true>(a, runs, g, lds, lane, wave);
        if (__any(bad) && lane == 0) flag_error(a.err, kErrHotRef);
        // The waves' sums, joined as prefix_merge_kernel joins the parts'.
        float *so = (float*)lds, *sm = so + 4 * 16 * P, *sl = sm + 64; // [wave][row]
        __syncthreads(); // every page has been read
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) *(float4_t*)(so + (wave * 16u + (uint32_t)li) * P + 16 * nb + 4 * lg) = oacc[nb];
        if (lg == 0) {
            sm[wave * 16u + (uint32_t)li] = l_run != 0.0f ? m_run : -INFINITY;
            sl[wave * 16u + (uint32_t)li] = l_run;
        }
        __syncthreads();
        const uint32_t t = wave * 64u + (uint32_t)lane, i = t >> 4, d = 4u * (t & 15u); // row, dims d .. + 3 (and d + 64 .. at 128)
        if (row0 + i >= row_end) return;
        const float M = fmaxf(fmaxf(sm[i], sm[16 + i]), fmaxf(sm[32 + i], sm[48 + i]));
        float L = 0.0f;
        float4_t o[HD / 64];
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) o[h] = (float4_t)0.0f;
#pragma unroll
        for (uint32_t w = 0; w < 4; ++w) {
            const float l = sl[w * 16u + i], f = l != 0.0f ? fast_exp2(sm[w * 16u + i] - M) : 0.0f;
            L = fmaf(f, l, L);
            if (l != 0.0f) // also where f is 0: an inf or NaN among the sums stays
#pragma unroll
                for (int h = 0; h < HD / 64; ++h) {
                    const float4_t x = *(const float4_t*)(so + (w * 16u + i) * P + 64 * h + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[h][e] = fmaf(f, x[e], o[h][e]);
                }
        }
        const uint32_t r = row0 + i;
        if (a.splits == 0) { // the request in one part: its rows
            uint16_t* out = a.out + ((uint64_t)(r / a.gqa) * a.q_heads + g * a.gqa + r % a.gqa) * HD + d;
#pragma unroll
            for (int h = 0; h < HD / 64; ++h) {
                half4_t y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (_Float16)(L == 0.0f ? 0.0f : o[h][e] / L);
                *(half4_t*)(out + 64 * h) = y;
            }
            return;
        }
        const uint64_t at = ((uint64_t)g * a.splits + slot) * a.rows + r;
        if (d == 0) {
            a.part_m[at] = M;
            a.part_l[at] = L;
        }
        if (L == 0.0f) return; // nothing seen: the merge takes no value of it
#pragma unroll
        for (int h = 0; h < HD / 64; ++h) *(float4_t*)(a.part_o + at * HD + 64 * h + d) = o[h];
    }
};

// Many rows to the prefix: a work-group takes kPrefixRows rows of one kv head, of
// whatever sequences (row r: sequence and query r / G, head r % G), x one part of the
// prefix, so that its pages are read once for all of them; 4 waves of 32 rows, TOK
// tokens a step.  K and V of a step go from memory straight into LDS, TOK / 16 pages of
// any place in the pool; tokens of a bad ref (page 0 is read) score -inf.
//   S^T = K Q^T on v_mfma_f32_32x32x16_f16 (lane l: row l % 32, hf = l / 32):
//     A = K (token l % 32, dims 16 j + 8 hf ..), B = Q^T from registers; a lane ends
//     with 16 of 32 tokens, 8 (i / 4) + 4 hf + i % 4, of its row: the softmax is per
//     lane but for one exchange with lane l ^ 32, and
//   O^T += V^T P^T takes P from the same registers: k-index 8 hf + j is token 4 hf + j
//     (j < 4) or 8 + 4 hf + j - 4; A = V^T by transposing LDS reads.
// Staged rows are HD / 8 16-byte chunks, chunk c of K row r at c ^ (r % chunks), of V
// row r at c ^ 4 (r % 4) ^ (r / 4) % 4 (128 dims): no bank conflict at 128 dims.
// Measured, 96 sequences of 32 / 8 heads x 128 behind 32768 tokens, 51.5 GFLOP: 86 us
// alone, 600 TFLOP/s (81 with sums rescaled seldom, see below; then its loads alone took 60
// to 76 us, its products and softmax alone 58 to 70), so it is bound by both at once.  32 or 128
// tokens a step, 3 or 4 buffers, 256 rows of 8 waves, two of these work-groups a CU: each
// slower there or for 64 sequences behind 8192 tokens.
constexpr uint32_t kPrefixRows = 128;
// A row's sums are rescaled whenever its maximum grows: its largest weight so far is exactly
// 1, as in the decode kernel, and its bits do not depend on the rows beside it (their
// growth multiplies its sums by 1).  Error against 64 bits, this and the decode kernel's
// on the same tokens (f16 outputs alone 2.1e-4): random scores 2.4e-4, 2.5e-4 at 8192
// tokens, 2.6e-4, 2.7e-4 at 32768; rows where a late token takes most of the weight
// 2.1e-4 to 2.5e-4, no more than the decode kernel's; two such tokens in the two halves of one
// step 2.3e-4 to 2.5e-4, up to 6% above it (its groups are of 32 tokens).  Measured, us: 64
// sequences behind 8192 tokens 27.4, 96 behind 32768 and their own 118.  Not taken: rescaling only
// after a growth of 2^8, 26.7 and 115, but errors up to 33% above the decode kernel's (the
// largest weight rounded, not its part of the sum) and a row's bits by its neighbours'
// growth; a second f16 term for what is left of the weights of a step's first 32 tokens,
// 2.0e-4 to 2.4e-4 but 29.6 and 127, or of all of them, f16 outputs' own error but 34.1
// and 167.
constexpr int kPrefixThreads = 256;
constexpr int kPrefixTok = 64, kPrefixBufs = 5; // tokens a step, steps of K or of V in LDS: two work-groups fill a CU's
constexpr size_t prefix_lds_bytes(int HD) { return (size_t)kPrefixBufs * kPrefixTok * HD * 2; }

// One work-group's part: rows [row0, row0 + kPrefixRows) of `rows` x `tokens` tokens in
// pages (and, NODES, after them nodes [node0, nodes) of a tree, each row those that its mask names).
struct TilePart {
    const uint16_t* q;          // row r: q_step * (r / gqa) + HD * (r % gqa) halves on
    const uint16_t *k, *v;      // the pools at this kv head
    const uint32_t* table;      // refs of the part's pages
    uint64_t q_step, blocks;
    uint32_t rstride;           // halves from token to token of a page
    uint32_t gqa, rows, row0, tokens;
    uint32_t q_and, q_xor;
    float scale_log2;
    float *m, *l, *o;           // sums of row 0 (and the rows after it)
    uint32_t* err;
    // NODES
    const uint16_t *nk, *nv;    // node 0 at this kv head
    uint64_t nk_step, nv_step;  // halves from node to node
    const uint32_t* mask;       // [nodes][mask_words] or null: the nodes up to the row's own
    uint32_t mask_words, node0, nodes; // node0 a multiple of the step
    uint16_t* out;              // not null: the whole of what the rows see, normed and stored (as q, o_step)
    uint64_t o_step;
};

template <int HD, bool NODES = false>
struct PrefixTile {
    static constexpr int TOK = kPrefixTok, BUFS = kPrefixBufs, PAGES = TOK / 16, TB = TOK / 32;
    static constexpr int CH = HD / 8, KS = HD / 16, NB = HD / 32;
    static constexpr int LPT = TOK * CH / kPrefixThreads; // loads per thread, operand and step
    static constexpr uint32_t OP = TOK * HD;              // halves per staged operand
    static constexpr int NS = TB * KS, NV = 2 * TB * NB;  // MFMAs of a step's scores, of its output
    static_assert(prefix_lds_bytes(HD) >= pages_lds_bytes(HD), "the other parts' LDS");
    static_assert(BUFS == 5 && NS - 4 >= 2 * LPT, "this step's loads are out before v_there");

    static __device__ __forceinline__ uint32_t ksw(uint32_t row) { return row & (uint32_t)(CH - 1); }
    static __device__ __forceinline__ uint32_t vsw(uint32_t row) {
        return CH == 16 ? ((row & 3u) << 2) | ((row >> 2) & 3u) : ((row >> 1) & 1u) << 2;
    }
    static __device__ __forceinline__ void barrier() {
        __builtin_amdgcn_sched_barrier(0);
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_barrier();
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }

    static __device__ __forceinline__ void run(const TilePart& a, _Float16* lds) {
        int tid = threadIdx.x;
        if constexpr (NODES) __asm__ volatile("" : "+v"(tid)); // what is made of it is made for each part, not kept between: no spills
        const int lane = tid & 63, li = lane & 31, hf = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t t1 = a.tokens;
        const int paged = (int)((t1 + (uint32_t)TOK - 1u) / (uint32_t)TOK); // steps over pages, > 0 without NODES
        const int steps = paged + (NODES ? (int)((a.nodes - a.node0 + (uint32_t)TOK - 1u) / (uint32_t)TOK) : 0);
        const uint32_t wrow0 = a.row0 + 32u * (uint32_t)wave; // the wave's rows
        const uint32_t row = wrow0 + (uint32_t)li;
        const bool wave_rows = wrow0 < a.rows;

        half8_t qop[KS];
        {
            const uint32_t r = min(row, a.rows - 1u);
            const uint16_t* p = a.q + (uint64_t)(r / a.gqa) * a.q_step + (r % a.gqa) * (uint32_t)HD;
#pragma unroll
            for (int j = 0; j < KS; ++j) qop[j] = prefix_query(p + 16 * j + 8 * hf, a.q_and, a.q_xor);
        }

        // Staging: load j fills slots tid + 256 j of the operand (slot -> row, chunk); a wave's
        // slots of one load lie in one page, at the same place of it for every j.
        const uint32_t rstride = a.rstride, page_halves = kBlockTokens * rstride; // halves
        const uint32_t srow = ((uint32_t)tid / CH) & 15u, schunk = (uint32_t)tid % CH;
        const uint16_t* kfrom = a.k + srow * rstride + 8u * (schunk ^ ksw(srow));
        const uint16_t* vfrom = a.v + srow * rstride + 8u * (schunk ^ vsw(srow));
        // Rows past the part's last token load that token's (and count for nothing).
        const uint32_t last = paged ? (t1 - 1u) / kBlockTokens : 0u;
        const int back = ((int)min(srow, (t1 - 1u) % kBlockTokens) - (int)srow) * (int)rstride;
        // Refs of 64 pages, one in each lane, and which of them count: the run of the newest K
        // step, the one before it, and (refs alone) the next.
        uint32_t held, ref_cur, ref_old, ref_next;
        uint64_t ok_cur, ok_old;
        bool bad = false;
        auto refs_from = [&](uint32_t run) { return !NODES || paged ? a.table[min(64u * run + (uint32_t)lane, last)] & kRefMask : 0u; };
        auto take = [&](uint32_t run) {
            held = run;
            ref_old = ref_cur;
            ok_old = ok_cur;
            const bool ok = ref_next < a.blocks || (NODES && !paged);
            ref_cur = ok ? ref_next : 0u;
            ok_cur = __ballot(ok);
            bad |= !ok;
            ref_next = refs_from(run + 1u);
        };
        // Load j of a step of K or (`v`) V; INNER: the step is not the last over pages.
        auto load = [&](auto inner, bool v, uint32_t refs, int step, _Float16* dst, int j) {
            const uint32_t p = (uint32_t)(CH == 16 ? j : 2 * j + (wave >> 1)); // page: 16 rows a load, or 32
            const uint32_t b = (uint32_t)step * (uint32_t)PAGES + p, at = decltype(inner)::value ? b : min(b, last);
            const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)refs, (int)(at & 63u));
            const uint16_t* src = (v ? vfrom : kfrom) + (uint64_t)ref * page_halves;
            if constexpr (!decltype(inner)::value) src += b >= last ? back : 0;
            if constexpr (NODES && !decltype(inner)::value)
                if (step >= paged) { // uniform; rows past the last node load that one
                    const uint32_t node = min(a.node0 + (uint32_t)(step - paged) * (uint32_t)TOK + 16u * p + srow, a.nodes - 1u);
                    src = v ? a.nv + node * a.nv_step + 8u * (schunk ^ vsw(srow)) : a.nk + node * a.nk_step + 8u * (schunk ^ ksw(srow));
                }
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                             (__attribute__((address_space(3))) void*)(dst + ((uint32_t)wave * 512u + (uint32_t)(kPrefixThreads * 8 * j))), 16, 0, 0);
        };
        // The loads that step i issues, V of step i + 1 and K of step i + 3, into the buffers
        // vbuf and kbuf: 2 LPT, x < LPT of V.  ready(i) first.
        uint32_t vrefs;
        auto ready = [&](int i) {
            if (i + 3 < steps && (uint32_t)(i + 3) * (uint32_t)PAGES / 64u != held) take(held + 1u); // a step's pages lie in one run of 64
            vrefs = (uint32_t)(i + 1) * (uint32_t)PAGES / 64u == held ? ref_cur : ref_old;
        };
        auto load_pair = [&](auto inner, int x, int i, uint32_t vbuf, uint32_t kbuf) {
            constexpr bool INNER = decltype(inner)::value;
            if (x < LPT) {
                if (INNER || (i >= -1 && i + 1 < steps)) load(inner, true, vrefs, i + 1, lds + vbuf * OP, x);
            } else if (INNER || i + 3 < steps) {
                load(inner, false, ref_cur, i + 3, lds + kbuf * OP, x - LPT);
            }
        };

        // LDS offsets (halves) of this lane's operands in a staged step, of the first k-step
        // and dim block; the others lie at these with a chunk's bits turned over.
        uint32_t kat, va, vb;
        {
            const uint32_t i16 = (uint32_t)lane & 15u, ra = 4u * (uint32_t)hf + (i16 >> 2), rb = ra + 8u;
            const uint32_t c = (((uint32_t)lane >> 4) & 1u) * 2u + ((i16 & 3u) >> 1), lo = 4u * (i16 & 1u);
            kat = (uint32_t)li * HD + 8u * ((uint32_t)hf ^ ksw((uint32_t)li));
            va = ra * HD + 8u * (c ^ vsw(ra)) + lo;
            vb = rb * HD + 8u * (c ^ vsw(rb)) + lo;
        }
        // MFMA x of the scores: tokens 32 (x % TB) .., k-step x / TB; of the output: tokens
        // 32 (x / 2 NB) + 16 (x / NB % 2) .., dims 32 (x % NB) ..
        auto kfrag = [&](const _Float16* sk, int x) { return *(const half8_t*)(sk + (kat ^ (16u * (x / TB))) + (x % TB) * 32 * HD); };
        auto vfrag = [&](const _Float16* sv, int x) {
            const int nb = x % NB, ro = (32 * (x / (2 * NB)) + 16 * ((x / NB) % 2)) * HD;
            return __builtin_bit_cast(half8_t, __builtin_shufflevector(lds_read_tr16_waited(sv + (va ^ (32u * nb)) + ro),
                                                                       lds_read_tr16_waited(sv + (vb ^ (32u * nb)) + ro), 0, 1, 2, 3, 4, 5, 6, 7));
        };

        float m_run, l_run;
        float16_t oacc[NB];
        // One step: the weights of `sc` (this step's scores) and its output, and beside them the
        // next step's scores into `sn`: NS products of the scores, then NV of the output, the
        // weights worked out beside the first NS + NV / 2 of them, those of the first 32 tokens
        // done before their products.  Operands are read four products ahead, in fours: with
        // loads into LDS under way the compiler waits for every LDS read before it uses one, so
        // reads are issued right after such a wait.  SPLIT: as in PrefixPages.
        auto process = [&](auto split, int step, const _Float16* sk, const _Float16* sv, float16_t (&sc)[TB], float16_t (&sn)[TB], auto load_x, auto v_there) {
            constexpr bool SPLIT = decltype(split)::value;
            const uint32_t c0 = (uint32_t)step * (uint32_t)TOK, b0 = (uint32_t)step * (uint32_t)PAGES;
            const uint32_t ok4 = (uint32_t)((b0 / 64u == held ? ok_cur : ok_old) >> (b0 & 63u)) & ((1u << PAGES) - 1u);
            __asm__ volatile("" : "+v"(kat), "+v"(va), "+v"(vb)); // their other forms are made in each step, not kept: no spills
            half8_t fr[8];
            auto read = [&](int z) { fr[z % 8] = z < NS ? kfrag(sk, z) : vfrag(sv, z - NS); };
#pragma unroll
            for (int z = 0; z < 4; ++z) read(z);
            uint32_t sees[TB]; // of the step's nodes, the row's
            const bool at_nodes = NODES && step >= paged; // wave-uniform
            if (at_nodes) {
                const uint32_t n0 = a.node0 + (uint32_t)(step - paged) * (uint32_t)TOK, node = min(row, a.rows - 1u) / a.gqa;
                auto low = [](uint32_t n, uint32_t from) { return n <= from ? 0u : n - from >= 32u ? ~0u : (1u << (n - from)) - 1u; };
#pragma unroll
                for (int tb = 0; tb < TB; ++tb) {
                    const uint32_t from = n0 + 32u * tb;
                    sees[tb] = !a.mask ? low(node + 1u, from) : from / 32u < a.mask_words ? a.mask[(uint64_t)node * a.mask_words + from / 32u] : 0u;
                    sees[tb] &= low(a.nodes, from);
                    const uint32_t half = sees[tb] >> (4 * hf);
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (!(half & (1u << (8 * (i / 4) + i % 4)))) sc[tb][i] = -INFINITY;
                }
            } else if (c0 + (uint32_t)TOK > t1 || ok4 != (1u << PAGES) - 1u) { // wave-uniform
                int see = (int)(t1 - c0) - 4 * hf;
                __asm__ volatile("" : "+v"(see)); // compared with constants here, not as 32 values kept over the loop
#pragma unroll
                for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        if (32 * tb + 8 * (i / 4) + i % 4 >= see || !((ok4 >> (2 * tb + i / 8)) & 1u)) sc[tb][i] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int at = 0; at < 32; ++at) mx = fmaxf(mx, sc[at / 16][at % 16]);
            const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx), __builtin_bit_cast(uint32_t, mx), false, false);
            const uint32_t sw0 = sw[0], sw1 = sw[1]; // the row's two halves
            mx = fmaxf(__builtin_bit_cast(float, sw0), __builtin_bit_cast(float, sw1)) * a.scale_log2;
            if (__any(mx > m_run)) { // wave-uniform; a row whose maximum stays is multiplied by 1
                const float mnew = fmaxf(m_run, mx);
                const float alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m_run - mnew);
                m_run = mnew;
                l_run *= alpha;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) oacc[nb] *= alpha;
            }
            const float mref = m_run == -INFINITY ? 0.0f : m_run;
            half8_t pop[TB][2];
            float ps[2] = {0.0f, 0.0f};
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) sn[tb] = (float16_t)0.0f;
            constexpr int SLOTS = NS + NV / 2;
            static_assert(TB == 2 && NS * 32 / SLOTS >= 16 && NS % 4 == 0, "");
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int z = 0; z < NS + NV; ++z) {
                if (z < NS) {
                    sn[z % TB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fr[z % 8], qop[z / TB], sn[z % TB], 0, 0, 0);
                } else {
                    const int y = z - NS;
                    half8_t v = fr[z % 8];
                    if constexpr (SPLIT) v = finite_part(v);
                    oacc[y % NB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pop[y / (2 * NB)][(y / NB) % 2], oacc[y % NB], 0, 0, 0);
                }
                __builtin_amdgcn_sched_barrier(0);
                if (z == NS - 4) v_there();
                if (z % 4 == 0)
#pragma unroll
                    for (int r = z + 4; r < z + 8 && r < NS + NV; ++r) read(r);
                if (z < 2 * LPT) load_x(z);
                if (z < SLOTS)
#pragma unroll
                    for (int at = z * 32 / SLOTS; at < (z + 1) * 32 / SLOTS; ++at) {
                        const int tb = at / 16, i = at % 16;
                        const float p = fast_exp2(fmaf(sc[tb][i], a.scale_log2, -mref));
                        ps[at % 2] += p;
                        pop[tb][i / 8][i % 8] = (_Float16)p;
                        if constexpr (SPLIT) sc[tb][i] = p;
                    }
                __builtin_amdgcn_sched_barrier(0);
            }
            l_run += ps[0] + ps[1];
            if constexpr (SPLIT) {
                auto nonfinite = [&](uint32_t r, uint32_t c) -> bool { // slot c of V row r
                    const uint4_t w = *(const uint4_t*)(sv + r * HD + 8u * c);
                    bool any = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const uint32_t v = w[e];
                        any |= (v & 0x7C00u) == 0x7C00u || (v & 0x7C000000u) == 0x7C000000u;
                    }
                    return any;
                };
                bool any = false; // row `lane`, from another slot on in each lane (banks)
#pragma unroll 1
                for (uint32_t c = 0; c < (uint32_t)CH; ++c)
                    any |= lane < TOK && nonfinite((uint32_t)lane % (uint32_t)TOK, (c + (uint32_t)lane) % (uint32_t)CH);
#pragma unroll 1
                for (uint64_t todo = __ballot(any); todo; todo &= todo - 1u) {
                    const uint32_t at = (uint32_t)__builtin_ctzll(todo);
                    const uint32_t slots = (uint32_t)__ballot(lane < CH && nonfinite(at, (uint32_t)lane % (uint32_t)CH));
                    const bool counts = at_nodes || (c0 + at < t1 && ((ok4 >> (at / 16u)) & 1u));
                    const bool see = !at_nodes || ((sees[at / 32u % TB] >> (at % 32u)) & 1u);
                    float p = 0.0f; // token `at`'s weight: register (at / 8 % 4) 4 + at % 4 of the half at / 4 % 2
#pragma unroll
                    for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            if ((at & ~4u) == (uint32_t)(32 * tb + 8 * (i / 4) + i % 4)) p = sc[tb][i];
                    p = __shfl(p, li + 32 * (int)((at >> 2) & 1u));
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                        for (int i = 0; i < 16; i += 4) {
                            const uint32_t slot = (uint32_t)(4 * nb + i / 4) ^ vsw(at);
                            if (!((slots >> slot) & 1u) || !counts) continue; // uniform
                            const half4_t v = *(const half4_t*)(sv + at * HD + 8u * slot + 4 * hf);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float f = (float)v[e];
                                if (see && !(fabsf(f) < INFINITY)) oacc[nb][i + e] = fmaf(p, f, oacc[nb][i + e]);
                            }
                        }
                }
            }
        };

        // Waits until at most `n` of this wave's newest steps of V or K are in flight.
        auto wait = [](auto n) {
            constexpr uint32_t vm = (uint32_t)decltype(n)::value * (uint32_t)LPT;
            __builtin_amdgcn_sched_barrier(0);
            __builtin_amdgcn_s_waitcnt((short)((vm & 15u) | ((vm >> 4) << 14) | (7u << 4) | (15u << 8))); // vmcnt(vm)
        };
        // Steps of K and V share a ring of 5 buffers in the order of their loads: K 0, K 1,
        // V 0, K 2, V 1, K 3, ..  While step i is worked, K of i + 1 is read, then V of i, and V
        // of i + 1 and K of i + 3 are loaded into what every wave read in step i - 1: K is
        // loaded almost two steps before its use, V one and a half.
        auto pass = [&](auto split) {
            using I0 = std::integral_constant<int, 0>;
            using I2 = std::integral_constant<int, 2>;
            using I3 = std::integral_constant<int, 3>;
            m_run = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) oacc[nb] = (float16_t)0.0f;
            ref_cur = 0;
            ok_cur = 0;
            ref_next = refs_from(0);
            take(0);
            vrefs = ref_cur; // 4 steps lie in the first run
            float16_t s0[TB], s1[TB];
#pragma unroll
            for (int i = -3; i < 0; ++i)
#pragma unroll
                for (int x = 0; x < 2 * LPT; ++x) load_pair(std::false_type{}, x, i, 2u, (uint32_t)(i < -1 ? i + 3 : 3));
            if (steps >= 3) wait(I3{});
            else wait(I0{});
            barrier();
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) s0[tb] = (float16_t)0.0f;
            if (wave_rows)
#pragma unroll
                for (int x = 0; x < NS; ++x)
                    s0[x % TB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kfrag(lds, x), qop[x / TB], s0[x % TB], 0, 0, 0);
            uint32_t kb = 1, vb = 2; // buffers of K i + 1 and V i; V i + 1 takes kb + 3, K i + 3 vb + 3 (mod 5)
            auto ring = [](uint32_t b) { return b >= 5u ? b - 5u : b; };
            // INNER: the steps that this one loads are there, and K's is not the part's last.
            auto step = [&](auto inner, int i, float16_t (&sc)[TB], float16_t (&sn)[TB]) {
                const bool whole = decltype(inner)::value || i + 2 < steps; // what step i - 1 loaded is whole
                if (whole) wait(I2{});
                else wait(I0{});
                __builtin_amdgcn_s_waitcnt((short)0xC07F); // lgkmcnt(0): what this wave read of step i - 1 is there
                barrier();
                ready(i);
                const uint32_t vnext = ring(kb + 3u), knext = ring(vb + 3u);
                auto load_x = [&](int x) { load_pair(inner, x, i, vnext, knext); };
                auto v_there = [&] {
                    if (decltype(inner)::value || i + 3 < steps) wait(I3{}); // this step's loads are whole too
                    else wait(I0{});
                    barrier();
                };
                if (wave_rows) {
                    process(split, i, lds + kb * OP, lds + vb * OP, sc, sn, load_x, v_there);
                } else {
#pragma unroll
                    for (int x = 0; x < 2 * LPT; ++x) load_x(x);
                    v_there();
                }
                kb = ring(kb + 2u);
                vb = ring(vb + 2u);
            };
            int i = 0;
            if constexpr (!decltype(split)::value)
                for (; i + 5 < paged; i += 2) {
                    step(std::true_type{}, i, s0, s1);
                    step(std::true_type{}, i + 1, s1, s0);
                }
#pragma unroll 1
            for (; i < steps; i += 2) {
                step(std::false_type{}, i, s0, s1);
                if (i + 1 < steps) step(std::false_type{}, i + 1, s1, s0);
            }
            wait(I0{});
            barrier(); // every step has been read
        };
        pass(std::false_type{});
        // An inf or NaN among the sums under finite weights: it comes from the values, and a
        // weight that f16 rounds to 0 makes it NaN.  The work-group then takes its part again.
        float l = l_run + __shfl_xor(l_run, 32), chk = 0.0f;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; ++i) chk = fmaf(oacc[nb][i], 0.0f, chk);
        uint32_t* flags = (uint32_t*)lds;
        const bool redo = __any(wave_rows && row < a.rows && chk != 0.0f && l * 0.0f == 0.0f);
        if (lane == 0) flags[wave] = redo ? 1u : 0u;
        __syncthreads();
        const uint32_t again = flags[0] | flags[1] | flags[2] | flags[3];
        __syncthreads();
        if (again) { // the same in every wave
            pass(std::true_type{});
            l = l_run + __shfl_xor(l_run, 32);
        }
        if (wave == 0 && __any(bad) && lane == 0) flag_error(a.err, kErrHotRef);
        uint32_t ro = row;
        __asm__ volatile("" : "+v"(ro)); // its addresses are made here, not kept over the loops
        if (ro >= a.rows) return;
        if constexpr (NODES)
            if (a.out) {
                const float inv = l == 0.0f ? 0.0f : 1.0f / l;
                uint16_t* po = a.out + (uint64_t)(ro / a.gqa) * a.o_step + (ro % a.gqa) * (uint32_t)HD;
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        half4_t y;
#pragma unroll
                        for (int e = 0; e < 4; ++e) y[e] = (_Float16)(l == 0.0f ? 0.0f : oacc[nb][i + e] * inv);
                        *(half4_t*)(po + 32 * nb + 2 * i + 4 * hf) = y;
                    }
                return;
            }
        if (hf == 0) {
            a.m[ro] = m_run;
            a.l[ro] = l;
        }
        if (l == 0.0f) return;
        // Past the L2, whose dirty lines would be written when the kernel ends: 64 sequences
        // behind 8192 tokens 28.1 us, through it 29.1; whole rows by way of LDS no better.
        float* po = a.o + (uint64_t)ro * HD;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                __builtin_nontemporal_store((float4_t){oacc[nb][i], oacc[nb][i + 1], oacc[nb][i + 2], oacc[nb][i + 3]},
                                            (float4_t*)(po + 32 * nb + 2 * i + 4 * hf));
    }
};

// Work-groups 0 .. prefix_wgs - 1 take the prefix in PrefixTile's parts (TILES), the others
// a unit's kv head each: 16 rows x a part of one table, or (splits == 0: small requests)
// all that they see, the prefix and their own pages, without a merge.
// Work-group b runs on XCD b % 8: the row tiles of one part of the prefix follow one
// another on one XCD, so its pages come from memory once, and so do the heads of a unit.
template <int HD, bool TILES>
__global__ __launch_bounds__(kPrefixThreads) __attribute__((amdgpu_waves_per_eu(2))) void prefix_kernel(PrefixArgs a) {
    extern __shared__ __attribute__((aligned(16))) _Float16 prefix_lds[];
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); }; // divisions run on the vector ALUs
    const int lane = threadIdx.x & 63;
    const uint32_t wave = uniform(threadIdx.x >> 6), xcd = blockIdx.x & 7u;
    uint32_t j = blockIdx.x >> 3;
    if constexpr (TILES) {
        if (blockIdx.x < a.prefix_wgs) { // a multiple of 8
            const uint32_t parts = a.kv_heads * a.prefix_splits, each = (parts + 7u) >> 3, i = uniform(j / a.prefix_tiles);
            const uint32_t part = xcd * each + i;
            if (part >= parts) return;
            const uint32_t s = uniform(part / a.kv_heads), g = part - s * a.kv_heads;
            const uint32_t t0 = s * a.prefix_span; // below prefix_tokens
            const uint64_t at = ((uint64_t)g * a.splits + s) * a.rows;
            TilePart w{};
            w.q = a.q + (uint64_t)g * a.gqa * HD;
            w.k = a.k + (uint64_t)g * HD;
            w.v = a.v + (uint64_t)g * HD;
            w.table = a.prefix_refs + t0 / kBlockTokens;
            w.q_step = (uint64_t)a.q_heads * HD;
            w.blocks = a.blocks;
            w.rstride = a.kv_heads * (uint32_t)HD;
            w.gqa = a.gqa;
            w.rows = a.rows;
            w.row0 = (j - i * a.prefix_tiles) * kPrefixRows;
            w.tokens = min(a.prefix_span, a.prefix_tokens - t0);
            w.q_and = a.q_and;
            w.q_xor = a.q_xor;
            w.scale_log2 = a.scale_log2;
            w.m = a.part_m + at;
            w.l = a.part_l + at;
            w.o = a.part_o + at * HD;
            w.err = a.err;
            PrefixTile<HD>::run(w, prefix_lds);
            return;
        }
        j -= a.prefix_wgs >> 3;
    }
    const uint32_t eight = uniform(j / a.kv_heads), g = j - eight * a.kv_heads, li = (uint32_t)lane & 15u;
    uint32_t unit = eight * 8u + xcd;
    PrefixPages<HD> w;
    if constexpr (!TILES) {
        if (unit < a.prefix_units) {
            const uint32_t s = uniform(unit / a.prefix_tiles), row0 = (unit - s * a.prefix_tiles) * 16u;
            const uint32_t t0 = s * a.prefix_span, t1 = min(t0 + a.prefix_span, a.prefix_tokens);
            const PageRun runs[1] = {{a.prefix_refs, t0 / 16u, (t1 + 15u) / 16u, a.prefix_tokens, a.prefix_tokens}};
            w.run(a, runs, g, min(row0 + li, a.rows - 1u), row0, a.rows, s, prefix_lds, lane, wave);
            return;
        }
        unit -= a.prefix_units;
    }
    if (unit >= a.own_units) return;
    const uint32_t s = uniform(unit / (a.batch * a.own_tiles)), bt = unit - s * a.batch * a.own_tiles, b = uniform(bt / a.own_tiles);
    const uint32_t r0 = (bt - b * a.own_tiles) * 16u, rc = min(r0 + li, a.own_rows - 1u);
    uint32_t n = a.seq_own ? a.seq_own[b] : a.own_max;
    if (n > a.own_max) {
        n = a.own_max;
        if (threadIdx.x == 0) flag_error(a.err, aw_engine_internal::kErrSeqBit);
    }
    n = uniform(n);
    const uint32_t i = rc / a.gqa; // query of the row: it sees n - queries + 1 + i tokens
    const uint32_t lim = a.causal ? (n + 1u + i > a.queries ? n + 1u + i - a.queries : 0u) : n;
    const uint32_t* table = a.refs + (uint64_t)b * a.refs_stride;
    const uint32_t base = b * a.own_rows;
    if constexpr (!TILES) {
        if (a.splits == 0) {
            const PageRun runs[2] = {{a.prefix_refs, 0, (a.prefix_tokens + 15u) / 16u, a.prefix_tokens, a.prefix_tokens}, {table, 0, (n + 15u) / 16u, n, lim}};
            w.run(a, runs, g, base + rc, base + r0, base + a.own_rows, 0, prefix_lds, lane, wave);
            return;
        }
    }
    const uint32_t t0 = s * a.own_span, p0 = t0 / 16u; // a sequence may end before this part
    const PageRun runs[1] = {{table, p0, t0 < n ? (min(t0 + a.own_span, n) + 15u) / 16u : p0, n, lim}};
    w.run(a, runs, g, base + rc, base + r0, base + a.own_rows, a.prefix_splits + s, prefix_lds, lane, wave);
}

// Joins a row's parts: the largest maximum, each part's sums times 2^(its maximum -
// that), added in an order of their own; zeros where no part saw a token.  An inf or NaN
// in a part's sum stays in the result, as NaN where the part's factor is 0.  W waves a
// row (4 where rows are few, their sums added in the order of the waves); a row of a part
// is HD / 4 lanes' float4, U loads in flight before the parts' factors are known.
template <int HD, int U, int W>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixArgs a) {
    constexpr int LP = HD / 4, PG = 64 / LP; // lanes of a part's row, parts of one load
    __shared__ float4_t s_sum[W > 1 ? W : 1][LP];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6, w = W > 1 ? wave : 0u;
    const uint64_t id = W > 1 ? (uint64_t)blockIdx.x : (uint64_t)blockIdx.x * 4u + wave;
    if (id >= (uint64_t)a.kv_heads * a.rows) return; // W > 1: the grid is exact
    const uint32_t g = (uint32_t)(id / a.rows), r = (uint32_t)(id % a.rows), S = a.splits;
    const uint64_t at = (uint64_t)g * S * a.rows + r;
    const uint32_t sub = lane / LP, d = 4u * (lane % LP);
    const float* po = a.part_o + at * HD + d;
    auto part = [&](uint32_t p0, int j) { return p0 + (uint32_t)(j * W * PG) + w * PG + sub; };
    float4_t v[U];
    auto load = [&](uint32_t p0) {
#pragma unroll
        for (int j = 0; j < U; ++j) v[j] = *(const float4_t*)(po + (uint64_t)min(part(p0, j), S - 1u) * a.rows * HD);
    };
    const uint64_t mine = at + (uint64_t)min(lane, S - 1u) * a.rows;
    float l = a.part_l[mine], m = a.part_m[mine];
    load(0);
    if (lane >= S) l = 0.0f;
    if (l == 0.0f) m = -INFINITY;
    const uint64_t held = __ballot(l != 0.0f); // a part that saw nothing holds no sums
    const float M = wave_max(m);
    const float f = l != 0.0f ? fast_exp2(m - M) : 0.0f;
    const float L = wave_sum(f * l);
    float4_t acc = (float4_t)0.0f;
    for (uint32_t p0 = 0; p0 < S; p0 += (uint32_t)(U * W * PG)) {
        if (p0) load(p0);
#pragma unroll
        for (int j = 0; j < U; ++j) {
            const uint32_t p = part(p0, j);
            const float fp = __shfl(f, (int)min(p, S - 1u));
            if (p < S && ((held >> p) & 1u))
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[e] = fmaf(fp, v[j][e], acc[e]);
        }
    }
#pragma unroll
    for (int o = LP; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    if constexpr (W > 1) {
        if (sub == 0) s_sum[wave][lane] = acc;
        __syncthreads();
        if (wave != 0) return;
        acc = s_sum[0][lane % LP];
#pragma unroll
        for (int i = 1; i < W; ++i) acc += s_sum[i][lane % LP];
    }
    if (sub != 0) return;
    half4_t h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (_Float16)(L == 0.0f ? 0.0f : acc[e] / L);
    *(half4_t*)(a.out + ((uint64_t)(r / a.gqa) * a.q_heads + g * a.gqa + r % a.gqa) * HD + d) = h;
}

} // namespace aw
