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
    float *part_m, *part_l;     // [2 work_groups][rows of a unit]
    float* part_o;              // [2 work_groups][rows of a unit][HD]
    uint32_t* cuts;             // [work_groups][kCutWords]
    uint32_t* err;
    uint64_t q_stride, k_stride, v_stride, out_stride, blocks;
    uint32_t batch, tokens, q_heads, kv_heads, gqa, hot_count, refs_stride, mask_words;
    uint32_t work_groups;       // a multiple of 8
    uint32_t q_and, q_xor;
    float scale_log2;           // > 0
};

// A sequence: its rows, its tokens in pages.
struct TreeSeq {
    uint32_t first, nodes, held;
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
    return s;
}

// ---- 16 NR query rows of a kv head: a work-group's waves take the pages (then the nodes, 16
// at a time) in turn, each on its own until their sums meet in LDS.  Products, layouts and
// the softmax are PrefixPages' (weights are f16 operands of the second product, their sums
// fp32: 2.5 to 2.8e-4 of the outputs against 64 bits, where the f16 store alone has
// 2.1e-4; operands of more bits would double those products); K and V pages are loaded one and a
// half to two pages ahead.
constexpr int kTreeBufs = 5; // pages of K or of V in LDS, a wave
constexpr size_t tree_pages_lds(int HD, int NW, int NR) {
    const size_t ring = (size_t)NW * kTreeBufs * 16 * HD * 2, sums = (size_t)NW * 16 * NR * (HD + 4) * 4 + NW * 16 * NR * 2 * 4;
    return ring > sums ? ring : sums;
}

// What the 16 NR rows of a work-group share: rows [row0, row_end), row r at q + q_step * (r / gqa) + HD * (r % gqa).
struct TreePart {
    const uint16_t *q, *k, *v;  // the pools at this kv head
    uint64_t q_step, blocks;
    uint32_t rstride;           // halves from token to token of a page
    uint32_t gqa, row0, row_end;
    uint32_t q_and, q_xor;
    float scale_log2;
    uint16_t* out;              // not null: all that the rows see, normed and stored (as q, o_step)
    uint64_t o_step;
    float *m, *l, *o;           // else sums of row 0 (and the rows after it)
    uint32_t* err;
    // the second run: a tree's nodes
    const uint16_t *nk, *nv;    // node 0 at this kv head
    uint64_t nk_step, nv_step;
    const uint32_t* mask;       // [nodes][mask_words] or null: the nodes up to the row's own
    uint32_t mask_words;
};

// NR: blocks of 16 rows that a wave's pages serve.
template <int HD, int NW, int NR>
struct TreePages {
    static constexpr int CH = HD / 8, KS = HD / 32, NB = HD / 16, P = HD + 4;
    static constexpr int LPP = CH / 4;                     // loads of a wave for a page of K (or V)
    static constexpr uint32_t OP = 16 * HD;                // halves of a staged page operand
    half8_t qop[NR][KS];
    float m_run[NR], l_run[NR];
    float4_t oacc[NR][NB];
    bool bad;

    static __device__ __forceinline__ uint32_t ksw(uint32_t row) { return row & (uint32_t)(CH - 1); }
    static __device__ __forceinline__ uint32_t vsw(uint32_t row) {
        return CH == 16 ? ((row & 3u) << 2) | ((row >> 2) & 3u) : ((row >> 1) & 1u) << 2;
    }
    // The largest of a row's four lanes (li, li + 16, li + 32, li + 48), in each of them.
    static __device__ __forceinline__ float row_max(float x) {
        const uint32_t u = __builtin_bit_cast(uint32_t, x);
        const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        const uint32_t h0 = h[0], h1 = h[1];
        const uint32_t y = __builtin_bit_cast(uint32_t, fmaxf(__builtin_bit_cast(float, h0), __builtin_bit_cast(float, h1)));
        const auto q = __builtin_amdgcn_permlane16_swap(y, y, false, false);
        const uint32_t q0 = q[0], q1 = q[1];
        return fmaxf(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
    }

    // This wave's pages of the runs.  SPLIT: the products take the values' finite part;
    // tokens whose values hold an inf or NaN are then added one by one, in fp32, to the
    // rows that see them.
    template <bool SPLIT>
    __device__ __forceinline__ void pass(const TreePart& a, const PageRun (&runs)[2], const uint32_t (&row)[NR], _Float16* lds, int lane, uint32_t wave) {
        const int li = lane & 15, lg = lane >> 4;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            m_run[r] = -INFINITY;
            l_run[r] = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) oacc[r][nb] = (float4_t)0.0f;
        }
        const uint32_t n0 = runs[0].p1 - runs[0].p0, n = n0 + (runs[1].p1 - runs[1].p0);
        if (wave >= n) return; // wave-uniform
        const uint32_t mine = (n - wave + NW - 1u) / NW; // pages wave, wave + NW, ..
        // Page i of this wave: its place in its run, and whether that is the second.
        auto place = [&](uint32_t i, uint32_t& p) {
            p = wave + (uint32_t)NW * i;
            const bool second = p >= n0;
            p = second ? runs[1].p0 + (p - n0) : runs[0].p0 + p;
            return second;
        };
        // Refs of this wave's pages, 64 at a time, one in each lane, and of the next 64.
        auto refs_from = [&](uint32_t from) {
            uint32_t p;
            const uint32_t i = min(from + (uint32_t)lane, mine - 1u), q = wave + (uint32_t)NW * i;
            const bool second = q >= n0;
            p = second ? runs[1].p0 + (q - n0) : runs[0].p0 + q;
            return second ? 0u : runs[0].table[p] & kRefMask;
        };
        uint32_t held = 0, ref_cur = 0, ref_next = refs_from(0);
        uint64_t ok_cur = 0, ok_old = 0;
        auto take = [&] {
            const bool ok = ref_next < a.blocks || n0 == 0u; // nodes alone: there may be no pool
            ref_cur = ok ? ref_next : 0u;
            ok_old = ok_cur;
            ok_cur = __ballot(ok);
            bad |= !ok;
        };
        take();
        ref_next = refs_from(64u);
        // Staging: load j of a page fills slots lane + 64 j (slot -> row, chunk).  Pages of K and
        // V share the ring in the order of their use, K 0, V 0, K 1, ..: operand x in buffer x % 5.
        const uint32_t rstride = a.rstride;
        _Float16* ring = lds + wave * (uint32_t)kTreeBufs * OP;
        uint32_t k_at[LPP], v_at[LPP]; // bytes of a page to this lane's pieces: rows of at most 2^16 values
#pragma unroll
        for (int j = 0; j < LPP; ++j) {
            const uint32_t slot = (uint32_t)(lane + 64 * j), row = slot / CH, c = slot % CH;
            k_at[j] = 2u * (row * rstride + 8u * (c ^ ksw(row)));
            v_at[j] = 2u * (row * rstride + 8u * (c ^ vsw(row)));
        }
        auto load = [&](uint32_t i, bool v, uint32_t buf) {
            if (!v && i / 64u != held) {
                held = i / 64u;
                take();
                ref_next = refs_from((held + 1u) * 64u);
            }
            uint32_t p;
            const bool second = place(i, p);
            const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)ref_cur, (int)(i & 63u));
            const uint32_t left = (second ? runs[1].end : runs[0].end) - p * 16u;
            const uint16_t* from = (v ? a.v : a.k) + (uint64_t)ref * (16u * rstride);
            _Float16* dst = ring + buf * OP;
            if (left >= 16u && !second) { // uniform: a whole page
#pragma unroll
                for (int j = 0; j < LPP; ++j) {
                    const uint16_t* src = (const uint16_t*)((const char*)from + (v ? v_at[j] : k_at[j]));
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                                     (__attribute__((address_space(3))) void*)(dst + 512u * j), 16, 0, 0);
                }
                return;
            }
            uint64_t step = rstride;
            if (second) {
                step = v ? a.nv_step : a.nk_step;
                from = (v ? a.nv : a.nk) + (uint64_t)(p * 16u) * step;
            }
#pragma unroll
            for (int j = 0; j < LPP; ++j) { // rows past the end load the last one (and count for nothing)
                const uint32_t slot = (uint32_t)(lane + 64 * j), row = slot / CH, c = slot % CH;
                const uint16_t* src = from + min(row, min(left, 16u) - 1u) * step + 8u * (c ^ (v ? vsw(row) : ksw(row)));
                __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                                 (__attribute__((address_space(3))) void*)(dst + 512u * j), 16, 0, 0);
            }
        };
        // Waits until at most the newest four operands are in flight, or (`last`: fewer follow) none.
        auto wait = [](bool last) {
            constexpr uint32_t vm = 4u * (uint32_t)LPP;
            __builtin_amdgcn_sched_barrier(0);
            if (last) __builtin_amdgcn_s_waitcnt((short)((7u << 4) | (15u << 8)));
            else __builtin_amdgcn_s_waitcnt((short)((vm & 15u) | ((vm >> 4) << 14) | (7u << 4) | (15u << 8))); // vmcnt(vm)
            __asm__ volatile("" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
        auto read_done = [] { // what this wave read of LDS is there: its buffer may be filled
            __builtin_amdgcn_sched_barrier(0);
            __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            __builtin_amdgcn_sched_barrier(0);
        };
#pragma unroll
        for (uint32_t x = 0; x < 5u; ++x)
            if (x / 2u < mine) load(x / 2u, x & 1u, x);
        uint32_t kb = 0; // buffer of K i; V i lies in the next
        for (uint32_t i = 0; i < mine; ++i) {
            const uint32_t vb = kb == 4u ? 0u : kb + 1u;
            uint32_t p;
            const bool second = place(i, p);
            wait(i + 2u >= mine); // K i
            const _Float16 *sk = ring + kb * OP, *sv = ring + vb * OP;
            float4_t sacc[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) sacc[r] = (float4_t)0.0f;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                const half8_t k = *(const half8_t*)(sk + li * HD + 8 * ((4 * j + lg) ^ (int)ksw((uint32_t)li)));
#pragma unroll
                for (int r = 0; r < NR; ++r) sacc[r] = mfma16x16x32(k, qop[r][j], sacc[r]);
            }
            read_done();
            if (i + 2u < mine) load(i + 2u, true, kb); // V i + 2 where K i was
            const bool ok = ((i / 64u == held ? ok_cur : ok_old) >> (i & 63u)) & 1u;
            uint32_t sees[NR]; // of the page, the row's
            float pf[NR][4];
            half4_t pop[NR];
#pragma unroll
            for (int r = 0; r < NR; ++r) {
                const uint32_t end = second ? runs[1].end : runs[0].end;
                uint32_t lim = second ? runs[1].lim : runs[0].lim;
                if (second && !a.mask) lim = row[r] / a.gqa + 1u;
                const uint32_t rlim = ok ? min(lim, end) : 0u;
                sees[r] = rlim <= p * 16u ? 0u : rlim - p * 16u >= 16u ? 0xFFFFu : (1u << (rlim - p * 16u)) - 1u;
                if (second && a.mask)
                    sees[r] &= p / 2u < a.mask_words ? a.mask[(uint64_t)(row[r] / a.gqa) * a.mask_words + p / 2u] >> (16u * (p & 1u)) : 0u;
                float mx = -INFINITY;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pf[r][e] = (sees[r] >> (4 * lg)) & (1u << e) ? sacc[r][e] * a.scale_log2 : -INFINITY;
                    mx = fmaxf(mx, pf[r][e]);
                }
                mx = row_max(mx);
                if (__any(mx > m_run[r])) { // wave-uniform; a row whose maximum stays is multiplied by 1
                    const float mnew = fmaxf(m_run[r], mx), alpha = mnew == -INFINITY ? 1.0f : fast_exp2(m_run[r] - mnew);
                    m_run[r] = mnew;
                    l_run[r] *= alpha;
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) oacc[r][nb] *= alpha;
                }
                const float mref = m_run[r] == -INFINITY ? 0.0f : m_run[r];
                float psum = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    pf[r][e] = fast_exp2(pf[r][e] - mref);
                    psum += pf[r][e];
                    pop[r][e] = (_Float16)pf[r][e];
                }
                l_run[r] += psum;
            }
            wait(i + 2u >= mine); // V i
            const uint32_t vr = 4u * (uint32_t)lg + ((uint32_t)li >> 2), vc = ((uint32_t)li & 3u) >> 1, vlo = 4u * ((uint32_t)li & 1u);
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                half4_t v = __builtin_bit_cast(half4_t, lds_read_tr16_waited(sv + vr * HD + 8u * ((2u * nb + vc) ^ vsw(vr)) + vlo));
                if constexpr (SPLIT) v = finite_part4(v);
#pragma unroll
                for (int r = 0; r < NR; ++r) oacc[r][nb] = __builtin_amdgcn_mfma_f32_16x16x16f16(v, pop[r], oacc[r][nb], 0, 0, 0);
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
#pragma unroll
                    for (int r = 0; r < NR; ++r) {
                        float w = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float x = __shfl(pf[r][e], li + 16 * (tok >> 2));
                            if (e == (tok & 3)) w = x;
                        }
                        const bool see = (sees[r] >> tok) & 1u;
#pragma unroll
                        for (int nb = 0; nb < NB; ++nb) {
                            const half4_t x = *(const half4_t*)(sv + tok * HD + 8 * ((2 * nb + (lg >> 1)) ^ (int)vsw((uint32_t)tok)) + 4 * (lg & 1));
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float f = (float)x[e];
                                if (see && !(fabsf(f) < INFINITY)) oacc[r][nb][e] = fmaf(w, f, oacc[r][nb][e]);
                            }
                        }
                    }
                }
            }
            read_done();
            if (i + 3u < mine) load(i + 3u, false, vb); // K i + 3 where V i was
            kb = kb >= 3u ? kb - 3u : kb + 2u;
        }
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            l_run[r] += __shfl_xor(l_run[r], 16);
            l_run[r] += __shfl_xor(l_run[r], 32);
        }
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

    __device__ __forceinline__ void run(const TreePart& a, const PageRun (&runs)[2], _Float16* lds, int lane, uint32_t wave) {
        __asm__ volatile("" : "+v"(lane)); // what is made of it is made for each part, not kept between
        constexpr uint32_t R = 16u * NR, TR = 256u / R, E = HD / (4 * TR); // rows, threads of a row in the join, float4s of each
        const int li = lane & 15, lg = lane >> 4;
        uint32_t row[NR]; // this lane's
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            row[r] = min(a.row0 + 16u * r + (uint32_t)li, a.row_end - 1u);
            const uint16_t* p = a.q + (uint64_t)(row[r] / a.gqa) * a.q_step + (row[r] % a.gqa) * (uint32_t)HD;
#pragma unroll
            for (int j = 0; j < KS; ++j) qop[r][j] = prefix_query(p + 32 * j + 8 * lg, a.q_and, a.q_xor);
        }
        bad = false;
        pass<false>(a, runs, row, lds, lane, wave);
        // An inf or NaN among the sums under finite weights comes from the values, and may
        // have reached rows that do not see it (0 * inf): once more, split.
        bool again = false;
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            float chk = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) chk = fmaf(oacc[r][nb][e], 0.0f, chk);
            again |= chk != 0.0f && l_run[r] * 0.0f == 0.0f;
        }
        if (__any(again)) pass<true>(a, runs, row, lds, lane, wave);
        if (__any(bad) && lane == 0) flag_error(a.err, kErrHotRef);
        // The waves' sums, joined as prefix_merge_kernel joins the parts'.
        float *so = (float*)lds, *sm = so + NW * R * P, *sl = sm + NW * R; // [wave][row]
        __syncthreads(); // every page has been read
#pragma unroll
        for (int r = 0; r < NR; ++r) {
            const uint32_t at = wave * R + 16u * r + (uint32_t)li;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) *(float4_t*)(so + at * P + 16 * nb + 4 * lg) = oacc[r][nb];
            if (lg == 0) {
                sm[at] = l_run[r] != 0.0f ? m_run[r] : -INFINITY;
                sl[at] = l_run[r];
            }
        }
        __syncthreads();
        const uint32_t t = wave * 64u + (uint32_t)lane, i = t / TR, d = 4u * (t % TR); // row, dims d .. + 3 (and 4 TR h further)
        if (t >= 256u || a.row0 + i >= a.row_end) return;
        float M = sm[i];
#pragma unroll
        for (uint32_t w = 1; w < NW; ++w) M = fmaxf(M, sm[w * R + i]);
        float L = 0.0f;
        float4_t o[E];
#pragma unroll
        for (uint32_t h = 0; h < E; ++h) o[h] = (float4_t)0.0f;
#pragma unroll
        for (uint32_t w = 0; w < NW; ++w) {
            const float l = sl[w * R + i], f = l != 0.0f ? fast_exp2(sm[w * R + i] - M) : 0.0f;
            L = fmaf(f, l, L);
            if (l != 0.0f) // also where f is 0: an inf or NaN among the sums stays
#pragma unroll
                for (uint32_t h = 0; h < E; ++h) {
                    const float4_t x = *(const float4_t*)(so + (w * R + i) * P + 4 * TR * h + d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[h][e] = fmaf(f, x[e], o[h][e]);
                }
        }
        const uint32_t r = a.row0 + i;
        if (a.out) { // the whole of what the rows see
            uint16_t* out = a.out + (uint64_t)(r / a.gqa) * a.o_step + (r % a.gqa) * (uint32_t)HD + d;
#pragma unroll
            for (uint32_t h = 0; h < E; ++h) {
                half4_t y;
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = (_Float16)(L == 0.0f ? 0.0f : o[h][e] / L);
                *(half4_t*)(out + 4 * TR * h) = y;
            }
            return;
        }
        if (d == 0) {
            a.m[r] = M;
            a.l[r] = L;
        }
        if (L == 0.0f) return; // nothing seen: the merge takes no value of it
#pragma unroll
        for (uint32_t h = 0; h < E; ++h) *(float4_t*)(a.o + (uint64_t)r * HD + 4 * TR * h + d) = o[h];
    }
};

// The work of a sequence, in one of two ways: units of kPrefixRows query rows of a kv head
// (PrefixTile) or of 16 NR rows (TreePages); a step is 64 tokens of a unit, first those in
// pages, then the nodes (TreePages: the nodes' first page may share a step with the last tokens').
constexpr uint32_t tree_rows(int NR) { return NR ? 16u * NR : kPrefixRows; } // of a unit; NR 0: PrefixTile
template <int NR>
struct TreeWork {
    uint32_t tiles, steps; // units of a kv head, steps of a unit
    __device__ TreeWork(const TreeArgs& a, const TreeSeq& s) {
        tiles = (s.nodes * a.gqa + tree_rows(NR) - 1u) / tree_rows(NR);
        steps = NR ? ((s.held + 15u) / 16u + (s.nodes + 15u) / 16u + 3u) / 4u : (s.held + 63u) / 64u + (s.nodes + 63u) / 64u;
    }
    __device__ uint32_t all(uint32_t kv_heads) const { return kv_heads * tiles * steps; }
};
constexpr uint64_t kTreeSteps = 4294960000; // of a request: below 2^32 also when rounded up to shares of all work-groups

constexpr size_t tree_lds(int HD, int NR) { return NR ? tree_pages_lds(HD, 4, NR) : prefix_lds_bytes(HD); }

// What a merge needs of a unit that is cut: its parts, its rows and where they go.
constexpr uint32_t kCutWords = 5; // parts (0: no unit begins and is cut here), rows, row0, first, kv head

// Sums over the lanes up to this one.
__device__ inline uint32_t lanes_scan(uint32_t x) {
#define AW_DPP_SCAN(ctrl, rmask) x += (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, ctrl, rmask, 0xF, false)
    AW_DPP_SCAN(0x111, 0xF); // row_shr:1
    AW_DPP_SCAN(0x112, 0xF); // row_shr:2
    AW_DPP_SCAN(0x114, 0xF); // row_shr:4
    AW_DPP_SCAN(0x118, 0xF); // row_shr:8
    AW_DPP_SCAN(0x142, 0xA); // row_bcast:15 into rows 1 and 3
    AW_DPP_SCAN(0x143, 0xC); // row_bcast:31 into rows 2 and 3
#undef AW_DPP_SCAN
    return x;
}

// The steps of all units, laid end to end (sequence, kv head, rows, tokens), are shared out
// equally: work-group w takes those from w / work_groups of them on, so lengths may differ as
// they like.  A unit that lies in one work-group is normed and stored; of one that is cut
// each part's sums go to the workspace, at most two of a work-group: slot 2 w + 1 for the
// unit that begins here and is cut, 2 w for one that began before.
// Bound: with few rows HBM (64 sequences x 8 nodes x 32 / 8 heads x 128 behind 4099 tokens, 32-row
// units: 175 us, 4.65 TB/s, and the merge), with many a wave's chain of products, softmax, products (16 x
// 64 nodes behind 8192, 128-row units: 127 us, 370 TFLOP/s, where 24 tiles a kv head hold
// 2104 rows, sequences of two tiles read K and V twice, 549 MB for 403, and the steps that test each
// load, the last ones of each piece and the nodes', are 19 % of all).  Two work-groups a CU, whose
// chains overlap: one takes 10 to 20 % longer.  Nothing may spill in the steps: a
// reload waits for all loads in flight, those into LDS too (227 for 193 us, 173 for 142).
template <int HD, int NR>
__global__ __launch_bounds__(kPrefixThreads) __attribute__((amdgpu_waves_per_eu(2))) void tree_kernel(TreeArgs a) {
    constexpr uint32_t kRows = tree_rows(NR);
    extern __shared__ __attribute__((aligned(16))) _Float16 prefix_lds[];
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = uniform(tid >> 6);
    // Work-group b runs on XCD b % 8: neighbours in the line, which read the same pages for
    // several tiles of rows, run on one XCD.
    const uint32_t w = (blockIdx.x & 7u) * (a.work_groups >> 3) + (blockIdx.x >> 3);
    uint32_t* s_sum = (uint32_t*)prefix_lds; // [4] sums of waves, [5] the sequence found, [4] sums of waves' upper parts
    // All steps; sequence tid of each 256.
    TreeSeq s{};
    // Counted exactly, in two parts: offsets that descend give rows to several sequences, or one has far more nodes than its
    // mask names; steps that pass 32 bits by that (both are reported) are not taken, and no sum below wraps.
    uint64_t mine = 0;
    for (uint32_t b = tid; b < a.batch; b += 256u) {
        s = tree_seq(a, b, blockIdx.x == 0);
        const TreeWork<NR> work(a, s);
        mine += min((uint64_t)a.kv_heads * work.tiles * work.steps, (uint64_t)1 << 40);
    }
    const uint32_t low = lanes_scan((uint32_t)mine & 0xFFFFu), high = lanes_scan((uint32_t)min(mine >> 16, (uint64_t)1 << 23));
    if (lane == 63u) {
        s_sum[wave] = low;
        s_sum[9u + wave] = high;
    }
    __syncthreads();
    const uint64_t steps = ((uint64_t)(s_sum[9] + s_sum[10] + s_sum[11] + s_sum[12]) << 16) + s_sum[0] + s_sum[1] + s_sum[2] + s_sum[3];
    const uint32_t total = uniform(steps < kTreeSteps ? (uint32_t)steps : 0u);
    const uint32_t each = uniform((total + a.work_groups - 1u) / a.work_groups);
    uint32_t pos = w * each;
    const uint32_t stop = min(pos + each, total);
    uint32_t* cut = a.cuts + (uint64_t)w * kCutWords;
    if (pos >= stop) {
        if (tid == 0) cut[0] = 0;
        return;
    }
    // The sequence that holds the first of them: 256 at a time.
    uint32_t base = 0, b = 0;
    for (uint32_t c0 = 0; c0 < a.batch; c0 += 256u) {
        if (a.batch > 256u) {
            s = TreeSeq{};
            if (c0 + tid < a.batch) s = tree_seq(a, c0 + tid, false);
        }
        const uint32_t x = TreeWork<NR>(a, s).all(a.kv_heads);
        uint32_t sum = lanes_scan(x);
        __syncthreads(); // the sums before have been read
        if (lane == 63u) s_sum[wave] = sum;
        __syncthreads();
        uint32_t all = 0;
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            if (i < wave) sum += s_sum[i];
            all += s_sum[i];
        }
        sum += base;
        if (sum - x <= pos && pos < sum) { // one thread
            s_sum[4] = sum - x;
            s_sum[5] = c0 + tid;
            s_sum[6] = s.first;
            s_sum[7] = s.nodes;
            s_sum[8] = s.held;
        }
        if (pos < base + all) break; // uniform
        base += all;
    }
    __syncthreads();
    base = uniform(s_sum[4]);
    b = uniform(s_sum[5]);
    s = {uniform(s_sum[6]), uniform(s_sum[7]), uniform(s_sum[8])};
    __syncthreads(); // what was found has been read
    uint32_t parts = 0, cut_rows = 0, cut_row0 = 0, cut_first = 0, cut_g = 0;
    for (;;) {
        const TreeWork<NR> work(a, s);
        const uint32_t all = work.all(a.kv_heads);
        while (pos < stop && pos - base < all) {
            const uint32_t unit = uniform((pos - base) / work.steps), s0 = (pos - base) - unit * work.steps, s1 = min(work.steps, s0 + (stop - pos));
            const uint32_t g = uniform(unit / work.tiles), row0 = (unit - g * work.tiles) * kRows, rows = s.nodes * a.gqa;
            const bool whole = s0 == 0 && s1 == work.steps;
            const uint64_t slot = (2ull * w + (s0 == 0 ? 1u : 0u)) * kRows;
            const uint64_t head = (uint64_t)g * a.gqa * HD, kv = (uint64_t)g * HD;
            const uint32_t* table = a.refs + (uint64_t)b * a.refs_stride;
            auto fill = [&](auto& p) {
                p.q = a.q + s.first * a.q_stride + head;
                p.k = a.hk + kv;
                p.v = a.hv + kv;
                p.q_step = a.q_stride;
                p.blocks = a.blocks;
                p.rstride = a.kv_heads * (uint32_t)HD;
                p.gqa = a.gqa;
                p.row0 = row0;
                p.q_and = a.q_and;
                p.q_xor = a.q_xor;
                p.scale_log2 = a.scale_log2;
                p.m = a.part_m + (int64_t)(slot - row0);
                p.l = a.part_l + (int64_t)(slot - row0);
                p.o = a.part_o + (int64_t)(slot - row0) * HD;
                p.err = a.err;
                p.nk = a.k + s.first * a.k_stride + kv;
                p.nv = a.v + s.first * a.v_stride + kv;
                p.nk_step = a.k_stride;
                p.nv_step = a.v_stride;
                p.mask = a.mask ? a.mask + (uint64_t)s.first * a.mask_words : nullptr;
                p.mask_words = a.mask_words;
                p.out = whole ? a.out + s.first * a.out_stride + head : nullptr;
                p.o_step = a.out_stride;
            };
            if constexpr (NR > 0) {
                TreePart p{};
                fill(p);
                p.row_end = min(row0 + kRows, rows);
                const uint32_t of = (s.held + 15u) / 16u, to = of + (s.nodes + 15u) / 16u; // pages, and the nodes'
                const PageRun runs[2] = {{table, min(4u * s0, of), min(4u * s1, of), s.held, s.held},
                                         {nullptr, max(4u * s0, of) - of, max(min(4u * s1, to), of) - of, s.nodes, s.nodes}};
                TreePages<HD, 4, NR> t;
                t.run(p, runs, prefix_lds, (int)lane, wave);
            } else {
                const uint32_t of = (s.held + 63u) / 64u;
                TilePart p{};
                fill(p);
                p.rows = rows;
                p.table = table + 4u * s0;
                p.tokens = min(64u * s1, s.held) - min(64u * s0, s.held);
                p.node0 = s0 > of ? 64u * (s0 - of) : 0u;
                p.nodes = s1 > of ? min(64u * (s1 - of), s.nodes) : p.node0;
                PrefixTile<HD, true>::run(p, prefix_lds);
            }
            __syncthreads(); // the unit's LDS has been read
            if (s0 == 0 && !whole) { // the last of this work-group
                cut_rows = min(kRows, rows - row0);
                cut_row0 = row0;
                cut_first = s.first;
                cut_g = g;
                parts = 1u + (work.steps - s1 + each - 1u) / each;
            }
            pos += s1 - s0;
        }
        if (pos >= stop) break;
        base += all;
        if (++b >= a.batch) break; // not met: the steps left are a later sequence's
        s = tree_seq(a, b, false);
        s = {uniform(s.first), uniform(s.nodes), uniform(s.held)};
    }
    if (tid == 0) {
        cut[0] = parts;
        cut[1] = cut_rows;
        cut[2] = cut_row0;
        cut[3] = cut_first;
        cut[4] = cut_g;
    }
}

// Small requests, in one launch: a work-group takes 16 query rows of one kv head over all
// that they see, its waves the pages in turn.  The sequences' units lie one behind another, as
// each work-group sums up itself; the grid has one more for each sequence's last, partial 16 rows
// than all rows fill, so the host need not know the lengths.  Bound: the chain offsets, lengths, refs, pages (a
// round trip each), then the waves' sums: 2 sequences x 5 nodes x 14 / 2 heads x 64 behind 700
// tokens 9.8 us, with 16 waves 3 pages of each.  As many waves as LDS holds where the work-groups
// are no more than the CUs, else 4.
template <int HD, int NW>
__global__ __launch_bounds__(NW * 64) void tree_pages_kernel(TreeArgs a) {
    extern __shared__ __attribute__((aligned(16))) _Float16 prefix_lds[];
    auto uniform = [](uint32_t x) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)x); };
    const uint32_t lane = threadIdx.x & 63u, wave = uniform(threadIdx.x >> 6);
    // The heads of some rows, then the next rows, on one XCD (b % 8).
    const uint32_t j = blockIdx.x >> 3, i = uniform(j / a.kv_heads), g = j - i * a.kv_heads;
    const uint32_t unit = (blockIdx.x & 7u) * (a.work_groups / a.kv_heads >> 3) + i;
    // The sequence that the unit is of, whose units begin behind those of the sequences before; bad offsets give none.
    uint32_t b = a.batch, row0 = 0, first = 0, nodes = 0, held = 0;
    for (uint32_t c0 = 0, units = 0; c0 < a.batch && b == a.batch; c0 += 256u) { // wave-uniform
        TreeSeq s[4];
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k)
            if (c0 + 64u * k < a.batch) s[k] = tree_seq(a, min(c0 + 64u * k + lane, a.batch - 1u), false); // uniform
#pragma unroll
        for (uint32_t k = 0; k < 4u; ++k) {
            if (c0 + 64u * k >= a.batch) break; // uniform
            const uint32_t x = c0 + 64u * k + lane < a.batch ? (s[k].nodes * a.gqa + 15u) / 16u : 0u, end = units + lanes_scan(x);
            const uint64_t hit = __ballot(end - x <= unit && unit < end);
            if (hit) { // one lane
                const int l = __builtin_ctzll(hit);
                b = c0 + 64u * k + (uint32_t)l;
                row0 = (unit - (uint32_t)__builtin_amdgcn_readlane((int)(end - x), l)) * 16u;
                first = (uint32_t)__builtin_amdgcn_readlane((int)s[k].first, l);
                nodes = (uint32_t)__builtin_amdgcn_readlane((int)s[k].nodes, l);
                held = (uint32_t)__builtin_amdgcn_readlane((int)s[k].held, l);
            }
            units = (uint32_t)__builtin_amdgcn_readlane((int)end, 63);
        }
    }
    if (b < a.batch) {
        const uint32_t rows = nodes * a.gqa;
        TreePart p{};
        p.q = a.q + first * a.q_stride + (uint64_t)g * a.gqa * HD;
        p.k = a.hk + (uint64_t)g * HD;
        p.v = a.hv + (uint64_t)g * HD;
        p.q_step = a.q_stride;
        p.blocks = a.blocks;
        p.rstride = a.kv_heads * (uint32_t)HD;
        p.gqa = a.gqa;
        p.row0 = row0;
        p.row_end = min(row0 + 16u, rows);
        p.q_and = a.q_and;
        p.q_xor = a.q_xor;
        p.scale_log2 = a.scale_log2;
        p.out = a.out + first * a.out_stride + (uint64_t)g * a.gqa * HD;
        p.o_step = a.out_stride;
        p.err = a.err;
        p.nk = a.k + first * a.k_stride + (uint64_t)g * HD;
        p.nv = a.v + first * a.v_stride + (uint64_t)g * HD;
        p.nk_step = a.k_stride;
        p.nv_step = a.v_stride;
        p.mask = a.mask ? a.mask + (uint64_t)first * a.mask_words : nullptr;
        p.mask_words = a.mask_words;
        const PageRun runs[2] = {{a.refs + (uint64_t)b * a.refs_stride, 0, (held + 15u) / 16u, held, held}, {nullptr, 0, (nodes + 15u) / 16u, nodes, nodes}};
        TreePages<HD, NW, 1> pages;
        pages.run(p, runs, prefix_lds, (int)lane, wave);
    }
    if (blockIdx.x == 0)
        for (uint32_t c = threadIdx.x; c < a.batch; c += NW * 64u) tree_seq(a, c, true);
}

// Joins the parts of the units that are cut, a wave a row: their largest maximum, each
// part's sums times 2^(its maximum - that), in the order of the parts; zeros where no part saw a
// token.  An inf or NaN in a part's sum stays, as in prefix_merge_kernel.  Bound: round trips
// (the cut's record; factors and sums together), so a row a wave: with four rows one after
// another a request took 2 to 4 us more (182.7 for 180.8, 82.7 for 78.9).
constexpr uint32_t kTreeMergeRows = 4; // of a work-group
template <int HD, int NR>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeArgs a) {
    constexpr uint32_t LP = HD / 4, PG = 64 / LP, U = 4; // lanes of a part's row, parts of one load, loads in flight
    const uint32_t w = blockIdx.x, lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t* cut = a.cuts + (uint64_t)w * kCutWords;
    const uint32_t S = cut[0], rows = cut[1], row0 = cut[2], first = cut[3], g = cut[4];
    if (!S) return;
    const uint32_t sub = lane / LP, d = 4u * (lane % LP);
    const uint32_t r = blockIdx.y * kTreeMergeRows + wave;
    if (r >= rows) return;
    auto slot = [&](uint32_t p) { return (p ? 2ull * (w + p) : 2ull * w + 1u) * tree_rows(NR) + r; };
    float4_t v[U];
    auto load = [&](uint32_t p0) {
#pragma unroll
        for (uint32_t j = 0; j < U; ++j) v[j] = *(const float4_t*)(a.part_o + slot(min(p0 + j * PG + sub, S - 1u)) * HD + d);
    };
    float l = a.part_l[slot(min(lane, S - 1u))], m = a.part_m[slot(min(lane, S - 1u))];
    load(0); // before the parts' factors are known
    if (lane >= S || l == 0.0f) { // a part that saw nothing holds no sums
        l = 0.0f;
        m = -INFINITY;
    }
    float M = m;
    for (uint32_t p = lane + 64u; p < S; p += 64u)
        if (a.part_l[slot(p)] != 0.0f) M = fmaxf(M, a.part_m[slot(p)]);
    M = wave_max(M);
    float L = 0.0f;
    float4_t acc = (float4_t)0.0f;
    for (uint32_t c0 = 0; c0 < S; c0 += 64u) { // 64 parts' factors in the lanes
        if (c0) {
            l = c0 + lane < S ? a.part_l[slot(c0 + lane)] : 0.0f;
            m = l != 0.0f ? a.part_m[slot(c0 + lane)] : -INFINITY;
        }
        const float f = l != 0.0f ? fast_exp2(m - M) : 0.0f;
        const uint64_t saw = __ballot(l != 0.0f);
        L += wave_sum(f * l);
        for (uint32_t p0 = 0; p0 < min(S - c0, 64u); p0 += U * PG) {
            if (c0 + p0) load(c0 + p0);
#pragma unroll
            for (uint32_t j = 0; j < U; ++j) {
                const uint32_t p = p0 + j * PG + sub; // < 64
                const float fp = __shfl(f, (int)p);
                if ((saw >> p) & 1u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[e] = fmaf(fp, v[j][e], acc[e]);
            }
        }
    }
#pragma unroll
    for (int o = LP; o < 64; o *= 2)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[e] += __shfl_xor(acc[e], o);
    if (sub) return;
    const uint32_t R = row0 + r;
    half4_t h;
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = (_Float16)(L == 0.0f ? 0.0f : acc[e] / L);
    *(half4_t*)(a.out + (first + R / a.gqa) * a.out_stride + (g * a.gqa + R % a.gqa) * (uint64_t)HD + d) = h;
}

} // namespace aw
