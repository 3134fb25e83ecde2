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
    uint32_t prefix_splits, own_splits, splits; // splits = prefix_splits + own_splits
    uint32_t prefix_span, own_span;             // tokens of a split, a multiple of 32
    uint32_t prefix_wgs, work_groups;           // work-groups of PrefixTile parts, all
    uint32_t prefix_units, own_units;           // one-wave parts, kv_heads each
    uint32_t prefix_tiles, own_tiles;
    uint64_t blocks;
    float scale_log2;           // > 0
    uint32_t q_and, q_xor;      // of two halves of q: the sign of the scale, or all zero for a scale of 0
};

// 8 halves of a query row.
__device__ __forceinline__ half8_t prefix_query(const PrefixArgs& a, const uint16_t* p) {
    uint4_t w = *(const uint4_t*)p;
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = (w[e] & a.q_and) ^ a.q_xor;
    return as_h8(w);
}

// Few rows to a table (a sequence's own pages; a prefix that at most kPrefixFewRows rows
// see): 16 query rows of one kv head x the tokens [t0, t1), one wave, as in the decode
// over hot blocks: S^T = K Q^T and O^T += V^T P^T on 16 x 16 x 32 MFMAs, 32 tokens a
// step, the next step's rows loading while this one is multiplied, V read back from LDS
// transposed.  A row's softmax keeps its running maximum and sum in fp32; weights are f16
// operands of the second product (each off by 2^-12 of itself, independently: less than
// the f16 store of the output).  Bound: HBM, the pages' bytes.
// Tokens past `end` and tokens of a bad ref count as zeros that score -inf.
constexpr uint32_t kPrefixFewRows = 32;

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
        if (t0 >= t1) return;
        // Refs of 64 blocks, one in each lane, and of the next 64.
        const uint32_t last = (end - 1u) / kBlockTokens, first = t0 / kBlockTokens;
        uint32_t held = 0;
        uint32_t refv = table[min(first + (uint32_t)lane, last)] & kRefMask;
        uint32_t refn = table[min(first + 64u + (uint32_t)lane, last)] & kRefMask;
        // The 32 tokens from c0 on: this lane's pieces of K and V (loads that nothing masks:
        // a bad ref reads block 0), and whether each block counts.
        auto load = [&](uint32_t c0, uint4_t (&kr)[2][KS], uint4_t (&vr)[2][KS], bool (&ok)[2]) {
            const uint32_t b0 = c0 / kBlockTokens - first;
            if (b0 / 64u != held) { // a step's two blocks lie in one run of 64
                held = b0 / 64u;
                refv = refn;
                refn = table[min(first + (held + 1u) * 64u + (uint32_t)lane, last)] & kRefMask;
            }
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)refv, (int)((b0 + (uint32_t)tb) & 63u));
                const bool in = c0 + 16u * tb < end;
                ok[tb] = in && ref < a.blocks;
                bad |= in && !ok[tb];
                const uint64_t at = (((uint64_t)(ok[tb] ? ref : 0u) * kBlockTokens + li) * a.kv_heads + g) * HD + 8 * lg;
#pragma unroll
                for (int j = 0; j < KS; ++j) kr[tb][j] = *(const uint4_t*)(a.k + at + 32 * j);
#pragma unroll
                for (int j = 0; j < KS; ++j) vr[tb][j] = *(const uint4_t*)(a.v + at + 32 * j);
            }
        };
        auto process = [&](uint32_t c0, uint4_t (&kr)[2][KS], uint4_t (&vr)[2][KS], const bool (&ok)[2]) {
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
                if (!ok[tb] || c0 + 16u * tb + (uint32_t)li >= end)
#pragma unroll
                    for (int j = 0; j < KS; ++j) kr[tb][j] = vr[tb][j] = (uint4_t)0u;
            float4_t sacc[2];
#pragma unroll
            for (int tb = 0; tb < 2; ++tb) {
                sacc[tb] = (float4_t)0.0f;
#pragma unroll
                for (int j = 0; j < KS; ++j) sacc[tb] = mfma16x16x32(as_h8(kr[tb][j]), qop[j], sacc[tb]);
            }
            wave_lds_order(); // the reads of the last step
#pragma unroll
            for (int tb = 0; tb < 2; ++tb)
#pragma unroll
                for (int j = 0; j < KS; ++j) *(uint4_t*)(lds + (16 * tb + li) * P + 32 * j + 8 * lg) = vr[tb][j];
            wave_lds_order();
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
        };
        // Two sets of registers in turn.
        uint4_t k0[2][KS], v0[2][KS], k1[2][KS], v1[2][KS];
        bool ok0[2], ok1[2];
        load(t0, k0, v0, ok0);
        for (uint32_t c0 = t0; c0 < t1; c0 += 64u) {
            const bool more = c0 + 32u < t1;
            if (more) load(c0 + 32u, k1, v1, ok1);
            process(c0, k0, v0, ok0);
            if (!more) break;
            if (c0 + 64u < t1) load(c0 + 64u, k0, v0, ok0);
            process(c0 + 32u, k1, v1, ok1);
        }
        l_run += __shfl_xor(l_run, 16);
        l_run += __shfl_xor(l_run, 32);
    }

    // LDS that one wave alone uses is written and read in order by the hardware; this keeps the compiler to it.
    static __device__ __forceinline__ void wave_lds_order() {
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    }

    __device__ __forceinline__ void run(const PrefixArgs& a, const uint32_t* table, uint32_t g, uint32_t row, bool valid,
                                        uint32_t t0, uint32_t t1, uint32_t end, uint32_t lim, uint32_t slot, _Float16* lds,
                                        int lane) {
        const int lg = lane >> 4;
        const uint32_t head = g * a.gqa + row % a.gqa;
        const uint16_t* p = a.q + ((uint64_t)(row / a.gqa) * a.q_heads + head) * HD;
#pragma unroll
        for (int j = 0; j < KS; ++j) qop[j] = prefix_query(a, p + 32 * j + 8 * lg);
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
constexpr uint32_t kPrefixRows = 128;
constexpr float kPrefixGrow = 8.0f;
constexpr int kPrefixThreads = 256;
constexpr int kPrefixTok = 64, kPrefixBufs = 2; // tokens a step, steps of K (and of V) in LDS
constexpr size_t prefix_lds_bytes(int HD) { return (size_t)kPrefixBufs * 2 * kPrefixTok * HD * 2; }

template <int HD>
struct PrefixTile {
    static constexpr int TOK = kPrefixTok, BUFS = kPrefixBufs, PAGES = TOK / 16, TB = TOK / 32;
    static constexpr int CH = HD / 8, KS = HD / 16, NB = HD / 32;
    static constexpr int LPT = TOK * CH / kPrefixThreads; // loads per thread, operand and step
    static constexpr uint32_t OP = TOK * HD;              // halves per staged operand
    static constexpr int NS = TB * KS, NV = 2 * TB * NB;  // MFMAs of a step's scores, of its output
    static constexpr int EXP = 16 * TB / NS;              // weights worked out beside one MFMA of the scores
    static constexpr int AHEAD = 4;                       // fragments read ahead of their MFMAs
    static_assert(prefix_lds_bytes(HD) >= (size_t)4 * 32 * (HD + 16) * 2, "the one-wave parts' LDS");
    static_assert(BUFS >= 2 && EXP % 2 == 0 && 16 * TB % NS == 0 && NS >= 2 * LPT && NS >= AHEAD && NV >= AHEAD, "");

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

    static __device__ __forceinline__ void run(const PrefixArgs& a, uint32_t g, uint32_t tile, uint32_t s, _Float16* lds) {
        const int tid = threadIdx.x, lane = tid & 63, li = lane & 31, hf = lane >> 5;
        const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
        const uint32_t t0 = s * a.prefix_span, t1 = min(t0 + a.prefix_span, a.prefix_tokens); // t0 < t1
        const int steps = (int)((t1 - t0 + (uint32_t)TOK - 1u) / (uint32_t)TOK);
        const uint32_t row = tile * kPrefixRows + 32u * (uint32_t)wave + (uint32_t)li;
        const bool wave_rows = tile * kPrefixRows + 32u * (uint32_t)wave < a.rows;

        half8_t qop[KS];
        {
            const uint32_t r = min(row, a.rows - 1u);
            const uint16_t* p = a.q + ((uint64_t)(r / a.gqa) * a.q_heads + g * a.gqa + r % a.gqa) * HD;
#pragma unroll
            for (int j = 0; j < KS; ++j) qop[j] = prefix_query(a, p + 16 * j + 8 * hf);
        }

        // Staging: load j fills slots tid + 256 j of the operand (slot -> row, chunk); a wave's
        // slots of one load lie in one page, at the same place of it for every j.
        const uint32_t rstride = a.kv_heads * (uint32_t)HD, page_halves = kBlockTokens * rstride; // halves
        const uint32_t srow = ((uint32_t)tid / CH) & 15u, schunk = (uint32_t)tid % CH;
        const uint16_t* kfrom = a.k + (uint64_t)g * HD + srow * rstride + 8u * (schunk ^ ksw(srow));
        const uint16_t* vfrom = a.v + (uint64_t)g * HD + srow * rstride + 8u * (schunk ^ vsw(srow));
        // Rows past the part's last token load that token's (and count for nothing).
        const uint32_t first = t0 / kBlockTokens, last = (t1 - 1u) / kBlockTokens - first;
        const int back = ((int)min(srow, (t1 - 1u) % kBlockTokens) - (int)srow) * (int)rstride;
        // Refs of 64 pages, one in each lane, and which of them count: the run of the newest K
        // step, the one before it, and (refs alone) the next.
        uint32_t held, ref_cur, ref_old, ref_next;
        uint64_t ok_cur, ok_old;
        bool bad = false;
        auto refs_from = [&](uint32_t run) { return a.prefix_refs[first + min(64u * run + (uint32_t)lane, last)] & kRefMask; };
        auto take = [&](uint32_t run) {
            held = run;
            ref_old = ref_cur;
            ok_old = ok_cur;
            const bool ok = ref_next < a.blocks;
            ref_cur = ok ? ref_next : 0u;
            ok_cur = __ballot(ok);
            bad |= !ok;
            ref_next = refs_from(run + 1u);
        };
        // Load j of a step of K or V; INNER: the step is not the part's last.
        auto load = [&](auto inner, const uint16_t* from, uint32_t refs, int step, _Float16* dst, int j) {
            const uint32_t p = (uint32_t)(CH == 16 ? j : 2 * j + (wave >> 1)); // page: 16 rows a load, or 32
            const uint32_t b = (uint32_t)step * (uint32_t)PAGES + p, at = decltype(inner)::value ? b : min(b, last);
            const uint32_t ref = (uint32_t)__builtin_amdgcn_readlane((int)refs, (int)(at & 63u));
            const uint16_t* src = from + (uint64_t)ref * page_halves;
            if constexpr (!decltype(inner)::value) src += b >= last ? back : 0;
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                             (__attribute__((address_space(3))) void*)(dst + ((uint32_t)wave * 512u + (uint32_t)(kPrefixThreads * 8 * j))), 16, 0, 0);
        };
        // The pair (V of step v into its buffer vbuf, K of step v + 1 into kbuf): 2 LPT loads, x < LPT of V.  ready() first.
        uint32_t vrefs;
        auto ready = [&](int v) {
            if (v + 1 < steps && (uint32_t)(v + 1) * (uint32_t)PAGES / 64u != held) take(held + 1u); // a step's pages lie in one run of 64
            vrefs = (uint32_t)v * (uint32_t)PAGES / 64u == held ? ref_cur : ref_old;
        };
        auto load_pair = [&](auto inner, int x, int v, uint32_t vbuf, uint32_t kbuf) {
            constexpr bool INNER = decltype(inner)::value;
            if (x < LPT) {
                if (INNER || (v >= 0 && v < steps)) load(inner, vfrom, vrefs, v, lds + (BUFS + vbuf) * OP, x);
            } else if (INNER || v + 1 < steps) {
                load(inner, kfrom, ref_cur, v + 1, lds + kbuf * OP, x - LPT);
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
        // One step: the weights of `sc` (this step's scores), this step's output, and beside
        // the weights the next step's scores into `sn`.  SPLIT: as in PrefixWave.
        auto process = [&](auto split, int step, const _Float16* sk, const _Float16* sv, float16_t (&sc)[TB], float16_t (&sn)[TB], auto load_x) {
            constexpr bool SPLIT = decltype(split)::value;
            const uint32_t c0 = t0 + (uint32_t)step * (uint32_t)TOK, b0 = (uint32_t)step * (uint32_t)PAGES;
            const uint32_t ok4 = (uint32_t)((b0 / 64u == held ? ok_cur : ok_old) >> (b0 & 63u)) & ((1u << PAGES) - 1u);
            __asm__ volatile("" : "+v"(kat), "+v"(va), "+v"(vb)); // their other forms are made in each step, not kept: no spills
            half8_t kf[AHEAD], vf[AHEAD];
#pragma unroll
            for (int x = 0; x < AHEAD; ++x) kf[x] = kfrag(sk, x);
            if (c0 + (uint32_t)TOK > t1 || ok4 != (1u << PAGES) - 1u) { // wave-uniform
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
            for (int tb = 0; tb < TB; ++tb)
#pragma unroll
                for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sc[tb][i]);
            const auto sw = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(uint32_t, mx), __builtin_bit_cast(uint32_t, mx), false, false);
            const uint32_t sw0 = sw[0], sw1 = sw[1]; // the row's two halves
            mx = fmaxf(__builtin_bit_cast(float, sw0), __builtin_bit_cast(float, sw1)) * a.scale_log2;
            if (__any(mx > m_run + kPrefixGrow)) {
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
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int x = 0; x < NS; ++x) {
                sn[x % TB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf[x % AHEAD], qop[x / TB], sn[x % TB], 0, 0, 0);
                if (x + AHEAD < NS) kf[x % AHEAD] = kfrag(sk, x + AHEAD);
                else vf[x + AHEAD - NS] = vfrag(sv, x + AHEAD - NS);
                if (x < 2 * LPT) load_x(x);
#pragma unroll
                for (int e = 0; e < EXP; ++e) {
                    const int at = x * EXP + e, tb = at / 16, i = at % 16;
                    const float p = fast_exp2(fmaf(sc[tb][i], a.scale_log2, -mref));
                    ps[e % 2] += p;
                    pop[tb][i / 8][i % 8] = (_Float16)p;
                    if constexpr (SPLIT) sc[tb][i] = p;
                }
                __builtin_amdgcn_sched_barrier(0);
            }
            l_run += ps[0] + ps[1];
#pragma unroll
            for (int x = 0; x < NV; ++x) {
                const int nb = x % NB;
                half8_t v = vf[x % AHEAD];
                if constexpr (SPLIT) v = finite_part(v);
                oacc[nb] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, pop[x / (2 * NB)][(x / NB) % 2], oacc[nb], 0, 0, 0);
                if (x + AHEAD < NV) vf[x % AHEAD] = vfrag(sv, x + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
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
                            if (!((slots >> slot) & 1u) || c0 + at >= t1 || !((ok4 >> (at / 16u)) & 1u)) continue; // uniform
                            const half4_t v = *(const half4_t*)(sv + at * HD + 8u * slot + 4 * hf);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                const float f = (float)v[e];
                                if (!(fabsf(f) < INFINITY)) oacc[nb][i + e] = fmaf(p, f, oacc[nb][i + e]);
                            }
                        }
                }
            }
        };

        // Waits until at most `pairs` of this wave's newest pairs of V and K are in flight, and its LDS reads are done.
        auto wait = [](auto pairs) {
            constexpr uint32_t vm = (uint32_t)decltype(pairs)::value * 2u * (uint32_t)LPT;
            __builtin_amdgcn_s_waitcnt((short)((vm & 15u) | ((vm >> 4) << 14) | (7u << 4))); // vmcnt(vm), lgkmcnt(0)
        };
        // Step i of K sits in buffer i % BUFS of K, of V likewise.  While step i is worked, V of
        // i and K of i + 1 are read, and the pair (V of i + BUFS - 1, K of i + BUFS) is loaded
        // into what every wave has read before.
        auto pass = [&](auto split) {
            using I0 = std::integral_constant<int, 0>;
            m_run = -INFINITY;
            l_run = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) oacc[nb] = (float16_t)0.0f;
            ref_cur = 0;
            ok_cur = 0;
            ref_next = refs_from(0);
            take(0);
            float16_t s0[TB], s1[TB];
#pragma unroll
            for (int v = -1; v < BUFS - 1; ++v) {
                vrefs = ref_cur; // BUFS steps lie in the first run
#pragma unroll
                for (int x = 0; x < 2 * LPT; ++x) load_pair(std::false_type{}, x, v, (uint32_t)(v + BUFS) % BUFS, (uint32_t)(v + 1));
            }
            if (steps >= BUFS) wait(std::integral_constant<int, BUFS - 1>{});
            else wait(I0{});
            barrier();
#pragma unroll
            for (int tb = 0; tb < TB; ++tb) s0[tb] = (float16_t)0.0f;
            if (wave_rows)
#pragma unroll
                for (int x = 0; x < NS; ++x)
                    s0[x % TB] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kfrag(lds, x), qop[x / TB], s0[x % TB], 0, 0, 0);
            uint32_t cur = 0, nxt = 1, old = BUFS - 1; // buffers of i, i + 1, i - 1
            // INNER: the pair that this step loads is whole, and not of the part's last step.
            auto step = [&](auto inner, int i, float16_t (&sc)[TB], float16_t (&sn)[TB]) {
                if (decltype(inner)::value || i - 1 + BUFS < steps) wait(std::integral_constant<int, BUFS - 2>{}); // every pair so far was whole
                else wait(I0{});
                barrier();
                ready(i + BUFS - 1);
                auto load_x = [&](int x) { load_pair(inner, x, i + BUFS - 1, old, cur); };
                if (wave_rows) {
                    process(split, i, lds + nxt * OP, lds + (BUFS + cur) * OP, sc, sn, load_x);
                } else {
#pragma unroll
                    for (int x = 0; x < 2 * LPT; ++x) load_x(x);
                }
                old = cur;
                cur = nxt;
                nxt = nxt + 1u == (uint32_t)BUFS ? 0u : nxt + 1u;
            };
            int i = 0;
            if constexpr (!decltype(split)::value)
                for (; i + 2 + BUFS < steps; i += 2) {
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
        if (bad && lane == 0 && wave == 0) flag_error(a.err, kErrHotRef);
        uint32_t ro = row;
        __asm__ volatile("" : "+v"(ro)); // its addresses are made here, not kept over the loops
        if (ro >= a.rows) return;
        const uint64_t at = ((uint64_t)g * a.splits + s) * a.rows + ro;
        if (hf == 0) {
            a.part_m[at] = m_run;
            a.part_l[at] = l;
        }
        if (l == 0.0f) return;
        float* po = a.part_o + at * HD;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(float4_t*)(po + 32 * nb + 2 * i + 4 * hf) =
                    (float4_t){oacc[nb][i], oacc[nb][i + 1], oacc[nb][i + 2], oacc[nb][i + 3]};
    }
};

// Work-groups 0 .. prefix_wgs - 1 take the prefix, the others four one-wave parts each.
// TILES: the prefix in PrefixTile's parts; else in one-wave parts too.
// Work-group b runs on XCD b % 8.  A head's rows lie kv_heads * HD apart, so an XCD that
// read one head alone would use a few of its L2's channels: each XCD takes all heads of
// what it reads, the parts of one stretch of tokens after another (tiles: a run of
// parts, each part's row tiles side by side, so that its pages come from memory once;
// one-wave parts: the heads of four units, a unit one sequence's part, in turn over the
// XCDs, since sequences differ in length).
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
            const uint32_t s = uniform(part / a.kv_heads);
            PrefixTile<HD>::run(a, part - s * a.kv_heads, j - i * a.prefix_tiles, s, prefix_lds);
            return;
        }
        j -= a.prefix_wgs >> 3;
    }
    const uint32_t chunk = uniform(j / a.kv_heads), item = (j - chunk * a.kv_heads) * 4u + wave; // of a chunk's 4 kv_heads items
    uint32_t unit = (chunk * 8u + xcd) * 4u + uniform(item / a.kv_heads);
    const uint32_t g = uniform(item % a.kv_heads);
    _Float16* lds = prefix_lds + wave * 32 * (HD + 16);
    const uint32_t li = (uint32_t)lane & 15u;
    PrefixWave<HD> w;
    if constexpr (!TILES) {
        if (unit < a.prefix_units) {
            const uint32_t s = uniform(unit / a.prefix_tiles), r = (unit - s * a.prefix_tiles) * 16u + li;
            const uint32_t t0 = s * a.prefix_span, t1 = min(t0 + a.prefix_span, a.prefix_tokens);
            w.run(a, a.prefix_refs, g, min(r, a.rows - 1u), r < a.rows, t0, t1, a.prefix_tokens, a.prefix_tokens, s, lds, lane);
            return;
        }
        unit -= a.prefix_units;
    }
    if (unit >= a.own_units) return;
    const uint32_t s = uniform(unit / (a.batch * a.own_tiles)), bt = unit - s * a.batch * a.own_tiles, b = uniform(bt / a.own_tiles);
    const uint32_t r = (bt - b * a.own_tiles) * 16u + li, rc = min(r, a.own_rows - 1u);
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

// A batch that sees no token at all: rows of zeros, 4 halves a lane.
__global__ __launch_bounds__(256) void prefix_zero_kernel(uint16_t* out, uint64_t n4) {
    for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < n4; i += (uint64_t)gridDim.x * 256u)
        ((half4_t*)out)[i] = (half4_t)(_Float16)0;
}

// Joins a row's parts: the largest maximum, each part's sums times 2^(its maximum -
// that), added in an order of their own; zeros where no part saw a token.  An inf or NaN
// in a part's sum stays in the result.  W waves a row (4 where rows are few, their sums
// added in the order of the waves); a row of a part is HD / 4 lanes' float4, U loads in
// flight before the parts' factors are known.
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
            if (p < S && fp != 0.0f) // a part that saw nothing holds no sums
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
