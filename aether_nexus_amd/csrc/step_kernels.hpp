// step_kernels.hpp — gfx950 kernels of a step over trees of drafted tokens, but for its
// attention: block tables from lengths, logits before a token is chosen, accepted trees.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "rotary_kernels.hpp"

#pragma clang fp contract(off)

namespace awo {

constexpr uint32_t kMaxNodes = 1024u;   // of a sequence's tree
constexpr uint32_t kErrFree = aw_engine_internal::kErrFreeBit;
constexpr uint32_t kNoPage = kPageMask; // an entry without a page

// First row and number of rows of sequence b, uniform; offsets that descend or pass the
// rows give none.
struct SeqRows {
    uint32_t first, n;
};
__device__ inline SeqRows seq_rows(const uint32_t* offsets, uint32_t tokens, uint32_t batch, uint32_t b, uint32_t* err) {
    if (!offsets) return {b * (tokens / batch), tokens / batch};
    const uint32_t first = offsets[b], end = offsets[b + 1u];
    if (first > end || end > tokens) {
        if (threadIdx.x == 0) flag(err, kErrSeq);
        return {0u, 0u};
    }
    return {first, end - first};
}

// The first sequence that ends behind row t (batch: none), as find_place searches.
__device__ inline uint32_t seq_behind(const uint32_t* offsets, uint32_t tokens, uint32_t batch, uint32_t t, uint32_t lane) {
    if (!offsets) return t / (tokens / batch);
    uint32_t b = 0, n = batch;
    while (n > 64u) {
        const uint32_t stretch = (n + 63u) / 64u, at = (lane + 1u) * stretch - 1u;
        const uint32_t skip = stretch * (uint32_t)__popcll(__ballot(at < n && offsets[b + min(at, n - 1u) + 1u] <= t));
        b += skip;
        n = n > skip ? min(n - skip, stretch) : 0u;
    }
    if (n) b += (uint32_t)__popcll(__ballot(lane < n && offsets[b + min(lane, n - 1u) + 1u] <= t));
    return b;
}

// ------------------------------------------------------- block tables from lengths

struct TablesArgs {
    uint32_t batch, tokens, hot_count, refs_stride, free_count, mask_words;
    const uint32_t *seq_held, *seq_new, *seq_pages, *free_pages, *free_first;
    const int32_t* parents;
    uint32_t *refs, *seq_hot, *pages_out, *token_offsets, *free_next;
    int64_t* slots;
    uint32_t *positions, *tree_mask;
    uint32_t* err;
};

// Sums over the work-group's 256 threads that stop at `cap` (addition that saturates is
// associative, so no length overflows them): x becomes the sum of the threads before
// this one, the sum of all is returned.
__device__ inline uint32_t capped_scan(uint32_t& x, uint32_t cap, uint32_t* s_wave) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t sum = x; // x, cap <= 2^30
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
        const uint32_t y = __shfl_up(sum, o);
        if (lane >= (uint32_t)o) sum = min(sum + y, cap);
    }
    __syncthreads(); // s_wave of a scan before has been read
    if (lane == 63u) s_wave[wave] = sum;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (uint32_t w = 0; w < 4u; ++w) {
        if (w < wave) before = min(before + s_wave[w], cap);
        all = min(all + s_wave[w], cap);
    }
    const uint32_t up = __shfl_up(sum, 1);
    x = lane ? min(before + up, cap) : before;
    return all;
}

// One launch: each work-group sums the lengths of all sequences before its 256 rows
// itself, 1024 sequences at a time (12 KB of L2 reads), and makes its rows; a page is entered
// by the row that begins it, so nothing waits for another work-group.  The first work-group
// writes what belongs to sequences.  A node's ancestors are walked in LDS.
// Bound: a launch and the chain lengths -> sums -> search -> page -> slot.
constexpr uint32_t kTablesRows = 256, kTablesSeqs = 1024;

template <bool TREE>
__global__ __launch_bounds__(256) void tables_kernel(TablesArgs a) {
    __shared__ uint32_t s_off[kTablesSeqs + 1], s_held[kTablesSeqs], s_pages[kTablesSeqs], s_start[kTablesSeqs], s_wave[4];
    __shared__ int32_t s_par[TREE ? kTablesRows + kMaxNodes : 1];
    const uint32_t tid = threadIdx.x, t0 = blockIdx.x * kTablesRows, t1 = min(t0 + kTablesRows, a.tokens), t = t0 + tid;
    const uint32_t p0 = t0 > kMaxNodes ? t0 - kMaxNodes : 0u; // parents from here on are at hand
    if constexpr (TREE)
        for (uint32_t i = p0 + tid; i < t1; i += 256u) s_par[i - p0] = a.parents[i];
    const uint32_t room = a.hot_count * kPageTokens; // <= 2^30
    uint32_t tokens = 0, pages = a.free_first ? min(a.free_first[0], 1u << 30) : 0u; // before the chunk
    bool bad_seq = false, bad_free = false;
    for (uint32_t c0 = 0; c0 < a.batch; c0 += kTablesSeqs) {
        uint32_t held[4], had[4], n[4], need[4];
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            const uint32_t s = c0 + 4u * tid + j;
            held[j] = had[j] = n[j] = 0;
            if (s < a.batch) {
                held[j] = a.seq_held[s];
                const uint32_t want = a.seq_new[s], most = held[j] < room ? room - held[j] : 0u;
                n[j] = min(min(want, most), min(a.tokens, TREE ? 32u * a.mask_words : a.tokens));
                bad_seq |= n[j] < want || held[j] > room;
                held[j] = min(held[j], 0xFFFFFFFFu - kPageTokens);
                const uint32_t least = (held[j] + kPageTokens - 1u) / kPageTokens;
                had[j] = a.seq_pages ? a.seq_pages[s] : least;
                bad_seq |= had[j] < least;
                had[j] = max(had[j], least);
            }
            sum = min(sum + n[j], a.tokens);
        }
        const uint32_t all = capped_scan(sum, a.tokens, s_wave);
        uint32_t off = min(tokens + sum, a.tokens), taken = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            const uint32_t end = min(off + n[j], a.tokens);
            bad_seq |= end - off < n[j];
            n[j] = end - off;
            const uint32_t after = n[j] ? (held[j] + n[j] + kPageTokens - 1u) / kPageTokens : 0u;
            need[j] = after > had[j] ? after - had[j] : 0u;
            taken = min(taken + need[j], 1u << 30);
            s_off[4u * tid + j] = off;
            s_held[4u * tid + j] = held[j];
            s_pages[4u * tid + j] = had[j];
            off = end;
        }
        const uint32_t all_pages = capped_scan(taken, 1u << 30, s_wave);
        uint32_t from = min(pages + taken, 1u << 30);
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            s_start[4u * tid + j] = from;
            from = min(from + need[j], 1u << 30);
            bad_free |= need[j] && from > a.free_count;
        }
        const uint32_t count = min(a.batch - c0, kTablesSeqs);
        tokens = min(tokens + all, a.tokens);
        pages = min(pages + all_pages, 1u << 30);
        if (tid == 0) s_off[kTablesSeqs] = tokens; // of the last sequence's end; those past `count` are empty
        if (blockIdx.x == 0) {
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                const uint32_t s = c0 + 4u * tid + j;
                if (s >= a.batch) continue;
                a.seq_hot[s] = held[j] + n[j];
                if (a.pages_out) a.pages_out[s] = had[j] + need[j];
                a.token_offsets[s] = s_off[4u * tid + j];
            }
        }
        __syncthreads();
        if (t < t1 && t >= s_off[0] && t < tokens) {
            uint32_t k = 0; // the last sequence that begins at or before t: it holds t
            for (uint32_t step = kTablesSeqs / 2; step; step /= 2)
                if (k + step < count && s_off[k + step] <= t) k += step;
            const uint32_t i = t - s_off[k], place = s_held[k] + i, page = place / kPageTokens;
            const uint64_t entry = (uint64_t)(c0 + k) * a.refs_stride + page;
            uint32_t ref;
            if (page >= s_pages[k]) { // a page taken here, named by the row that begins it
                const uint32_t f = s_start[k] + (page - s_pages[k]);
                ref = f < a.free_count ? a.free_pages[f] & kPageMask : kNoPage;
                if (place % kPageTokens == 0u) a.refs[entry] = ref;
            } else {
                ref = a.refs[entry] & kPageMask;
            }
            if (a.slots) a.slots[t] = ref == kNoPage ? -1 : (int64_t)ref * kPageTokens + place % kPageTokens;
            uint32_t position = place;
            if constexpr (TREE) {
                uint32_t* row = a.tree_mask + (uint64_t)t * a.mask_words;
                const uint32_t base = t - i - p0; // of the tree's parents at hand (mod 2^32: the nodes needed are)
                uint32_t cur = i, word = i / 32u, bits = 1u << (i % 32u), depth = 0;
                for (uint32_t w = word + 1u; w < a.mask_words; ++w) row[w] = 0;
                for (int32_t p = s_par[base + i]; p >= 0; p = s_par[base + cur]) { // nodes descend: at most i steps
                    if ((uint32_t)p >= cur) {
                        bad_seq = true;
                        break;
                    }
                    cur = (uint32_t)p;
                    ++depth;
                    while (word > cur / 32u) {
                        row[word--] = bits;
                        bits = 0;
                    }
                    bits |= 1u << (cur % 32u);
                }
                row[word] = bits;
                while (word > 0) row[--word] = 0;
                position = s_held[k] + depth;
            }
            if (a.positions) a.positions[t] = position;
        }
        __syncthreads(); // the chunk has been read
        if (blockIdx.x && tokens >= t1) break; // uniform
    }
    if (t < t1 && t >= tokens) { // behind the last sequence
        if (a.slots) a.slots[t] = -1;
        if (a.positions) a.positions[t] = 0;
        if constexpr (TREE)
            for (uint32_t w = 0; w < a.mask_words; ++w) a.tree_mask[(uint64_t)t * a.mask_words + w] = 0;
    }
    if (blockIdx.x == 0 && tid == 0) {
        a.token_offsets[a.batch] = tokens;
        if (a.free_next) a.free_next[0] = min(pages, max(a.free_count, a.free_first ? a.free_first[0] : 0u));
    }
    if (__any(bad_seq) && (tid & 63u) == 0u) flag(a.err, kErrSeq);
    if (__any(bad_free) && (tid & 63u) == 0u) flag(a.err, kErrFree);
}

// ------------------------------------------------------- logits before a token is chosen

struct LogitsArgs {
    uint32_t rows, vocab, batch, mask_words, history_stride, bias_stride, allowed_rows;
    uint64_t logits_stride, out_stride, allowed_stride;
    const void* logits;
    void* out;
    int32_t* best;
    uint64_t* keys; // [rows][slices] where there are several slices
    const uint32_t *token_offsets, *history, *history_count, *prompt_count;
    const float *repetition, *frequency, *presence;
    const uint32_t *node_tokens, *tree_mask, *bias_ids;
    const float* bias_values;
    const uint32_t *bias_count, *allowed;
    const int32_t* allowed_index;
    uint32_t* err;
    uint32_t slices, group; // rows of a work-group
};

// A token's word in LDS: how often it counts, its bias entry + 1, and whether it is in the prompt.
constexpr uint32_t kCountBits = 21, kBiasBits = 10;
constexpr uint32_t kCountMask = (1u << kCountBits) - 1u, kBiasMask = (1u << kBiasBits) - 1u;

// An fp32 value (-0 taken as 0) and a token as one word: the largest word is the largest
// value's, the lowest of its tokens.
__device__ inline uint64_t best_key(float x, uint32_t token) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.0f);
    return (uint64_t)(b >> 31 ? ~b : b | 0x80000000u) << 32 | (uint32_t)~token;
}
__device__ inline int32_t best_token(uint64_t key) {
    return (uint32_t)(key >> 32) <= 0x007FFFFFu ? -1 : (int32_t) ~(uint32_t)key; // at most -inf
}
constexpr uint64_t kNoRow = ~0ull; // a row of no sequence: above the key of any number

__device__ inline uint64_t wave_max64(uint64_t x) {
#pragma unroll
    for (int o = 32; o; o /= 2) {
        const uint64_t y = (uint64_t)__shfl_xor((uint32_t)(x >> 32), o) << 32 | __shfl_xor((uint32_t)x, o);
        x = x > y ? x : y;
    }
    return x;
}

template <typename T>
struct LogitsVec; // 16 bytes of logits at an element's alignment
template <>
struct LogitsVec<float> {
    typedef float type __attribute__((ext_vector_type(4), aligned(4)));
};
template <>
struct LogitsVec<_Float16> {
    typedef _Float16 type __attribute__((ext_vector_type(8), aligned(2)));
};

// Work-group = `group` rows x a slice of 1024 IT (f16: 2048 IT) tokens.  The slice's
// counts are a word a token in LDS: made once for a sequence from its history and
// biases (integer atomics: no order shows in them), and for each row the tokens of its own
// nodes are added and those of the row before taken off.  Logits go by in 16-byte pieces, read before the counts are
// ready; tokens without a word take none of the arithmetic.
// Bound: HBM, each logit read and written once.
template <typename T, int IT, bool WORDS>
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs a) {
    typedef typename LogitsVec<T>::type vec_t;
    constexpr uint32_t VEC = 16 / sizeof(T), SLICE = 256u * VEC * IT;
    __shared__ __attribute__((aligned(16))) uint32_t s_word[WORDS ? SLICE : 1];
    __shared__ uint64_t s_key[4];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    const uint32_t group = blockIdx.x / a.slices, slice = blockIdx.x - group * a.slices;
    const uint32_t v0 = slice * SLICE, len = min(SLICE, a.vocab - v0);
    const uint32_t r0 = group * a.group, r1 = min(r0 + a.group, a.rows);
    uint32_t b = 0, first = 0, end = a.rows, before = ~0u; // the sequence and its rows; the row whose nodes are counted
    const bool ragged = a.batch != 0u; // else the rows stand for themselves
    if (ragged) {
        b = (uint32_t)__builtin_amdgcn_readfirstlane((int)seq_behind(a.token_offsets, a.rows, a.batch, r0, lane));
        end = r0; // looked up below
    }
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    auto count_nodes = [&](uint32_t r, uint32_t by) { // the tokens that row r's mask names
        const uint32_t n = min(end - first, 32u * a.mask_words);
        for (uint32_t j = tid; j < n; j += 256u)
            if (a.tree_mask[(uint64_t)r * a.mask_words + j / 32u] >> (j % 32u) & 1u) {
                const uint32_t id = a.node_tokens[first + j] - v0;
                if (id < len) atomicAdd(&s_word[id], by);
            }
    };
    for (uint32_t r = r0; r < r1; ++r) {
        if (ragged && r >= end) { // uniform
            if (r != r0) ++b;
            SeqRows at{0, 0};
            for (; b < a.batch; ++b) {
                at = seq_rows(a.token_offsets, a.rows, a.batch, b, a.err);
                if (at.first + at.n > r) break;
            }
            if (b >= a.batch || r < at.first) { // rows of no sequence
                for (; r < r1; ++r)
                    if (tid == 0 && a.best && a.slices > 1u) a.keys[(uint64_t)r * a.slices + slice] = kNoRow;
                return;
            }
            first = at.first;
            end = at.first + at.n;
            before = ~0u;
            if (a.repetition) rep = a.repetition[b];
            if (a.frequency) freq = a.frequency[b];
            if (a.presence) pres = a.presence[b];
            if constexpr (WORDS) {
                for (uint32_t i = 4u * tid; i < SLICE; i += 1024u) *(uint4_t*)(s_word + i) = (uint4_t)0u;
                __syncthreads();
                if (a.bias_ids) {
                    const uint32_t n = a.bias_count ? a.bias_count[b] : a.bias_stride;
                    if (n > a.bias_stride && tid == 0) flag(a.err, kErrSeq);
                    for (uint32_t i = tid; i < min(n, a.bias_stride); i += 256u) {
                        const uint32_t id = a.bias_ids[(uint64_t)b * a.bias_stride + i] - v0;
                        if (id < len) atomicMax(&s_word[id], (i + 1u) << kCountBits); // the last entry holds
                    }
                    __syncthreads();
                }
                if (a.history) {
                    const uint32_t n = a.history_count[b], prompt = a.prompt_count ? a.prompt_count[b] : 0u;
                    if (n > a.history_stride && tid == 0) flag(a.err, kErrSeq);
                    for (uint32_t i = tid; i < min(n, a.history_stride); i += 256u) {
                        const uint32_t id = a.history[(uint64_t)b * a.history_stride + i] - v0;
                        if (id < len) {
                            if (i < prompt) atomicOr(&s_word[id], 1u << 31);
                            else atomicAdd(&s_word[id], 1u);
                        }
                    }
                }
            }
        }
        const T* src = (const T*)a.logits + (uint64_t)r * a.logits_stride + v0;
        vec_t x[IT];
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const uint32_t at = ((uint32_t)it * 256u + tid) * VEC;
            if (at + VEC <= len) {
                x[it] = *(const vec_t*)(src + at);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < VEC; ++e) x[it][e] = at + e < len ? src[at + e] : (T)0.0f;
            }
        }
        if (WORDS && a.node_tokens) {
            if (before != ~0u) count_nodes(before, ~0u);
            count_nodes(r, 1u);
            before = r;
        }
        if constexpr (WORDS) __syncthreads();
        // The grammar's row: none, one of the table, or (an index past it) one that allows nothing.
        const uint32_t* allowed = nullptr;
        bool nothing = false;
        if (a.allowed) {
            const int32_t at = a.allowed_index ? a.allowed_index[r] : (int32_t)r;
            nothing = at >= 0 && (uint32_t)at >= a.allowed_rows;
            if (at >= 0 && !nothing) allowed = a.allowed + (uint64_t)at * a.allowed_stride + v0 / 32u;
            if (nothing && tid == 0) flag(a.err, kErrToken);
        }
        float top = -INFINITY;
        uint32_t token = 0;
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            const uint32_t at = ((uint32_t)it * 256u + tid) * VEC;
            if (at >= len) continue;
            const uint32_t may = allowed ? allowed[at / 32u] >> (at % 32u) : (nothing ? 0u : ~0u);
            vec_t y;
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e) {
                float f = (float)x[it][e];
                if constexpr (WORDS) {
                    const uint32_t w = s_word[at + e];
                    if (w) {
                        const uint32_t c = w & kCountMask, entry = w >> kCountBits & kBiasMask;
                        if (c || w >> 31) f = f > 0.0f ? f / rep : f * rep;
                        if (c) {
                            f = f - freq * (float)c;
                            f = f - pres;
                        }
                        if (entry) f = f + a.bias_values[(uint64_t)b * a.bias_stride + entry - 1u];
                    }
                }
                if (!(may >> e & 1u)) f = -INFINITY;
                if (at + e < len && f > top) {
                    top = f;
                    token = v0 + at + e;
                }
                y[e] = (T)f;
            }
            if (a.out) {
                T* dst = (T*)a.out + (uint64_t)r * a.out_stride + v0 + at;
                if (at + VEC <= len) {
                    *(vec_t*)dst = y;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < VEC; ++e)
                        if (at + e < len) dst[e] = y[e];
                }
            }
        }
        if (a.best) {
            const uint64_t key = wave_max64(best_key(top, token));
            if (lane == 0) s_key[wave] = key;
            __syncthreads();
            if (tid == 0) {
                uint64_t k = s_key[0];
#pragma unroll
                for (int w = 1; w < 4; ++w) k = k > s_key[w] ? k : s_key[w];
                if (a.slices > 1u) a.keys[(uint64_t)r * a.slices + slice] = k;
                else a.best[r] = best_token(k);
            }
        }
        __syncthreads(); // words and keys have been read
    }
}

// The best token of a row among its slices', a wave a row.
__global__ __launch_bounds__(256) void logits_best_kernel(LogitsArgs a) {
    const uint32_t lane = threadIdx.x & 63u, r = blockIdx.x * 4u + (threadIdx.x >> 6);
    if (r >= a.rows) return;
    uint64_t k = 0;
    for (uint32_t s = lane; s < a.slices; s += 64u) {
        const uint64_t y = a.keys[(uint64_t)r * a.slices + s];
        k = k > y ? k : y;
    }
    k = wave_max64(k);
    if (lane == 0 && k != kNoRow) a.best[r] = best_token(k);
}

// ------------------------------------------------------- accepted trees

struct AcceptArgs {
    uint32_t batch, tokens, layers, row; // row: values of a token's K (or V) row
    uint32_t history_stride;
    uint64_t hot_blocks, k_stride, v_stride, k_layer, v_layer, hot_layer;
    const int32_t* parents;
    const uint32_t *node_tokens, *targets, *token_offsets, *seq_held;
    const int64_t* slots;
    const uint16_t *k, *v;
    uint16_t *hot_k, *hot_v;
    uint32_t* accepted;
    int32_t* next_token;
    uint32_t* seq_hot;
    int32_t* path;
    uint32_t* history;
    const uint32_t* history_count;
    uint32_t* history_count_out;
    uint32_t* err;
};

// Work-group = a sequence x a layer: each walks the tree itself (one wave, 64 nodes a
// step: those that continue the kept node with its target's token, the lowest of them) and moves its layer's rows;
// the first layer's writes what belongs to the sequence.  VEC: rows in 16-byte pieces.
// Bound: the chain offsets -> nodes -> walk -> rows; with many layers HBM.
template <bool VEC>
__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a) {
    __shared__ int32_t s_parent[kMaxNodes], s_path[kMaxNodes];
    __shared__ uint32_t s_token[kMaxNodes], s_target[kMaxNodes], s_kept;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, b = blockIdx.x, layer = blockIdx.y;
    const SeqRows rows = seq_rows(a.token_offsets, a.tokens, a.batch, b, a.err);
    const uint32_t n = min(rows.n, kMaxNodes);
    const uint32_t count = a.history && layer == 0 ? a.history_count[b] : 0u; // before a barrier: history_count_out may be it
    for (uint32_t i = tid; i < n; i += 256u) {
        s_parent[i] = a.parents[rows.first + i];
        s_token[i] = a.node_tokens[rows.first + i];
        s_target[i] = a.targets[rows.first + i];
    }
    __syncthreads();
    if (tid < 64u) {
        uint32_t kept = n ? 1u : 0u, cur = 0;
        if (lane == 0) s_path[0] = 0;
        for (uint32_t c = 0; n && c < n;) { // nodes c .. of this step: each pass moves on, or to a later node
            const uint32_t i = c + lane;
            const uint64_t m = __ballot(i < n && i > cur && s_parent[min(i, n - 1u)] == (int32_t)cur &&
                                        s_token[min(i, n - 1u)] == s_target[cur]);
            if (m) {
                cur = c + (uint32_t)__builtin_ctzll(m);
                if (lane == 0) s_path[kept] = (int32_t)cur;
                ++kept;
                c = cur + 1u;
            } else {
                c += 64u;
            }
        }
        if (lane == 0) s_kept = kept;
    }
    __syncthreads();
    const uint32_t kept = s_kept;
    if (layer == 0) {
        for (uint32_t i = tid; i < rows.n; i += 256u) a.path[rows.first + i] = i < kept ? s_path[i] : -1;
        if (a.history) {
            const uint32_t had = min(count, a.history_stride), fits = min(kept, a.history_stride - had);
            for (uint32_t i = tid; i < fits; i += 256u) a.history[(uint64_t)b * a.history_stride + had + i] = s_token[s_path[i]];
            if (tid == 0) {
                a.history_count_out[b] = had + fits;
                if (fits < kept) flag(a.err, kErrSeq);
            }
        }
        if (tid == 0) {
            a.accepted[b] = kept;
            a.next_token[b] = kept ? (int32_t)s_target[s_path[kept - 1u]] : -1;
            a.seq_hot[b] = a.seq_held[b] + kept;
            if (rows.n > kMaxNodes) flag(a.err, kErrSeq);
        }
    }
    if (layer >= a.layers) return; // layers 0
    typedef typename std::conditional<VEC, uint4_t, uint16_t>::type piece_t;
    const uint32_t per = VEC ? a.row / 8u : a.row, total = kept * per, width = VEC ? 8u : 1u;
    for (uint32_t i = tid; i < total; i += 256u) {
        const uint32_t j = i / per, at = (i - j * per) * width;
        const int64_t slot = a.slots[rows.first + j];
        if (slot < 0) continue;
        if ((uint64_t)slot >= a.hot_blocks * kPageTokens) {
            flag(a.err, kErrPage);
            continue;
        }
        const uint64_t node = rows.first + (uint32_t)s_path[j], to = (uint64_t)layer * a.hot_layer + (uint64_t)slot * a.row + at;
        const piece_t k = *(const piece_t*)(a.k + (uint64_t)layer * a.k_layer + node * a.k_stride + at);
        if (a.v) *(piece_t*)(a.hot_v + to) = *(const piece_t*)(a.v + (uint64_t)layer * a.v_layer + node * a.v_stride + at);
        *(piece_t*)(a.hot_k + to) = k;
    }
}

} // namespace awo
