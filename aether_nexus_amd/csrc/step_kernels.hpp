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
// A sequence's first page in the list, where it takes none: past any list.  kTooMany: of more nodes than the mask's.
constexpr uint32_t kTakesNone = 1u << 30, kTooMany = kTakesNone + 1u;
constexpr int64_t kNoSlot = AW_NO_SLOT;

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
// by the row that begins it, so nothing waits for another work-group.  A sequence's rows are its
// seq_new whatever its table holds, so one that is past it moves no other's.  The first work-group
// writes what belongs to sequences.  A node's ancestors are walked in LDS.
// Bound: a launch and the chain lengths -> sums -> search -> page -> slot: 64 sequences of
// one new token 4.8 us, 256 trees of up to 48 nodes 6.4, 260000 rows of 509 prompts 6.9.
constexpr uint32_t kTablesRows = 256, kTablesSeqs = 1024;

template <bool TREE>
__global__ __launch_bounds__(256) void tables_kernel(TablesArgs a) {
    __shared__ uint32_t s_off[kTablesSeqs], s_held[kTablesSeqs], s_pages[kTablesSeqs], s_start[kTablesSeqs], s_wave[4];
    __shared__ int32_t s_par[TREE ? kTablesRows + kMaxNodes : 1];
    const uint32_t tid = threadIdx.x, t0 = blockIdx.x * kTablesRows, t1 = min(t0 + kTablesRows, a.tokens), t = t0 + tid;
    const uint32_t p0 = t0 > kMaxNodes ? t0 - kMaxNodes : 0u; // parents from here on are at hand
    if constexpr (TREE)
        for (uint32_t i = p0 + tid; i < t1; i += 256u) s_par[i - p0] = a.parents[i];
    const uint32_t room = a.hot_count * kPageTokens; // <= 2^30
    uint32_t tokens = 0, pages = a.free_first ? min(a.free_first[0], 1u << 30) : 0u; // before the chunk
    bool bad_seq = false, bad_free = false;
    for (uint32_t c0 = 0; c0 < a.batch; c0 += kTablesSeqs) {
        uint32_t held[4], had[4], n[4], need[4], lacks = 0; // bit j: pages for the tokens that it holds; bit j + 4: mask words for its nodes
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            const uint32_t s = c0 + 4u * tid + j;
            held[j] = had[j] = n[j] = 0;
            if (s < a.batch) {
                held[j] = a.seq_held[s];
                const uint32_t want = a.seq_new[s], most = held[j] < room ? room - held[j] : 0u;
                n[j] = min(want, a.tokens);
                bad_seq |= n[j] < want || want > most || held[j] > room;
                if (TREE && want > 32u * a.mask_words) lacks |= 16u << j;
                held[j] = min(held[j], 0xFE000000u); // no place passes 32 bits
                const uint32_t least = (held[j] + kPageTokens - 1u) / kPageTokens;
                had[j] = a.seq_pages ? a.seq_pages[s] : least;
                lacks |= (had[j] < least ? 1u : 0u) << j;
            }
            sum = min(sum + n[j], a.tokens);
        }
        bad_seq |= lacks != 0u;
        const uint32_t all = capped_scan(sum, a.tokens, s_wave);
        uint32_t off = min(tokens + sum, a.tokens), taken = 0;
#pragma unroll
        for (uint32_t j = 0; j < 4u; ++j) {
            const uint32_t end = min(off + n[j], a.tokens);
            bad_seq |= end - off < n[j];
            n[j] = end - off;
            const uint32_t after = n[j] ? (min(held[j] + n[j], room) + kPageTokens - 1u) / kPageTokens : 0u;
            need[j] = after > had[j] && !(lacks >> j & (TREE ? 17u : 1u)) ? after - had[j] : 0u;
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
            s_start[4u * tid + j] = TREE && lacks >> j & 16u ? kTooMany : lacks >> j & 1u ? kTakesNone : from;
            from = min(from + need[j], 1u << 30);
            bad_free |= need[j] && from > a.free_count;
        }
        const uint32_t count = min(a.batch - c0, kTablesSeqs);
        tokens = min(tokens + all, a.tokens);
        pages = min(pages + all_pages, 1u << 30);
        if (blockIdx.x == 0) {
#pragma unroll
            for (uint32_t j = 0; j < 4u; ++j) {
                const uint32_t s = c0 + 4u * tid + j;
                if (s >= a.batch) continue;
                a.seq_hot[s] = held[j] + n[j];
                if (a.pages_out) a.pages_out[s] = had[j] + min(need[j], a.free_count - min(s_start[4u * tid + j], a.free_count));
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
            uint32_t ref = kNoPage;
            if (place < room) { // else past the table
                if (page >= s_pages[k]) { // a page taken here, named by the row that begins it; or there is none
                    const uint32_t f = s_start[k] + (page - s_pages[k]);
                    ref = f < a.free_count ? a.free_pages[f] & kPageMask : kNoPage;
                    if (place % kPageTokens == 0u || i == 0u) a.refs[entry] = ref;
                } else {
                    ref = a.refs[entry] & kPageMask;
                    bad_free |= ref == kNoPage; // an entry that an earlier step found no page for
                    if (TREE && s_start[k] == kTooMany) ref = kNoPage;
                }
            }
            if (a.slots) a.slots[t] = ref == kNoPage ? kNoSlot : (int64_t)ref * kPageTokens + place % kPageTokens;
            uint32_t position = place;
            if constexpr (TREE) {
                uint32_t* row = a.tree_mask + (uint64_t)t * a.mask_words;
                const uint32_t base = t - i - p0; // of the tree's parents at hand (mod 2^32: the nodes needed are)
                const bool inside = i < 32u * a.mask_words; // else it sees nothing, and its parents need not be at hand
                uint32_t cur = i, word = inside ? i / 32u : 0u, bits = inside ? 1u << (i % 32u) : 0u, depth = 0;
                for (uint32_t w = word + 1u; w < a.mask_words; ++w) row[w] = 0;
                for (int32_t p = inside ? s_par[base + i] : -1; p >= 0; p = s_par[base + cur]) { // nodes descend: at most i steps
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
// The key of a wave's largest value and, of the lanes that have it, the lowest token: two
// reductions by DPP (rows of 16 lanes, then broadcasts), the sum in lane 63.
__device__ inline uint64_t wave_best(float top, uint32_t token) {
#define AWO_DPP(id, v, ctrl, rmask) __builtin_amdgcn_update_dpp(__builtin_bit_cast(int, id), __builtin_bit_cast(int, v), ctrl, rmask, 0xF, false)
#define AWO_DPP_ALL(STEP) STEP(0x111, 0xF) STEP(0x112, 0xF) STEP(0x114, 0xF) STEP(0x118, 0xF) STEP(0x142, 0xA) STEP(0x143, 0xC)
    float m = top;
#define AWO_DPP_MAX(ctrl, rmask) m = fmaxf(m, __builtin_bit_cast(float, AWO_DPP(-INFINITY, m, ctrl, rmask)));
    AWO_DPP_ALL(AWO_DPP_MAX)
    m = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, m), 63));
    uint32_t t = top == m ? token : ~0u;
#define AWO_DPP_MIN(ctrl, rmask) t = min(t, (uint32_t)AWO_DPP(-1, t, ctrl, rmask));
    AWO_DPP_ALL(AWO_DPP_MIN)
    t = (uint32_t)__builtin_amdgcn_readlane((int)t, 63);
#undef AWO_DPP_MIN
#undef AWO_DPP_MAX
#undef AWO_DPP_ALL
#undef AWO_DPP
    return best_key(m, t);
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

// Where the rows of a sequence lie: its number (batch: none), its rows.
struct SeqAt {
    uint32_t b, first, end;
};
// The sequence of row t, as find_place searches; both its offsets come with the search's last
// round trip.
__device__ inline SeqAt seq_at(const uint32_t* offsets, uint32_t tokens, uint32_t batch, uint32_t t, uint32_t lane) {
    if (!offsets) {
        const uint32_t each = tokens / batch, b = t / each;
        return {b, b * each, b * each + each};
    }
    uint32_t b = 0, n = batch;
    while (n > 64u) {
        const uint32_t stretch = (n + 63u) / 64u, at = (lane + 1u) * stretch - 1u;
        const uint32_t skip = stretch * (uint32_t)__popcll(__ballot(at < n && offsets[b + min(at, n - 1u) + 1u] <= t));
        b += skip;
        n = n > skip ? min(n - skip, stretch) : 0u;
    }
    if (n == 0u) return {batch, 0u, 0u};
    const uint32_t at = b + min(lane, n - 1u), lo = offsets[at], hi = offsets[at + 1u];
    const uint32_t k = (uint32_t)__popcll(__ballot(lane < n && hi <= t));
    if (k >= n) return {batch, 0u, 0u};
    return {b + k, (uint32_t)__builtin_amdgcn_readlane((int)lo, (int)k), (uint32_t)__builtin_amdgcn_readlane((int)hi, (int)k)};
}

// Work-group = `group` rows x a slice of 1024 IT (f16: 2048 IT) tokens.  The slice's counts
// are a word a token in LDS: made once for a sequence from its history and biases (integer
// atomics: no order shows in them), and for each row the tokens of its own nodes are added
// and those of the row before taken off.  Logits go by in 16-byte pieces, the last of a slice
// beginning earlier and making some values twice: with words from what was read before the row's
// first write (a barrier lies between), without them perhaps from a value already written in
// place, which the grammar alone has changed and changes no further (-inf or as it was).  The
// few tokens that have a word are taken one after another.  A row's logits, the
// first 2048 tokens of the history and the biases are asked for before their counts are known
// (history_stride and bias_stride entries are there whatever the counts), so a work-group
// waits for memory two or three times.
// Bound: HBM, each logit read and written once: 526 x 49155 f16 that no cache holds, without
// words, 25 us with the best (4.1 TB/s), 27 with a grammar, 31 with both.  With words the vector
// unit is busy 60 % of the time: 47 us with histories of 2048 tokens, the nodes of 16 trees, a
// grammar and the best (no part alone is what it waits for); 64 x 128256 f32 with histories of
// 4096 and 300 biases 25.7 us, 2.6 TB/s.
template <typename T, int IT, bool WORDS>
__global__ __launch_bounds__(256) void logits_kernel(LogitsArgs a) {
    typedef typename LogitsVec<T>::type vec_t;
    constexpr uint32_t VEC = 16 / sizeof(T), SLICE = 256u * VEC * IT, HIST = 8, BIAS = WORDS ? 4 : 1;
    __shared__ __attribute__((aligned(16))) uint32_t s_word[WORDS ? SLICE : 1];
    __shared__ float s_bias[WORDS ? 256 * BIAS : 1];
    __shared__ uint64_t s_key[2][4];
    uint32_t tid = threadIdx.x;
    const uint32_t lane = tid & 63u, wave = tid >> 6;
    const uint32_t group = blockIdx.x / a.slices, slice = blockIdx.x - group * a.slices;
    const uint32_t v0 = slice * SLICE, len = min(SLICE, a.vocab - v0);
    const uint32_t r0 = group * a.group, r1 = min(r0 + a.group, a.rows);
    const bool narrow = len < VEC; // a last slice shorter than a piece
    // Where this thread's piece `it` begins (tokens of the slice).
    auto place = [&](int it) { return min(((uint32_t)it * 256u + tid) * VEC, narrow ? 0u : len - VEC); };
    auto within = [&](int it) { return ((uint32_t)it * 256u + tid) * VEC < len; };
    vec_t x[IT];
    auto fetch = [&](uint32_t r) {
        const char* src = (const char*)a.logits + ((uint64_t)r * a.logits_stride + v0) * sizeof(T);
        if (narrow) {
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e) x[0][e] = ((const T*)src)[min(e, len - 1u)];
            return;
        }
#pragma unroll
        for (int it = 0; it < IT; ++it)
            if (within(it)) x[it] = *(const vec_t*)(src + place(it) * (uint32_t)sizeof(T));
    };
    fetch(r0);
    const bool ragged = a.batch != 0u; // else the rows stand for themselves
    SeqAt seq{0, 0, a.rows};
    if (ragged) seq.end = r0; // looked up below
    float rep = 1.0f, freq = 0.0f, pres = 0.0f;
    uint32_t node = 0, named = 0, nodes = 0; // token of node tid, whether the row before names it, nodes of the masks
    for (uint32_t r = r0; r < r1; ++r) {
        __asm__ volatile("" : "+v"(tid)); // what is made of it is made in each row, not kept: 172 registers otherwise
        if (ragged && r >= seq.end) { // uniform
            seq = seq_at(a.token_offsets, a.rows, a.batch, r, lane);
            seq = {(uint32_t)__builtin_amdgcn_readfirstlane((int)seq.b), (uint32_t)__builtin_amdgcn_readfirstlane((int)seq.first),
                   (uint32_t)__builtin_amdgcn_readfirstlane((int)seq.end)};
            const bool bad = seq.b < a.batch && (seq.first > r || seq.end <= r || seq.end > a.rows); // offsets that descend, pass the rows or begin behind them
            if (bad && tid == 0) flag(a.err, kErrSeq);
            if (seq.b >= a.batch || bad) { // rows of no sequence
                for (; r < r1; ++r)
                    if (tid == 0 && a.best && a.slices > 1u) a.keys[(uint64_t)r * a.slices + slice] = kNoRow;
                break;
            }
            if (a.repetition) rep = a.repetition[seq.b];
            if (a.frequency) freq = a.frequency[seq.b];
            if (a.presence) pres = a.presence[seq.b];
            if constexpr (WORDS) {
                const uint32_t* hist = a.history + (uint64_t)seq.b * a.history_stride;
                uint32_t h[HIST];
                auto history = [&](uint32_t from) { // tokens from + tid + 256 k
#pragma unroll
                    for (uint32_t k = 0; k < HIST; ++k) h[k] = hist[min(from + tid + 256u * k, a.history_stride - 1u)];
                };
                uint32_t held = 0, prompt = 0, entries = 0, id[BIAS];
                float value[BIAS];
                if (a.history) {
                    history(0);
                    held = a.history_count[seq.b];
                    if (a.prompt_count) prompt = a.prompt_count[seq.b];
                }
                if (a.bias_ids) {
                    entries = a.bias_count ? a.bias_count[seq.b] : a.bias_stride;
                    const uint32_t* ids = a.bias_ids + (uint64_t)seq.b * a.bias_stride;
                    const float* values = a.bias_values + (uint64_t)seq.b * a.bias_stride;
#pragma unroll
                    for (uint32_t k = 0; k < BIAS; ++k)
                        if (256u * k < a.bias_stride) { // uniform
                            const uint32_t i = min(tid + 256u * k, a.bias_stride - 1u);
                            id[k] = ids[i];
                            value[k] = values[i];
                        }
                }
                nodes = a.node_tokens ? min(seq.end - seq.first, 32u * a.mask_words) : 0u;
                if (tid < nodes) node = a.node_tokens[seq.first + tid] - v0;
                named = 0;
                for (uint32_t i = 4u * tid; i < SLICE; i += 1024u) *(uint4_t*)(s_word + i) = (uint4_t)0u;
                __syncthreads();
                if (a.bias_ids) {
                    if (entries > a.bias_stride && tid == 0) flag(a.err, kErrSeq);
                    entries = min(entries, a.bias_stride);
#pragma unroll
                    for (uint32_t k = 0; k < BIAS; ++k) {
                        const uint32_t i = tid + 256u * k, v = id[k] - v0;
                        if (i < entries) {
                            s_bias[i] = value[k];
                            if (v < len) atomicMax(&s_word[v], (i + 1u) << kCountBits); // the last entry holds
                        }
                    }
                    __syncthreads();
                }
                if (a.history) {
                    if (held > a.history_stride && tid == 0) flag(a.err, kErrSeq);
                    held = min(held, a.history_stride);
                    for (uint32_t from = 0;;) {
#pragma unroll
                        for (uint32_t k = 0; k < HIST; ++k) {
                            const uint32_t i = from + tid + 256u * k, v = h[k] - v0;
                            if (v < len && i < held) {
                                if (i < prompt) atomicOr(&s_word[v], 1u << 31);
                                else atomicAdd(&s_word[v], 1u);
                            }
                        }
                        from += 256u * HIST;
                        if (from >= held) break; // uniform
                        history(from);
                    }
                }
            }
        }
        // The grammar's row: none, one of the table, or (an index past it) nothing.
        uint32_t may[IT];
        {
            int32_t at = -1;
            if (a.allowed_index) at = a.allowed_index[r];
            else if (a.allowed) at = (int32_t)r;
            const bool nothing = at >= 0 && (uint32_t)at >= a.allowed_rows;
            if (nothing && tid == 0) flag(a.err, kErrToken);
            const char* bits = (const char*)(a.allowed + (uint64_t)(uint32_t)at * a.allowed_stride + v0 / 32u);
#pragma unroll
            for (int it = 0; it < IT; ++it) {
                may[it] = nothing ? 0u : ~0u;
                if (at >= 0 && !nothing) { // uniform; a piece may lie in two words
                    const uint32_t t = place(it), k = t / 32u * 4u;
                    may[it] = *(const uint32_t*)(bits + k) >> (t % 32u);
                    if (t % 32u > 32u - VEC) may[it] |= *(const uint32_t*)(bits + min(k + 4u, (len - 1u) / 32u * 4u)) << (32u - t % 32u);
                }
            }
        }
        if (WORDS && nodes) { // uniform: the tokens that the row's mask names, but not the row's before, and the other way
            const uint32_t* mask = a.tree_mask + (uint64_t)r * a.mask_words;
            if (tid < nodes) {
                const uint32_t now = mask[tid / 32u] >> (tid % 32u) & 1u;
                if (now != named && node < len) atomicAdd(&s_word[node], now - named);
                named = now;
            }
            for (uint32_t i = tid + 256u; i < nodes; i += 256u) { // wide trees: what the row before named is read again
                const uint32_t now = mask[i / 32u] >> (i % 32u) & 1u;
                const uint32_t was = r > r0 && r > seq.first ? mask[(int32_t)(i / 32u) - (int32_t)a.mask_words] >> (i % 32u) & 1u : 0u;
                const uint32_t v = a.node_tokens[seq.first + i] - v0;
                if (now != was && v < len) atomicAdd(&s_word[v], now - was);
            }
        }
        if constexpr (WORDS) __syncthreads();
        float top = -INFINITY;
        uint32_t token = 0;
        char* dst = (char*)a.out + ((uint64_t)r * a.out_stride + v0) * sizeof(T);
#pragma unroll
        for (int it = 0; it < IT; ++it) {
            if (!within(it)) continue;
            const uint32_t at = place(it);
            float f[VEC];
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e) f[e] = (float)x[it][e];
            if constexpr (WORDS) {
                uint32_t word[VEC], hit = 0; // tokens that have a word: few, taken one after another
#pragma unroll
                for (uint32_t e = 0; e < VEC; ++e) {
                    word[e] = s_word[at + e];
                    hit |= (word[e] ? 1u : 0u) << e;
                }
#pragma unroll 1
                for (; hit; hit &= hit - 1u) {
                    const uint32_t e = (uint32_t)__builtin_ctz(hit);
                    uint32_t w = word[0];
                    float y = f[0];
#pragma unroll
                    for (uint32_t k = 1; k < VEC; ++k) {
                        w = e == k ? word[k] : w;
                        y = e == k ? f[k] : y;
                    }
                    const uint32_t c = w & kCountMask, entry = w >> kCountBits & kBiasMask;
                    if (c || w >> 31) y = y > 0.0f ? y / rep : y * rep;
                    if (c) {
                        y = y - freq * (float)c;
                        y = y - pres;
                    }
                    if (entry) y = y + s_bias[entry - 1u];
#pragma unroll
                    for (uint32_t k = 0; k < VEC; ++k) f[k] = e == k ? y : f[k];
                }
            }
            vec_t y;
#pragma unroll
            for (uint32_t e = 0; e < VEC; ++e) {
                if (!(may[it] >> e & 1u)) f[e] = -INFINITY;
                if (f[e] > top && (!narrow || e < len)) {
                    top = f[e];
                    token = v0 + at + e;
                }
                y[e] = (T)f[e];
            }
            if (a.out) {
                if (!narrow) {
                    *(vec_t*)(dst + at * (uint32_t)sizeof(T)) = y;
                } else {
#pragma unroll
                    for (uint32_t e = 0; e < VEC; ++e)
                        if (e < len) ((T*)dst)[e] = y[e];
                }
            }
        }
        if (r + 1u < r1) fetch(r + 1u); // while this row's best is found
        uint64_t* keys = s_key[r & 1u]; // of the row before: thread 0 may still read them
        if (a.best) {
            const uint64_t key = wave_best(top, token);
            if (lane == 0) keys[wave] = key;
        }
        __syncthreads(); // words have been read
        if (a.best && tid == 0) {
            uint64_t k = keys[0];
#pragma unroll
            for (int w = 1; w < 4; ++w) k = k > keys[w] ? k : keys[w];
            if (a.slices > 1u) a.keys[(uint64_t)r * a.slices + slice] = k;
            else a.best[r] = best_token(k);
        }
    }
    if (blockIdx.x == 0 && a.token_offsets) // reported wherever they are, also where no row's search meets them
        for (uint32_t b = threadIdx.x; b < a.batch; b += 256u)
            if (a.token_offsets[b] > a.token_offsets[b + 1u] || a.token_offsets[b + 1u] > a.rows) flag(a.err, kErrSeq);
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

// Work-group = a sequence x a layer: each walks the tree itself (one wave, 64 nodes a step:
// those that continue the kept node with its target's token, the lowest of them) and moves
// its layer's rows; the first layer's writes what belongs to the sequence.  VEC: rows in
// 16-byte pieces.  Bound: the chain offsets -> nodes -> walk -> rows, 2 sequences of 24 layers
// 4.6 us; 64 sequences of 32 layers of 8 x 128 10.6, 43 MB of rows (4 TB/s) behind the same chain.
template <bool VEC>
__global__ __launch_bounds__(256) void accept_kernel(AcceptArgs a) {
    __shared__ int32_t s_parent[kMaxNodes], s_path[kMaxNodes];
    __shared__ uint32_t s_token[kMaxNodes], s_target[kMaxNodes], s_kept;
    const uint32_t tid = threadIdx.x, lane = tid & 63u, b = blockIdx.x, layer = blockIdx.y;
    const SeqRows rows = seq_rows(a.token_offsets, a.tokens, a.batch, b, a.err);
    const uint32_t n = min(rows.n, kMaxNodes);
    const uint32_t count = a.history && layer == 0 ? a.history_count[b] : 0u; // before a barrier: history_count_out may be it
    const int64_t* slots = a.slots ? a.slots + rows.first : nullptr;
    const bool none = slots && lane < n && slots[lane] == kNoSlot; // no page for the node kept lane-th
    for (uint32_t i = tid; i < n; i += 256u) {
        s_parent[i] = a.parents[rows.first + i];
        s_token[i] = a.node_tokens[rows.first + i];
        s_target[i] = a.targets[rows.first + i];
    }
    __syncthreads();
    if (tid < 64u) {
        uint32_t room = n; // nodes that may be kept
        uint64_t m = __ballot(none);
        for (uint32_t c = 0;;) {
            if (m) room = c + (uint32_t)__builtin_ctzll(m);
            c += 64u;
            if (m || c >= n || !slots) break;
            m = __ballot(slots[min(c + lane, n - 1u)] == kNoSlot);
        }
        uint32_t kept = room ? 1u : 0u, cur = 0;
        if (lane == 0) s_path[0] = 0;
        for (uint32_t c = 0; kept < room && c < n;) { // nodes c .. of this step: each pass moves on, or to a later node
            const uint32_t i = c + lane;
            const uint64_t m = __ballot(i < n && i > cur && s_parent[min(i, n - 1u)] == (int32_t)cur &&
                                        s_token[min(i, n - 1u)] == s_target[cur] && s_target[cur] != ~0u);
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
            a.next_token[b] = kept ? (int32_t)s_target[s_path[kept - 1u]] : n ? (int32_t)s_token[0] : -1;
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
