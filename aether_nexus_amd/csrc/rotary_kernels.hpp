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
    float magnitude, eps, inv_hd; // inv_hd = 1 / hd
    // append
    uint32_t batch, hot_count, refs_stride;
    uint64_t hot_blocks;
    const uint32_t *refs, *seq_hot, *token_offsets; // token_offsets null: tokens / batch each
    uint32_t* err;
    // rotary_rows_kernel
    uint32_t slices;    // waves of a token
    uint32_t lanes_log; // log2 of the lanes of a head
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
// the same token; the offsets ascend, so it is found among 64 equal stretches of them at
// a time: a round trip to L2 up to 64 sequences, two up to 4096, four up to 2^24, the
// most that the host lets through.  Offsets that descend end the search as well, at
// some sequence, and a token that is not within its rows is reported below.
__device__ inline Place find_place(const RotaryArgs& a, uint32_t t, uint32_t lane, bool report) {
    uint32_t b, first, end;
    if (a.token_offsets) {
        uint32_t n = a.batch; // the sequences that end at or before t are the first b .. b + n
        b = 0;
        while (n > 64u) {
            const uint32_t stretch = (n + 63u) / 64u, at = (lane + 1u) * stretch - 1u;
            const uint32_t skip = stretch * (uint32_t)__popcll(__ballot(at < n && a.token_offsets[b + min(at, n - 1u) + 1u] <= t));
            b += skip;
            n = min(n - skip, stretch);
        }
        if (n) b += (uint32_t)__popcll(__ballot(lane < n && a.token_offsets[b + min(lane, n - 1u) + 1u] <= t));
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

// 16 bytes at an element's alignment: one access on gfx950.
typedef uint32_t uint4_el_t __attribute__((ext_vector_type(4), aligned(2)));

// Two values rounded to f16, the first in the low half.
__device__ inline uint32_t f2h_pair(float x, float y) {
    typedef float float2_v __attribute__((ext_vector_type(2)));
    typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((float2_v){x, y}, half2_v));
}

// Sum over the 2^log lanes of a head, in each of them: quad permutes and row mirrors up
// to 16 lanes (a mirror meets a lane of the other half, whose lanes hold equal sums).
__device__ inline float lanes_sum(float x, uint32_t log) {
#define AWO_DPP_ADD(n, ctrl) \
    if (log > n) x += __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), ctrl, 0xF, 0xF, false))
    AWO_DPP_ADD(0, 0xB1);  // quad_perm [1,0,3,2]
    AWO_DPP_ADD(1, 0x4E);  // quad_perm [2,3,0,1]
    AWO_DPP_ADD(2, 0x141); // row_half_mirror
    AWO_DPP_ADD(3, 0x140); // row_mirror
#undef AWO_DPP_ADD
    if (log > 4) x += __shfl_xor(x, 16);
    if (log > 5) x += __shfl_xor(x, 32);
    return x;
}

// 16 dims of a head in a lane, as two 16-byte pieces, the heads of a wave's step side by
// side.  A turned lane holds 8 pairs from p0 on: dims p0 .. and rotary_dim / 2 + p0 ..
// (half), or 2 p0 .. 2 p0 + 15 (interleaved), so the same 8 cosines and sines serve every
// head of its token; a passing lane holds dims as they lie.  Where the dims do not
// divide, the last lane starts earlier and makes some values twice, the same bits (`skip`
// keeps them out of the norm's sum).  ODD: fewer than 16 turned dims lie in one lane with
// those behind them, 1 to 7 passing dims are stored one by one (8192 tokens of 32 / 8 heads
// x 128, 10 turned dims 38 us, 122 63 us; in rotary_kernel 93 and 87).  Work-group = 4 waves,
// each a token or a slice of its heads, none waiting for another: a wave works its
// token's cosines and sines out once, a pair a lane, into LDS of its own, while its
// first kStep steps of rows are on the way.
// Bound: HBM, each row read and written once (8192 tokens of 32 / 8 heads x 128, 168 MB:
// 33 us, 5.0 TB/s, the rate of a large copy); a token or two: the launch.
// Dims of a head that the turned lanes hold: rotary_dim, or 16 where it is less.
__host__ __device__ inline uint32_t rotary_turn_dims(uint32_t n) { return n ? (n < 16u ? 16u : n) : 0u; }
__host__ __device__ inline bool rotary_rows_odd(uint32_t hd, uint32_t n) {
    return rotary_turn_dims(n) != n || (hd > n && hd - rotary_turn_dims(n) < 8u);
}
// Lanes of a head that hold turned dims, passing ones.
__host__ __device__ inline uint32_t rotary_turn_lanes(uint32_t n) { return (n + 15u) / 16u; }
__host__ __device__ inline uint32_t rotary_pass_lanes(uint32_t hd, uint32_t n) { return (hd - rotary_turn_dims(n) + 15u) / 16u; }
// Heads of at least 16 dims (8 where none turn) that the lanes of a wave hold.
__host__ __device__ inline bool rotary_rows_take(uint32_t hd, uint32_t n) {
    return hd >= 8u && hd >= rotary_turn_dims(n) && rotary_turn_lanes(n) + rotary_pass_lanes(hd, n) <= 64u;
}

// The pairs (p, p + H) of the 16 dims of a lane.
template <int H>
__device__ __forceinline__ void turn_few(float (&f)[16], const float (&c)[8], const float (&sn)[8]) {
#pragma unroll
    for (int p = 0; p < H; ++p) {
        const float x = f[p], y = f[p + H];
        f[p] = fmaf(x, c[p], -(y * sn[p]));
        f[p + H] = fmaf(x, sn[p], y * c[p]);
    }
}

template <bool APPEND, bool NORM, bool INTER, bool ODD>
__global__ __launch_bounds__(256) void rotary_rows_kernel(RotaryArgs a) {
    // Steps whose rows are loaded together.  Measured, us, 1 and 2, heads of 128 dims: 6000
    // tokens of 12 / 2 heads with norms 9.6, 10.9; 6147 tokens of 32 / 8 heads appended with
    // norms 36.7, 35.1; 8192 tokens of those turned alone 34.6, 34.1; 3, 4 and 6 no better.  (ODD: 2
    // would take 180 registers.)
    constexpr int kStep = ODD || (NORM && !APPEND) ? 1 : 2;
    __shared__ float2 s_turns[4][kRotaryMaxDim / 2];
    const uint32_t lane = threadIdx.x & 63u, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t id = blockIdx.x * 4u + wave; // below 2^26
    const uint32_t t = (uint32_t)__builtin_amdgcn_readfirstlane((int)(id / a.slices)), slice = id - t * a.slices;
    if (t >= a.tokens) return; // no barrier follows
    const uint32_t n = a.rotary_dim, half = n / 2, hd = a.hd;
    const uint32_t u = lane & ((1u << a.lanes_log) - 1u), slot = lane >> a.lanes_log, per = 64u >> a.lanes_log;
    const uint32_t turn_lanes = rotary_turn_lanes(n), unit = u - turn_lanes;
    const bool turning = u < turn_lanes, used = u < turn_lanes + rotary_pass_lanes(hd, n);
    const uint32_t m = ODD ? rotary_turn_dims(n) : n;
    const bool few = ODD && m != n;                 // the turned dims lie in one lane, as they lie
    const bool tail = ODD && hd - m < 8u && hd > m; // 1 to 7 passing dims
    uint32_t at0, at1, p0 = 0, skip0, skip1; // dims of the pieces, leading values that another lane holds too
    if (few && turning) {
        at0 = skip0 = skip1 = 0;
        at1 = 8;
    } else if (turning) {
        p0 = min(8u * u, half - 8u);
        at0 = INTER ? 2u * p0 : p0;
        at1 = INTER ? 2u * p0 + 8u : half + p0;
        const uint32_t twice = 8u * u - p0; // pairs
        skip0 = INTER ? min(2u * twice, 8u) : twice;
        skip1 = INTER ? 2u * twice - skip0 : twice;
    } else {
        const uint32_t d = m + 16u * unit;
        at0 = min(d, hd - 8u);
        at1 = min(d + 8u, hd - 8u);
        skip0 = d - at0;
        skip1 = d + 8u - at1;
    }
    const bool whole = m % 16u == 0u && (hd - m) % 16u == 0u; // no value is held twice
    const uint32_t heads = a.q_heads + a.kv_heads + (APPEND && a.v_out ? a.kv_heads : 0u);
    const uint32_t steps = (heads + per - 1u) / per;
    const uint32_t s1 = (uint32_t)((uint64_t)steps * (slice + 1u) / a.slices);
    uint32_t s = (uint32_t)((uint64_t)steps * slice / a.slices);
    uint4_el_t x0[kStep] = {}, x1[kStep] = {}; // zeros where a lane has no dims
    auto load = [&] {
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
            const uint32_t h = (s + (uint32_t)j) * per + slot;
            if (s + (uint32_t)j >= s1 || h >= heads || !used) continue;
            const bool is_q = h < a.q_heads, is_v = APPEND && h >= a.q_heads + a.kv_heads;
            const uint16_t* p = is_q ? a.q + t * a.q_stride + (uint64_t)h * hd
                                     : (is_v ? a.v + t * a.v_stride + (uint64_t)(h - a.q_heads - a.kv_heads) * hd
                                             : a.k + t * a.k_stride + (uint64_t)(h - a.q_heads) * hd);
            x0[j] = *(const uint4_el_t*)(p + at0);
            x1[j] = *(const uint4_el_t*)(p + at1);
        }
    };
    load();
    uint4_el_t w0[2] = {}, w1[2] = {}; // weights of q, of k
    if constexpr (NORM) {
        if (used && a.q_norm) {
            w0[0] = *(const uint4_el_t*)(a.q_norm + at0);
            w1[0] = *(const uint4_el_t*)(a.q_norm + at1);
        }
        if (used && a.k_norm) {
            w0[1] = *(const uint4_el_t*)(a.k_norm + at0);
            w1[1] = *(const uint4_el_t*)(a.k_norm + at1);
        }
    }
    Place place{true, true, t, 0};
    if constexpr (APPEND) place = find_place(a, t, lane, slice == 0);
    if (!place.rows) return;
    float c[8], sn[8];
    if (n) {
        const uint32_t position = a.positions ? a.positions[t] : a.start + place.at;
        for (uint32_t p = lane; p < half; p += 64u) s_turns[wave][p] = turn_of(a, p, position);
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float2 cs = s_turns[wave][p0 + (uint32_t)e]; // p0 = 0 in passing lanes
            c[e] = cs.x;
            sn[e] = cs.y;
        }
    }
    auto half_of = [](const uint4_el_t& v, int e) { return (uint16_t)(v[e / 2] >> (16 * (e % 2))); };
    for (;;) {
#pragma unroll
        for (int j = 0; j < kStep; ++j) {
            if (s + (uint32_t)j >= s1) break; // wave-uniform
            const uint32_t h = (s + (uint32_t)j) * per + slot;
            const bool is_q = h < a.q_heads, is_v = APPEND && h >= a.q_heads + a.kv_heads;
            const bool normed = NORM && !is_v && (is_q ? a.q_norm != nullptr : a.k_norm != nullptr);
            float f0[8], f1[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                f0[e] = h2f(half_of(x0[j], e));
                f1[e] = h2f(half_of(x1[j], e));
            }
            if constexpr (NORM) {
                float sum = 0.0f;
                if (whole) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum = fmaf(f1[e], f1[e], fmaf(f0[e], f0[e], sum));
                } else {
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        sum = (uint32_t)e >= skip0 ? fmaf(f0[e], f0[e], sum) : sum;
                        sum = (uint32_t)e >= skip1 ? fmaf(f1[e], f1[e], sum) : sum;
                    }
                }
                sum = lanes_sum(sum, a.lanes_log);
                if (normed) {
                    const float inv = rsqrtf(fmaf(sum, a.inv_hd, a.eps));
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        f0[e] = f0[e] * inv * h2f(half_of(is_q ? w0[0] : w0[1], e));
                        f1[e] = f1[e] * inv * h2f(half_of(is_q ? w1[0] : w1[1], e));
                    }
                }
            }
            if (h >= heads || !used) continue;
            uint16_t* y;
            if (is_q) {
                y = a.q_out + t * a.q_out_stride + (uint64_t)h * hd;
            } else if constexpr (APPEND) {
                if (!place.page) continue;
                y = is_v ? a.v_out + (place.row * a.kv_heads + (h - a.q_heads - a.kv_heads)) * hd
                         : a.k_out + (place.row * a.kv_heads + (h - a.q_heads)) * hd;
            } else {
                y = a.k_out + t * a.k_out_stride + (uint64_t)(h - a.q_heads) * hd;
            }
            uint4_el_t r0 = x0[j], r1 = x1[j];
            const bool turn = turning && !is_v;
            if (turn) {
                float g0[8], g1[8];
                if (ODD && few && !INTER) {
                    float f[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) f[e] = e < 8 ? f0[e] : f1[e - 8];
                    switch (half) { // wave-uniform
                    case 1: turn_few<1>(f, c, sn); break;
                    case 2: turn_few<2>(f, c, sn); break;
                    case 3: turn_few<3>(f, c, sn); break;
                    case 4: turn_few<4>(f, c, sn); break;
                    case 5: turn_few<5>(f, c, sn); break;
                    case 6: turn_few<6>(f, c, sn); break;
                    default: turn_few<7>(f, c, sn); break;
                    }
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        g0[e] = f[e];
                        g1[e] = f[e + 8];
                    }
                } else
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    if constexpr (INTER) { // pairs of neighbours: e and e + 1 of one piece
                        float(&f)[8] = e < 4 ? f0 : f1;
                        float(&g)[8] = e < 4 ? g0 : g1;
                        const int i = 2 * (e % 4);
                        if (few && (uint32_t)e >= half) { // these pass
                            g[i] = f[i];
                            g[i + 1] = f[i + 1];
                            continue;
                        }
                        g[i] = fmaf(f[i], c[e], -(f[i + 1] * sn[e]));
                        g[i + 1] = fmaf(f[i], sn[e], f[i + 1] * c[e]);
                    } else {
                        g0[e] = fmaf(f0[e], c[e], -(f1[e] * sn[e]));
                        g1[e] = fmaf(f0[e], sn[e], f1[e] * c[e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    f0[e] = g0[e];
                    f1[e] = g1[e];
                }
            }
            if (turn || normed) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    r0[i] = f2h_pair(f0[2 * i], f0[2 * i + 1]);
                    r1[i] = f2h_pair(f1[2 * i], f1[2 * i + 1]);
                    if (few && !normed) { // dims that pass keep their bits
                        if (2u * (uint32_t)i >= n) r0[i] = x0[j][i];
                        if (2u * (uint32_t)i + 8u >= n) r1[i] = x1[j][i];
                    }
                }
            }
            if (tail && !turning) { // its other dims are the turned lanes'
#pragma unroll
                for (int e = 1; e < 8; ++e)
                    if ((uint32_t)e >= skip0) y[at0 + (uint32_t)e] = half_of(r0, e);
                continue;
            }
            *(uint4_el_t*)(y + at0) = r0;
            *(uint4_el_t*)(y + at1) = r1;
        }
        s += (uint32_t)kStep;
        if (s >= s1) return;
        load();
    }
}

// The other heads (of fewer than 16 dims, of 65 lanes): work-group = one token, a wave per head in
// turn, lanes over the pairs and then over the dims that pass.  Tokens past a grid row's
// kRotaryGridRow go to further rows: a row of 2^24 work-groups would be 2^32 threads, one
// more than a launch takes.
constexpr uint32_t kRotaryGridRow = 1u << 20;
template <bool APPEND>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
    __shared__ float2 s_turn[kRotaryMaxDim / 2];
    const uint32_t t = blockIdx.y * kRotaryGridRow + blockIdx.x, tid = threadIdx.x, lane = tid & 63u, wave = tid >> 6;
    if (t >= a.tokens) return; // the whole work-group
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
            inv = rsqrtf(fmaf(sum, a.inv_hd, a.eps));
        }
        auto value = [&](uint32_t d) { return w ? h2f(x[d]) * inv * h2f(w[d]) : h2f(x[d]); };
        for (uint32_t p = lane; p < half; p += 64u) {
            const uint32_t d0 = a.interleaved ? 2u * p : p, d1 = a.interleaved ? 2u * p + 1u : p + half;
            const float x0 = value(d0), x1 = value(d1);
            const float2 cs = s_turn[p];
            y[d0] = f2h(fmaf(x0, cs.x, -(x1 * cs.y)));
            y[d1] = f2h(fmaf(x0, cs.y, x1 * cs.x));
        }
        for (uint32_t d = a.rotary_dim + lane; d < a.hd; d += 64u) y[d] = w ? f2h(value(d)) : x[d];
    }
}

} // namespace awo
