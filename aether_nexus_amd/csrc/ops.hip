// ops.hip — C ABI of the dense transformer ops (include/aether_ops.h).
//
// Replaces the dispatch methods of the reference's Ops engine
// (nexus-core/src/ops.rs:166-462); the kernels are in ops_kernels.hpp.  Beside them the
// rows of a batch over pages, which the reference does not have: rotary positions, head
// norms and appends (rotary_kernels.hpp), and a step over trees of drafted tokens: tables,
// logits, acceptance (step_kernels.hpp).  Every entry point validates its arguments on
// the host, picks the 16-byte vector variant of a kernel when the pointers and sizes allow
// it, and enqueues on the caller's stream.  There is no CPU fallback.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <tuple>
#include <type_traits>

#include "../../include/aether_ops.h"
#include "engine_internal.hpp"
#include "gemm_kernels.hpp"
#include "ops_kernels.hpp"
#include "rotary_kernels.hpp"
#include "step_kernels.hpp"

namespace {

namespace ei = aw_engine_internal;
using ei::Rows;
using ei::rows_meet;
using ei::rows_same;

uint64_t cdiv64(uint64_t a, uint64_t b) { return (a + b - 1) / b; }
bool aligned(const void* p, uintptr_t a) { return ((uintptr_t)p & (a - 1)) == 0; }

#define OPS_HIP(e, call)                                                                        \
    do {                                                                                        \
        const hipError_t err_ = (call);                                                         \
        if (err_ != hipSuccess) return ei::fail(e, AW_E_HIP, "%s: %s", #call, hipGetErrorString(err_)); \
    } while (0)

int enter(aw_engine* e) {
    if (!e) return AW_E_INVALID_ARG;
    OPS_HIP(e, hipSetDevice(ei::device(e)));
    return AW_OK;
}

// Grid of an HBM-bound grid-strided kernel: enough work-groups for `units`
// threads' worth of work, at most 16 per CU.
uint32_t stream_grid(aw_engine* e, uint64_t units) {
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(cdiv64(units, 256), (uint64_t)ei::compute_units(e) * 16));
}

template <awo::Ew OP>
int launch_ew(aw_engine* e, const awo::EwArgs& p, bool vec, hipStream_t st) {
    if (p.n == 0) return AW_OK;
    const uint32_t grid = stream_grid(e, vec ? std::max<uint64_t>(p.n / 8, 1) : p.n);
    if (vec)
        hipLaunchKernelGGL((awo::ew_kernel<OP, true>), dim3(grid), dim3(256), 0, st, p);
    else
        hipLaunchKernelGGL((awo::ew_kernel<OP, false>), dim3(grid), dim3(256), 0, st, p);
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

// One weight matrix of a product: B [n][k] (and B2, the up weights of a fused
// SiLU gate), output C [m][n].
struct Product {
    const uint16_t* b;
    const uint16_t* b2;
    void* c;
    uint32_t n;
};

// The tiles of a product of more than 64 rows.
using GemmTiles = std::tuple<awo::GemmTile<4, 2, 4, 8, 2, 3>, awo::GemmTile<4, 2, 4, 5, 3>, awo::GemmTile<4, 2, 4, 4, 3>,
                             awo::GemmTile<4, 2, 2, 4, 3>, awo::GemmTile<4, 2, 2, 2, 3>, awo::GemmTile<4, 2, 1, 3, 4>,
                             awo::GemmTile<4, 2, 1, 2, 4>, awo::GemmTile<2, 2, 2, 1, 6>>;

// f(T{}) for each tile.
template <typename F>
void each_tile(F f) {
    std::apply([&](auto... t) { (f(t), ...); }, GemmTiles{});
}

// Tiles of all groups.
template <typename T>
uint64_t tile_count(const awo::GemmArgs& g) {
    uint64_t n = 0;
    for (uint32_t i = 0; i < g.groups; ++i) n += cdiv64(g.g[i].N, T::TN);
    return n * cdiv64(g.M, T::TM);
}

// Estimated time (us) of a product on tile T, fitted to this GPU (M 72 .. 2048, N 896
// .. 14336, K 896 .. 14336; the estimate's choice is within 10% of the fastest tile).
// A 64-k stage takes a CU 2.2 ns per staged row (its loads, 58 bytes a ns), 1.9 with
// two work-groups on it, or, with every CU busy, its products at 1.25 PFLOP/s (the
// power limit); a tile starts and stores in 1.5 us and 15 halves a ns.  Measured, us:
// 2048 x 14336 x 4096 256 x 256 tiles 222, 256 x 128 259; 2048 x 4096 x 14336 256 x
// 128 217, 256 x 256 256; 512 x 4096 x 14336 128 x 64 95, 64 x 64 114, 128 x 128
// 129; 117 x 3072 x 2048 64 x 32 8.3, 64 x 64 8.9, 128 x 64 11.3.
template <typename T>
double tile_us(const awo::GemmArgs& g, uint32_t n_cu) {
    const uint64_t tiles = tile_count<T>(g), rounds = cdiv64(tiles, n_cu);
    const double per_row = rounds > 1 && T::kLdsBytes <= 80 * 1024 ? 1.9e-3 : 2.2e-3;
    const double area = (double)T::TM * T::TN, busy = (double)tiles / ((double)rounds * n_cu);
    const double stage = std::max(per_row * (T::TM + T::TN), 2.6e-5 * area * busy);
    return (double)rounds * ((double)cdiv64(g.K, awo::kStageK) * stage + 1.5 + area / 15e3);
}

// f(T{}) for the tile of the least estimate; false where no tile's grid fits.
template <typename F>
bool with_tile(const awo::GemmArgs& g, uint32_t n_cu, F f) {
    double best = 0.0;
    int pick = -1, i = 0;
    each_tile([&](auto t) {
        using T = decltype(t);
        const double us = tile_us<T>(g, n_cu);
        if (tile_count<T>(g) <= 0x7FFFFFFFull && (pick < 0 || us < best)) {
            best = us;
            pick = i;
        }
        ++i;
    });
    i = 0;
    each_tile([&](auto t) {
        if (i++ == pick) f(t);
    });
    return pick >= 0;
}

template <typename T, bool F32, awo::Epi EPI>
void launch_tile(const awo::GemmArgs& a, hipStream_t st) {
    awo::GemmArgs g = a;
    for (uint32_t i = 0; i < g.groups; ++i) g.g[i].tiles = (uint32_t)cdiv64(g.g[i].N, T::TN);
    hipLaunchKernelGGL((awo::gemm_tile_kernel<T, F32, EPI>), dim3((uint32_t)tile_count<T>(g)), dim3(T::kThreads),
                       T::kLdsBytes, st, g);
}

// The products `p[0 .. np)` over the same activations a [m][k], one launch when
// m <= 64 (skinny) or on gemm_tile_kernel, one launch each otherwise.  EPI picks the
// store; F32 the scaled fp32 output of matmul_scaled.
template <awo::Epi EPI, bool F32>
int launch_products(aw_engine* e, const char* what, const uint16_t* a, const Product* p, int np, uint32_t m,
                    uint32_t k, float scale, hipStream_t st) {
    if (m == 0) return AW_OK;
    if (!a) return ei::fail(e, AW_E_INVALID_ARG, "%s: null pointer", what);
    awo::GemmArgs g{};
    g.A = a;
    g.M = m;
    g.K = k;
    g.scale = scale;
    bool vec = k % 8 == 0 && aligned(a, 16);
    uint64_t tiles = 0;
    for (int i = 0; i < np; ++i) {
        if (!p[i].b || !p[i].c || (EPI == awo::Epi::SiluGate && !p[i].b2))
            return ei::fail(e, AW_E_INVALID_ARG, "%s: null pointer", what);
        vec = vec && aligned(p[i].b, 16) && (EPI != awo::Epi::SiluGate || aligned(p[i].b2, 16));
        g.g[g.groups].B = p[i].b;
        g.g[g.groups].B2 = p[i].b2;
        g.g[g.groups].C = p[i].c;
        g.g[g.groups].N = p[i].n;
        g.g[g.groups].tiles = (uint32_t)cdiv64(p[i].n, 16);
        g.g[g.groups].vec_out = p[i].n % 4 == 0 && aligned(p[i].c, F32 ? 16 : 8);
        tiles += cdiv64(p[i].n, 16);
        if (p[i].n) ++g.groups; // empty products drop out
    }
    if (!g.groups) return AW_OK;
    if (m > 64) {
        if (EPI == awo::Epi::SiluGate)
            return ei::fail(e, AW_E_UNSUPPORTED, "%s: m = %u rows (the fused gate takes m <= 64; use matmul and "
                                                 "silu_gate)", what, m);
        if (cdiv64(m, awo::kTileM) > 65535u)
            return ei::fail(e, AW_E_UNSUPPORTED, "%s: m = %u rows exceed the grid", what, m);
        if constexpr (EPI != awo::Epi::SiluGate) {
            // 16-byte rows, a tile's rows below the buffer loads' limit.
            if (vec && (uint64_t)k * 512 <= awo::kTileBytesMax) {
                if (!with_tile(g, ei::compute_units(e), [&](auto t) { launch_tile<decltype(t), F32, EPI>(g, st); }))
                    return ei::fail(e, AW_E_UNSUPPORTED, "%s: grid too large", what);
            } else {
                for (uint32_t i = 0; i < g.groups; ++i) { // one launch per product, group 0 of its own arguments
                    awo::GemmArgs t = g;
                    t.g[0] = g.g[i];
                    t.groups = 1;
                    const dim3 grid((uint32_t)cdiv64(t.g[0].N, awo::kTileN), (uint32_t)cdiv64(m, awo::kTileM));
                    if (vec)
                        hipLaunchKernelGGL((awo::gemm_tiled_kernel<true, F32, EPI>), grid, dim3(256), 0, st, t);
                    else
                        hipLaunchKernelGGL((awo::gemm_tiled_kernel<false, F32, EPI>), grid, dim3(256), 0, st, t);
                }
            }
        }
        OPS_HIP(e, hipGetLastError());
        return AW_OK;
    }
    if (tiles > 0x7FFFFFFFull) return ei::fail(e, AW_E_UNSUPPORTED, "%s: grid too large", what);
    const dim3 grid((uint32_t)tiles);
    // Few weight tiles (up to 4 work-groups per CU): 16 waves per tile, so a K of
    // 4096 is in flight at once; many tiles: 8 waves, more work-groups resident
    // (measured at M = 1: 4096 x 4096 10.8 -> 9.6 us, 14336 x 4096 33.1 -> 28.6 us
    // with 16 waves; 128256 x 4096 183 us with 8 waves, 214 with 16).  The wave
    // count does not change the sums.
    const bool wide = tiles <= 4ull * ei::compute_units(e);
#define AW_SKINNY(MT, NW)                                                                                        \
    do {                                                                                                         \
        if (vec)                                                                                                 \
            hipLaunchKernelGGL((awo::gemm_skinny_kernel<MT, NW, true, F32, EPI>), grid, dim3(NW * 64), 0, st, g);  \
        else                                                                                                     \
            hipLaunchKernelGGL((awo::gemm_skinny_kernel<MT, NW, false, F32, EPI>), grid, dim3(NW * 64), 0, st, g); \
    } while (0)
    if (m <= 16 && wide)
        AW_SKINNY(1, 16);
    else if (m <= 16)
        AW_SKINNY(1, 8);
    else if (m <= 32 && wide)
        AW_SKINNY(2, 16);
    else if (m <= 32)
        AW_SKINNY(2, 8);
    else
        AW_SKINNY(4, 8);
#undef AW_SKINNY
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

int refuse(char* msg, size_t len, int code, const char* fmt, ...) __attribute__((format(printf, 4, 5)));
int refuse(char* msg, size_t len, int code, const char* fmt, ...) {
    if (msg && len) {
        va_list ap;
        va_start(ap, fmt);
        vsnprintf(msg, len, fmt, ap);
        va_end(ap);
    }
    return code;
}

// Waves per CU that a token's heads are cut for.  Measured, us, 4, 8, 16, of 32 / 8 heads x
// 128: 1024 tokens appended with norms 6.85, 6.32, 6.08; 2048 turned 9.06, 9.06, 8.67; 509
// tokens 4.2 each.
constexpr uint64_t kRotaryWaves = 16;
constexpr uint32_t kMostTokens = 1u << 24; // waves of a call, and threads of a grid's row, stay below 2^32
constexpr uint32_t kMostSequences = 1u << 24; // of an append: a search of its offsets in four steps, in 32 bits
constexpr uint64_t kMostStride = 1ull << 30; // elements: tokens * stride * 2 bytes stays below 2^63

// The checks that the three rotary calls share, and their kernel arguments.
int rotary_args(const char* what, const aw_rotary_desc* d, bool append, awo::RotaryArgs* out, char* msg, size_t len) {
    auto bad = [&](const char* why) { return refuse(msg, len, AW_E_INVALID_ARG, "%s: %s", what, why); };
    if (d->reserved) return bad("reserved must be 0");
    if (d->head_dim == 0) return bad("head_dim is 0");
    if (d->head_dim > awo::kRotaryMaxDim)
        return refuse(msg, len, AW_E_UNSUPPORTED, "%s: head_dim %u exceeds %u", what, d->head_dim, awo::kRotaryMaxDim);
    if (d->rotary_dim % 2 || d->rotary_dim > d->head_dim)
        return refuse(msg, len, AW_E_INVALID_ARG, "%s: rotary_dim %u must be even and at most head_dim %u", what,
                      d->rotary_dim, d->head_dim);
    if (d->layout != AW_ROTARY_HALF && d->layout != AW_ROTARY_INTERLEAVED)
        return refuse(msg, len, AW_E_INVALID_ARG, "%s: layout %u", what, d->layout);
    if (d->rotary_dim && !d->inv_freq) return bad("inv_freq is required");
    if (d->rotary_dim && !std::isfinite(d->magnitude)) return bad("magnitude must be finite");
    if ((d->q_norm || d->k_norm) && !(d->eps >= 0.0f && std::isfinite(d->eps))) return bad("eps must be finite and not negative");
    if (d->num_tokens && ((d->q_heads && (!d->q || !d->q_out)) || (d->kv_heads && (!d->k || (!append && !d->k_out)))))
        return bad("null pointer");
    if (d->num_tokens > kMostTokens || d->q_heads > 0xFFFFu || d->kv_heads > 0xFFFFu)
        return refuse(msg, len, AW_E_UNSUPPORTED, "%s: too many tokens or heads", what);
    awo::RotaryArgs& a = *out;
    a = awo::RotaryArgs{};
    const uint64_t q_row = (uint64_t)d->q_heads * d->head_dim, k_row = (uint64_t)d->kv_heads * d->head_dim;
    a.q_stride = d->q_stride ? d->q_stride : q_row;
    a.q_out_stride = d->q_out_stride ? d->q_out_stride : q_row;
    a.k_stride = d->k_stride ? d->k_stride : k_row;
    a.k_out_stride = d->k_out_stride ? d->k_out_stride : k_row;
    if (a.q_stride < q_row || a.q_out_stride < q_row || a.k_stride < k_row || a.k_out_stride < k_row)
        return bad("a stride is shorter than a token's heads");
    if (std::max(std::max(a.q_stride, a.q_out_stride), std::max(a.k_stride, a.k_out_stride)) > kMostStride)
        return refuse(msg, len, AW_E_UNSUPPORTED, "%s: a stride exceeds 2^30 elements", what);
    const Rows q{d->q, a.q_stride, q_row, d->num_tokens}, q_out{d->q_out, a.q_out_stride, q_row, d->num_tokens};
    const Rows k{d->k, a.k_stride, k_row, d->num_tokens}, k_out{append ? nullptr : d->k_out, a.k_out_stride, k_row, d->num_tokens};
    if ((!rows_same(q, q_out) && rows_meet(q, q_out)) || (!rows_same(k, k_out) && rows_meet(k, k_out)))
        return bad("the output overlaps its input, and is not the input itself");
    if (rows_meet(q, k_out) || rows_meet(k, q_out) || rows_meet(q_out, k_out)) return bad("rows of q and k overlap, and one is an output");
    a.q = d->q;
    a.k = d->k;
    a.q_out = d->q_out;
    a.k_out = d->k_out;
    a.q_norm = d->q_norm;
    a.k_norm = d->k_norm;
    a.positions = d->positions;
    a.inv_freq = d->inv_freq;
    a.tokens = d->num_tokens;
    a.q_heads = d->q_heads;
    a.kv_heads = d->kv_heads;
    a.hd = d->head_dim;
    a.rotary_dim = d->rotary_dim;
    a.interleaved = d->layout == AW_ROTARY_INTERLEAVED ? 1u : 0u;
    a.start = d->start_position;
    a.magnitude = d->magnitude;
    a.eps = d->eps;
    a.inv_hd = 1.0f / (float)d->head_dim;
    return AW_OK;
}

// aw_ops_rotary (norms false) and aw_ops_qk_norm_rotary.
int rows_args(const aw_rotary_desc* d, bool norms, awo::RotaryArgs* a, char* msg, size_t len) {
    const char* what = norms ? "qk_norm_rotary" : "rotary";
    if (!d) return refuse(msg, len, AW_E_INVALID_ARG, "%s: null descriptor", what);
    if (!norms && (d->q_norm || d->k_norm))
        return refuse(msg, len, AW_E_INVALID_ARG, "rotary: norm weights given (qk_norm_rotary takes them)");
    if (!norms && d->rotary_dim == 0) return refuse(msg, len, AW_E_INVALID_ARG, "rotary: rotary_dim is 0");
    if (norms && ((d->q_heads && !d->q_norm) || (d->kv_heads && !d->k_norm)))
        return refuse(msg, len, AW_E_INVALID_ARG, "qk_norm_rotary: norm weights are required");
    return rotary_args(what, d, false, a, msg, len);
}

int append_args(const aw_append_desc* d, awo::RotaryArgs* a, char* msg, size_t len) {
    auto bad = [&](const char* why) { return refuse(msg, len, AW_E_INVALID_ARG, "append_paged: %s", why); };
    if (!d) return bad("null descriptor");
    if (int rc = rotary_args("append_paged", &d->rows, true, a, msg, len)) return rc;
    if (d->reserved) return bad("reserved must be 0");
    if (d->rows.kv_heads == 0) return bad("kv_heads is 0");
    if (d->rows.k_out) return bad("k_out must be NULL (k goes to hot_k)");
    if (d->v && !d->hot_v) return bad("v given without hot_v");
    if (!d->hot_k || (d->rows.num_tokens && (d->hot_v && !d->v)) || (d->rows.num_tokens && d->batch && (!d->refs || !d->seq_hot)))
        return bad("null pointer");
    if (d->hot_blocks == 0 || d->hot_count == 0) return bad("hot_blocks and hot_count must be >= 1");
    if (d->hot_blocks > 1ull << 31) return bad("hot_blocks exceeds 2^31, the refs' range");
    if (d->refs_stride < d->hot_count)
        return refuse(msg, len, AW_E_INVALID_ARG, "append_paged: refs_stride %u < hot_count %u", d->refs_stride, d->hot_count);
    if (d->batch > kMostSequences) return refuse(msg, len, AW_E_UNSUPPORTED, "append_paged: batch %u exceeds 2^24", d->batch);
    if (!d->token_offsets && d->batch && d->rows.num_tokens % d->batch)
        return refuse(msg, len, AW_E_INVALID_ARG, "append_paged: %u tokens over %u sequences need token_offsets",
                      d->rows.num_tokens, d->batch);
    const uint64_t row = (uint64_t)d->rows.kv_heads * d->rows.head_dim;
    a->v_stride = d->v_stride ? d->v_stride : row;
    if (a->v_stride < row) return bad("a stride is shorter than a token's heads");
    if (a->v_stride > kMostStride) return refuse(msg, len, AW_E_UNSUPPORTED, "append_paged: a stride exceeds 2^30 elements");
    const uint64_t pool = d->hot_blocks * awo::kPageTokens * row, n = d->rows.num_tokens;
    const Rows hot[2] = {{d->hot_k, pool, pool, 1}, {d->hot_v, pool, pool, 1}}, v{d->v, a->v_stride, row, n};
    const Rows q{d->rows.q, a->q_stride, (uint64_t)a->q_heads * a->hd, n}, q_out{d->rows.q_out, a->q_out_stride, q.row, n};
    const Rows k{d->rows.k, a->k_stride, row, n};
    if (rows_meet(q_out, v)) return bad("rows of q_out and v overlap");
    for (const Rows& h : hot)
        if (rows_meet(h, q) || rows_meet(h, q_out) || rows_meet(h, k) || rows_meet(h, v)) return bad("a pool overlaps the rows");
    if (rows_meet(hot[0], hot[1])) return bad("hot_k and hot_v overlap");
    a->v = d->v;
    a->k_out = d->hot_k;
    a->v_out = d->hot_v;
    a->batch = d->batch;
    a->hot_count = d->hot_count;
    a->refs_stride = d->refs_stride;
    a->hot_blocks = d->hot_blocks;
    a->refs = d->refs;
    a->seq_hot = d->seq_hot;
    a->token_offsets = d->token_offsets;
    return AW_OK;
}

template <bool APPEND>
int launch_rotary(aw_engine* e, awo::RotaryArgs& a, hipStream_t st) {
    a.err = ei::error_word(e);
    if (!awo::rotary_rows_take(a.hd, a.rotary_dim)) {
        const dim3 tokens(std::min(a.tokens, awo::kRotaryGridRow), (uint32_t)cdiv64(a.tokens, awo::kRotaryGridRow));
        hipLaunchKernelGGL(awo::rotary_kernel<APPEND>, tokens, dim3(256), 0, st, a);
        OPS_HIP(e, hipGetLastError());
        return AW_OK;
    }
    const uint32_t lanes = awo::rotary_turn_lanes(a.rotary_dim) + awo::rotary_pass_lanes(a.hd, a.rotary_dim);
    while ((1u << a.lanes_log) < lanes) ++a.lanes_log;
    const uint32_t heads = a.q_heads + a.kv_heads + (APPEND && a.v_out ? a.kv_heads : 0u);
    const uint64_t steps = cdiv64(heads, 64u >> a.lanes_log);
    // Few tokens: a token's heads over several waves.
    a.slices = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(steps, cdiv64(kRotaryWaves * (uint64_t)ei::compute_units(e), a.tokens)));
    const dim3 grid((uint32_t)cdiv64((uint64_t)a.tokens * a.slices, 4)), block(256);
    auto launch = [&](auto norm, auto inter, auto odd) {
        hipLaunchKernelGGL((awo::rotary_rows_kernel<APPEND, decltype(norm)::value, decltype(inter)::value, decltype(odd)::value>),
                           grid, block, 0, st, a);
    };
    auto odd = [&](auto norm, auto inter) {
        if (awo::rotary_rows_odd(a.hd, a.rotary_dim)) launch(norm, inter, std::true_type{});
        else launch(norm, inter, std::false_type{});
    };
    auto inter = [&](auto norm) {
        if (a.interleaved) odd(norm, std::true_type{});
        else odd(norm, std::false_type{});
    };
    if (a.q_norm || a.k_norm) inter(std::true_type{});
    else inter(std::false_type{});
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

// A stretch of memory that a call reads or writes.
struct Span {
    const void* at;
    uint64_t bytes;
};
bool spans_meet(const Span& p, const Span& o) {
    const uintptr_t x = (uintptr_t)p.at, y = (uintptr_t)o.at;
    return p.at && o.at && p.bytes && o.bytes && x < y + o.bytes && y < x + p.bytes;
}
// Whether an output meets an input or another output.
template <size_t N, size_t M>
bool outputs_meet(const Span (&out)[N], const Span (&in)[M]) {
    for (size_t i = 0; i < N; ++i) {
        for (size_t j = 0; j < i; ++j)
            if (spans_meet(out[i], out[j])) return true;
        for (const Span& x : in)
            if (spans_meet(out[i], x)) return true;
    }
    return false;
}

constexpr uint32_t kMostStepSequences = 1u << 20;

// What the three calls of a step ask of their rows; `what` begins the text.
int step_rows(const char* what, uint32_t batch, uint32_t tokens, const void* offsets, bool divide, char* msg, size_t len) {
    if (tokens > kMostTokens) return refuse(msg, len, AW_E_UNSUPPORTED, "%s: num_tokens %u exceeds 2^24", what, tokens);
    if (batch > kMostStepSequences) return refuse(msg, len, AW_E_UNSUPPORTED, "%s: batch %u exceeds 2^20", what, batch);
    if (divide && !offsets && batch && tokens % batch)
        return refuse(msg, len, AW_E_INVALID_ARG, "%s: %u tokens over %u sequences need token_offsets", what, tokens, batch);
    return AW_OK;
}

int tables_args(const aw_tables_desc* d, awo::TablesArgs* a, char* msg, size_t len) {
    auto bad = [&](const char* why) { return refuse(msg, len, AW_E_INVALID_ARG, "page_tables: %s", why); };
    if (!d) return bad("null descriptor");
    if (int rc = step_rows("page_tables", d->batch, d->num_tokens, nullptr, false, msg, len)) return rc;
    if (d->hot_count > 1u << 26) return refuse(msg, len, AW_E_UNSUPPORTED, "page_tables: hot_count %u exceeds 2^26", d->hot_count);
    if (d->refs_stride < d->hot_count)
        return refuse(msg, len, AW_E_INVALID_ARG, "page_tables: refs_stride %u < hot_count %u", d->refs_stride, d->hot_count);
    if (d->free_count > 1u << 30) return refuse(msg, len, AW_E_UNSUPPORTED, "page_tables: free_count %u exceeds 2^30", d->free_count);
    if (d->mask_words > AW_MAX_NODES / 32) return refuse(msg, len, AW_E_UNSUPPORTED, "page_tables: mask_words %u exceeds 32", d->mask_words);
    // Rows (and below lists) of no elements have no address.
    if (d->num_tokens && (!d->parents != !d->mask_words || !d->parents != !d->tree_mask)) return bad("parents, mask_words and tree_mask go together");
    if (!d->token_offsets || (d->batch && (!d->seq_held || !d->seq_new || !d->seq_hot || (d->hot_count && !d->refs))) ||
        (d->free_count && !d->free_pages))
        return bad("null pointer");
    const uint64_t b = 4ull * d->batch, t = d->num_tokens;
    const Span out[] = {{d->refs, d->batch ? 4ull * ((uint64_t)(d->batch - 1) * d->refs_stride + d->hot_count) : 0}, {d->seq_hot, b},
                        {d->pages_out, b}, {d->token_offsets, b + 4}, {d->free_next, 4}, {d->slots, 8 * t}, {d->positions, 4 * t},
                        {d->tree_mask, 4 * t * d->mask_words}};
    const Span in[] = {{d->seq_held, b}, {d->seq_new, b}, {d->seq_pages, b}, {d->free_pages, 4ull * d->free_count}, {d->free_first, 4},
                       {d->parents, 4 * t}};
    if (outputs_meet(out, in)) return bad("an output overlaps an input or another output");
    *a = awo::TablesArgs{};
    a->batch = d->batch;
    a->tokens = d->num_tokens;
    a->hot_count = d->hot_count;
    a->refs_stride = d->refs_stride;
    a->free_count = d->free_count;
    a->mask_words = d->mask_words;
    a->seq_held = d->seq_held;
    a->seq_new = d->seq_new;
    a->seq_pages = d->seq_pages;
    a->free_pages = d->free_pages;
    a->free_first = d->free_first;
    a->parents = d->parents;
    a->refs = d->refs;
    a->seq_hot = d->seq_hot;
    a->pages_out = d->pages_out;
    a->token_offsets = d->token_offsets;
    a->free_next = d->free_next;
    a->slots = d->slots;
    a->positions = d->positions;
    a->tree_mask = d->tree_mask;
    return AW_OK;
}

int logits_args(const aw_logits_desc* d, awo::LogitsArgs* a, char* msg, size_t len) {
    auto bad = [&](const char* why) { return refuse(msg, len, AW_E_INVALID_ARG, "adjust_logits: %s", why); };
    auto over = [&](const char* why) { return refuse(msg, len, AW_E_UNSUPPORTED, "adjust_logits: %s", why); };
    if (!d) return bad("null descriptor");
    if (int rc = step_rows("adjust_logits", d->batch, d->num_tokens, d->token_offsets, true, msg, len)) return rc;
    if (d->flags & ~AW_LOGITS_F16) return bad("unknown flags");
    if (d->vocab_size == 0) return bad("vocab_size is 0");
    if (d->vocab_size > 1u << 24) return over("vocab_size exceeds 2^24");
    if (d->history_stride > 1u << 20) return over("history_stride exceeds 2^20");
    if (d->bias_stride > 1023) return over("bias_stride exceeds 1023");
    if (d->mask_words > AW_MAX_NODES / 32) return over("mask_words exceeds 32");
    if (!d->out && !d->best && d->num_tokens) return bad("neither out nor best is asked for");
    if (!d->logits && d->num_tokens) return bad("null pointer");
    if ((d->history || d->repetition || d->frequency || d->presence || d->bias_ids || d->node_tokens || d->token_offsets) && !d->batch &&
        d->num_tokens)
        return bad("batch is 0");
    if (d->history && !d->history_count) return bad("history needs history_count");
    if (d->prompt_count && !d->history && d->history_stride) return bad("prompt_count without history");
    if (d->num_tokens && (!d->node_tokens != !d->tree_mask || !d->node_tokens != !d->mask_words)) return bad("node_tokens, tree_mask and mask_words go together");
    if (d->bias_stride && (!d->bias_ids != !d->bias_values || (d->bias_count && !d->bias_ids))) return bad("bias_ids and bias_values go together");
    if (d->allowed_index && !d->allowed && d->allowed_rows) return bad("allowed_index without allowed");
    const uint32_t size = d->flags & AW_LOGITS_F16 ? 2u : 4u;
    const uint64_t words = cdiv64(d->vocab_size, 32);
    const uint64_t stride = d->logits_stride ? d->logits_stride : d->vocab_size, out_stride = d->out_stride ? d->out_stride : d->vocab_size;
    const uint64_t allowed = d->allowed_stride ? d->allowed_stride : words;
    if (stride < d->vocab_size || out_stride < d->vocab_size || allowed < words) return bad("a stride is shorter than a row");
    if (stride > kMostStride || out_stride > kMostStride || allowed > kMostStride) return over("a stride exceeds 2^30 elements");
    if (((uintptr_t)d->logits | (uintptr_t)d->out) & (size - 1u)) return refuse(msg, len, AW_E_ALIGN, "adjust_logits: rows at their elements' alignment");
    if (d->allowed && !d->allowed_index && d->allowed_rows < d->num_tokens) return bad("fewer allowed rows than rows");
    const uint64_t t = d->num_tokens, b = 4ull * d->batch;
    auto rows = [&](uint64_t n, uint64_t s, uint64_t row) { return n ? (n - 1) * s + row : 0; };
    const Span out[] = {{d->out, size * rows(t, out_stride, d->vocab_size)}, {d->best, 4 * t}};
    const Span in[] = {{d->token_offsets, b + 4}, {d->history, b * d->history_stride}, {d->history_count, b}, {d->prompt_count, b}, {d->repetition, b},
                       {d->frequency, b}, {d->presence, b}, {d->node_tokens, 4 * t}, {d->tree_mask, 4 * t * d->mask_words},
                       {d->bias_ids, b * d->bias_stride}, {d->bias_values, b * d->bias_stride}, {d->bias_count, b},
                       {d->allowed, 4 * rows(d->allowed_rows, allowed, words)}, {d->allowed_index, 4 * t},
                       {d->out == d->logits && stride == out_stride ? nullptr : d->logits, size * rows(t, stride, d->vocab_size)}};
    if (outputs_meet(out, in) || spans_meet(out[1], {d->logits, size * rows(t, stride, d->vocab_size)}))
        return bad("an output overlaps an input or another output");
    *a = awo::LogitsArgs{};
    a->rows = d->num_tokens;
    a->vocab = d->vocab_size;
    a->batch = d->batch;
    a->mask_words = d->mask_words;
    a->history_stride = d->history_stride;
    a->bias_stride = d->bias_stride;
    a->allowed_rows = d->allowed_rows;
    a->logits_stride = stride;
    a->out_stride = out_stride;
    a->allowed_stride = allowed;
    a->logits = d->logits;
    a->out = d->out;
    a->best = d->best;
    a->token_offsets = d->token_offsets;
    a->history = d->history_stride ? d->history : nullptr;
    a->history_count = d->history_count;
    a->prompt_count = d->prompt_count;
    a->repetition = d->repetition;
    a->frequency = d->frequency;
    a->presence = d->presence;
    a->node_tokens = d->node_tokens;
    a->tree_mask = d->tree_mask;
    a->bias_ids = d->bias_stride ? d->bias_ids : nullptr;
    a->bias_values = d->bias_values;
    a->bias_count = d->bias_count;
    a->allowed = d->allowed;
    a->allowed_index = d->allowed_index;
    if (!a->history && !a->node_tokens && !a->bias_ids && !a->token_offsets) a->batch = 0; // nothing is counted: the rows stand for themselves
    return AW_OK;
}

int accept_args(const aw_accept_desc* d, awo::AcceptArgs* a, char* msg, size_t len) {
    auto bad = [&](const char* why) { return refuse(msg, len, AW_E_INVALID_ARG, "accept_tree: %s", why); };
    auto over = [&](const char* why) { return refuse(msg, len, AW_E_UNSUPPORTED, "accept_tree: %s", why); };
    if (!d) return bad("null descriptor");
    if (int rc = step_rows("accept_tree", d->batch, d->num_tokens, d->token_offsets, true, msg, len)) return rc;
    if (d->layers > 65535u) return over("layers exceed 65535");
    if (d->history_stride > 1u << 30) return over("history_stride exceeds 2^30");
    const uint64_t t = d->num_tokens, b = 4ull * d->batch, row = (uint64_t)d->kv_heads * d->head_dim;
    if (d->batch && (!d->seq_held || !d->accepted || !d->next_token || !d->seq_hot)) return bad("null pointer");
    if (d->batch && t && (!d->parents || !d->node_tokens || !d->targets || !d->path)) return bad("null pointer");
    if (!d->history != !d->history_count || !d->history != !d->history_count_out) return bad("history and its two counts go together");
    uint64_t ks = d->k_stride ? d->k_stride : row, vs = d->v_stride ? d->v_stride : row;
    uint64_t kl = d->k_layer_stride ? d->k_layer_stride : t * ks, vl = d->v_layer_stride ? d->v_layer_stride : t * vs;
    uint64_t hl = d->hot_layer_stride ? d->hot_layer_stride : d->hot_blocks * awo::kPageTokens * row;
    Span k{}, v{}, hk{}, hv{};
    if (d->layers) {
        if (row == 0) return bad("kv_heads or head_dim is 0");
        if (row > 1u << 20) return over("a token's row exceeds 2^20 values");
        if (t && (!d->k || !d->hot_k || !d->slots)) return bad("null pointer");
        if (t && !d->v != !d->hot_v) return bad("v and hot_v go together");
        if (d->hot_blocks == 0) return bad("hot_blocks is 0");
        if (d->hot_blocks > 1ull << 31) return bad("hot_blocks exceeds 2^31, the refs' range");
        if (ks < row || vs < row || (d->layers > 1 && hl < d->hot_blocks * awo::kPageTokens * row)) return bad("a stride is shorter than what it steps over");
        if (std::max(ks, vs) > kMostStride || std::max({kl, vl, hl}) > 1ull << 46) return over("a stride is too long");
        const uint64_t rows = t ? (t - 1) : 0, pool = 2 * ((d->layers - 1) * hl + d->hot_blocks * awo::kPageTokens * row);
        k = {d->k, t ? 2 * ((d->layers - 1) * kl + rows * ks + row) : 0};
        v = {d->v, t ? 2 * ((d->layers - 1) * vl + rows * vs + row) : 0};
        hk = {d->hot_k, pool};
        hv = {d->hot_v, pool};
    }
    const uint64_t hist = b * d->history_stride;
    const Span out[] = {hk, {d->accepted, b}, {d->next_token, b}, {d->seq_hot, b}, {d->path, 4 * t}, {d->history, hist}, {d->history_count_out, b}};
    const Span rest[] = {hv, out[1], out[2], out[3], out[4], out[5], out[6]}; // the pools' layers may lie between each other's
    const Span in[] = {k, v, {d->parents, 4 * t}, {d->node_tokens, 4 * t}, {d->targets, 4 * t}, {d->token_offsets, b + 4},
                       {d->seq_held == d->seq_hot ? nullptr : d->seq_held, b}, {d->slots, 8 * t},
                       {d->history_count == d->history_count_out ? nullptr : d->history_count, b}};
    const uint64_t layer = d->hot_blocks * awo::kPageTokens * row;
    if (outputs_meet(out, in) || outputs_meet(rest, in) || (d->layers && rows_meet({d->hot_k, hl, layer, d->layers}, {d->hot_v, hl, layer, d->layers})))
        return bad("an output overlaps an input or another output");
    // The two inputs that an output may be are nobody else's.
    for (const Span& o : {hk, hv, out[1], out[2], out[3], out[4], out[5], out[6]})
        if ((o.at != d->seq_hot && spans_meet(o, {d->seq_held, b})) || (o.at != d->history_count_out && spans_meet(o, {d->history_count, b})))
            return bad("an output overlaps an input or another output");
    *a = awo::AcceptArgs{};
    a->batch = d->batch;
    a->tokens = d->num_tokens;
    a->layers = d->layers;
    a->row = (uint32_t)row;
    a->history_stride = d->history_stride;
    a->hot_blocks = d->hot_blocks;
    a->k_stride = ks;
    a->v_stride = vs;
    a->k_layer = kl;
    a->v_layer = vl;
    a->hot_layer = hl;
    a->parents = d->parents;
    a->node_tokens = d->node_tokens;
    a->targets = d->targets;
    a->token_offsets = d->token_offsets;
    a->seq_held = d->seq_held;
    a->slots = d->slots;
    a->k = d->k;
    a->v = d->v;
    a->hot_k = d->hot_k;
    a->hot_v = d->hot_v;
    a->accepted = d->accepted;
    a->next_token = d->next_token;
    a->seq_hot = d->seq_hot;
    a->path = d->path;
    a->history = d->history;
    a->history_count = d->history_count;
    a->history_count_out = d->history_count_out;
    return AW_OK;
}

template <typename T, int IT>
int launch_logits(aw_engine* e, awo::LogitsArgs& a, hipStream_t st) {
    const uint32_t slice = 256u * (16u / (uint32_t)sizeof(T)) * IT;
    const bool words = a.history || a.node_tokens || a.bias_ids;
    a.slices = (uint32_t)cdiv64(a.vocab, slice);
    // Rows of a work-group: a sequence's counts serve several, where that leaves 8 work-groups a
    // CU.  526 rows x 49155 f16 of 16 sequences, groups of 1, 2, 3 (taken), 4, 16: 47.4, 44.2, 43.8, 46.8,
    // 78.6 us; 64 rows x 128256 f32 of 64 sequences, whose rows share nothing, 1 (taken), 2, 4: 26.5, 26.8, 37.3.
    a.group = words ? (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(16, (uint64_t)a.rows * a.slices / (8ull * ei::compute_units(e)))) : 1u;
    const uint64_t grid = cdiv64(a.rows, a.group) * a.slices;
    if (grid > 0xFFFFFFull) return ei::fail(e, AW_E_UNSUPPORTED, "adjust_logits: too many rows"); // 256 threads each, below 2^32
    if (a.best && a.slices > 1) {
        void* keys = nullptr;
        if (int rc = ei::workspace(e, 8ull * a.rows * a.slices, st, &keys)) return rc;
        a.keys = (uint64_t*)keys;
    }
    if (words)
        hipLaunchKernelGGL((awo::logits_kernel<T, IT, true>), dim3((uint32_t)grid), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((awo::logits_kernel<T, IT, false>), dim3((uint32_t)grid), dim3(256), 0, st, a);
    OPS_HIP(e, hipGetLastError());
    if (a.best && a.slices > 1) {
        hipLaunchKernelGGL(awo::logits_best_kernel, dim3((uint32_t)cdiv64(a.rows, 4)), dim3(256), 0, st, a);
        OPS_HIP(e, hipGetLastError());
    }
    return AW_OK;
}

} // namespace

namespace aw_engine_internal {

bool ops_set_lds_limits(size_t max_lds) {
    bool ok = true;
    auto set = [&](const void* f) {
        if (hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, (int)max_lds) != hipSuccess) {
            ok = false;
            (void)hipGetLastError();
        }
    };
    each_tile([&](auto t) {
        using T = decltype(t);
        ok = ok && max_lds >= T::kLdsBytes;
        set((const void*)awo::gemm_tile_kernel<T, false, awo::Epi::Store>);
        set((const void*)awo::gemm_tile_kernel<T, true, awo::Epi::Store>);
        set((const void*)awo::gemm_tile_kernel<T, false, awo::Epi::Residual>);
    });
    return ok;
}

} // namespace aw_engine_internal

extern "C" {

int aw_ops_copy_buffer(aw_engine* e, const uint16_t* src, uint16_t* dst, uint32_t count, uint32_t src_off,
                       uint32_t dst_off, void* stream) {
    int rc = enter(e);
    if (rc || count == 0) return rc;
    if (!src || !dst) return ei::fail(e, AW_E_INVALID_ARG, "copy_buffer: null pointer");
    awo::EwArgs p{};
    p.a = src + src_off;
    p.out = dst + dst_off;
    p.n = count;
    return launch_ew<awo::Ew::Copy>(e, p, aligned(p.a, 16) && aligned(p.out, 16), (hipStream_t)stream);
}

int aw_ops_embed_lookup(aw_engine* e, const uint32_t* token_ids, const uint16_t* table, uint16_t* out,
                        uint32_t hidden_size, uint32_t seq_len, uint32_t vocab_size, void* stream) {
    int rc = enter(e);
    if (rc || hidden_size == 0 || seq_len == 0) return rc;
    if (!token_ids || !table || !out) return ei::fail(e, AW_E_INVALID_ARG, "embed_lookup: null pointer");
    if (vocab_size == 0) return ei::fail(e, AW_E_INVALID_ARG, "embed_lookup: vocab_size is 0");
    const bool vec = hidden_size % 8 == 0 && aligned(table, 16) && aligned(out, 16);
    const uint32_t cw = (uint32_t)cdiv64(vec ? hidden_size / 8 : hidden_size, 256);
    const uint64_t blocks = (uint64_t)cw * seq_len;
    if (blocks > 0x7FFFFFFFull) return ei::fail(e, AW_E_UNSUPPORTED, "embed_lookup: grid too large");
    hipStream_t st = (hipStream_t)stream;
    if (vec)
        hipLaunchKernelGGL(awo::embed_kernel<true>, dim3((uint32_t)blocks), dim3(256), 0, st, token_ids, table, out,
                           hidden_size, cw, vocab_size, ei::error_word(e));
    else
        hipLaunchKernelGGL(awo::embed_kernel<false>, dim3((uint32_t)blocks), dim3(256), 0, st, token_ids, table, out,
                           hidden_size, cw, vocab_size, ei::error_word(e));
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

int aw_ops_rms_norm(aw_engine* e, const uint16_t* input, const uint16_t* weight, uint16_t* output,
                    uint32_t hidden_size, uint32_t num_tokens, float eps, void* stream) {
    int rc = enter(e);
    if (rc || hidden_size == 0 || num_tokens == 0) return rc;
    if (!input || !weight || !output) return ei::fail(e, AW_E_INVALID_ARG, "rms_norm: null pointer");
    if (num_tokens > 0x7FFFFFFFu) return ei::fail(e, AW_E_UNSUPPORTED, "rms_norm: too many tokens");
    const bool vec = hidden_size % 8 == 0 && aligned(input, 16) && aligned(weight, 16) && aligned(output, 16);
    hipStream_t st = (hipStream_t)stream;
    if (vec)
        hipLaunchKernelGGL(awo::rms_norm_kernel<true>, dim3(num_tokens), dim3(256), 0, st, input, weight, output,
                           hidden_size, eps);
    else
        hipLaunchKernelGGL(awo::rms_norm_kernel<false>, dim3(num_tokens), dim3(256), 0, st, input, weight, output,
                           hidden_size, eps);
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

int aw_ops_rope(aw_engine* e, uint16_t* q, uint16_t* k, uint32_t num_tokens, uint32_t q_heads, uint32_t kv_heads,
                uint32_t head_dim, uint32_t start_position, float theta, void* stream) {
    int rc = enter(e);
    if (rc || num_tokens == 0 || q_heads + kv_heads == 0) return rc;
    if (head_dim == 0 || head_dim % 2) return ei::fail(e, AW_E_INVALID_ARG, "rope: head_dim %u must be even", head_dim);
    if ((q_heads && !q) || (kv_heads && !k)) return ei::fail(e, AW_E_INVALID_ARG, "rope: null pointer");
    if (!(theta > 0.0f)) return ei::fail(e, AW_E_INVALID_ARG, "rope: theta must be positive");
    const uint64_t heads = (uint64_t)q_heads + kv_heads, pairs = (uint64_t)num_tokens * (head_dim / 2);
    if (cdiv64(pairs * heads, 256) > 0x7FFFFFFFull) return ei::fail(e, AW_E_UNSUPPORTED, "rope: grid too large");
    // Heads of one thread: as many as leave every CU two work-groups, at most 8 (a
    // longer run is a longer chain of loads).
    const uint32_t per = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(8, pairs * heads / (512ull * ei::compute_units(e))));
    hipLaunchKernelGGL(awo::rope_kernel, dim3((uint32_t)cdiv64(pairs * cdiv64(heads, per), 256)), dim3(256), 0,
                       (hipStream_t)stream, q, k, num_tokens, q_heads, kv_heads, head_dim, start_position, theta, per);
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

int aw_ops_matmul(aw_engine* e, const uint16_t* a, const uint16_t* b, uint16_t* output, uint32_t m, uint32_t n,
                  uint32_t k, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    const Product p{b, nullptr, output, n};
    return launch_products<awo::Epi::Store, false>(e, "matmul", a, &p, 1, m, k, 1.0f, (hipStream_t)stream);
}

int aw_ops_matmul_scaled(aw_engine* e, const uint16_t* a, const uint16_t* b, float* output, uint32_t m, uint32_t n,
                         uint32_t k, float scale, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    const Product p{b, nullptr, output, n};
    return launch_products<awo::Epi::Store, true>(e, "matmul_scaled", a, &p, 1, m, k, scale, (hipStream_t)stream);
}

int aw_ops_matmul_add_residual(aw_engine* e, const uint16_t* a, const uint16_t* b, uint16_t* x, uint32_t m,
                               uint32_t n, uint32_t k, float residual_multiplier, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    const Product p{b, nullptr, x, n};
    return launch_products<awo::Epi::Residual, false>(e, "matmul_add_residual", a, &p, 1, m, k, residual_multiplier,
                                                      (hipStream_t)stream);
}

int aw_ops_matmul_silu_gate(aw_engine* e, const uint16_t* a, const uint16_t* b_gate, const uint16_t* b_up,
                            uint16_t* output, uint32_t m, uint32_t n, uint32_t k, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    const Product p{b_gate, b_up, output, n};
    return launch_products<awo::Epi::SiluGate, false>(e, "matmul_silu_gate", a, &p, 1, m, k, 1.0f,
                                                      (hipStream_t)stream);
}

int aw_ops_matmul_qkv(aw_engine* e, const uint16_t* a, const uint16_t* b_q, const uint16_t* b_k, const uint16_t* b_v,
                      uint16_t* q, uint16_t* k_out, uint16_t* v_out, uint32_t m, uint32_t n_q, uint32_t n_kv,
                      uint32_t k, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    const Product p[3] = {{b_q, nullptr, q, n_q}, {b_k, nullptr, k_out, n_kv}, {b_v, nullptr, v_out, n_kv}};
    return launch_products<awo::Epi::Store, false>(e, "matmul_qkv", a, p, 3, m, k, 1.0f, (hipStream_t)stream);
}

int aw_ops_silu_gate(aw_engine* e, const uint16_t* gate, const uint16_t* up, uint16_t* output, uint32_t size,
                     void* stream) {
    int rc = enter(e);
    if (rc || size == 0) return rc;
    if (!gate || !up || !output) return ei::fail(e, AW_E_INVALID_ARG, "silu_gate: null pointer");
    awo::EwArgs p{};
    p.a = gate;
    p.b = up;
    p.out = output;
    p.n = size;
    const bool vec = aligned(gate, 16) && aligned(up, 16) && aligned(output, 16);
    return launch_ew<awo::Ew::Silu>(e, p, vec, (hipStream_t)stream);
}

int aw_ops_add_residual(aw_engine* e, uint16_t* x, const uint16_t* residual, uint32_t size, void* stream) {
    int rc = enter(e);
    if (rc || size == 0) return rc;
    if (!x || !residual) return ei::fail(e, AW_E_INVALID_ARG, "add_residual: null pointer");
    awo::EwArgs p{};
    p.a = x;
    p.b = residual;
    p.out = x;
    p.n = size;
    return launch_ew<awo::Ew::Add>(e, p, aligned(x, 16) && aligned(residual, 16), (hipStream_t)stream);
}

int aw_ops_add_bias(aw_engine* e, uint16_t* x, const uint16_t* bias, uint32_t hidden_size, uint32_t num_tokens,
                    void* stream) {
    int rc = enter(e);
    if (rc || hidden_size == 0 || num_tokens == 0) return rc;
    if (!x || !bias) return ei::fail(e, AW_E_INVALID_ARG, "add_bias: null pointer");
    awo::EwArgs p{};
    p.a = x;
    p.b = bias;
    p.out = x;
    p.n = (uint64_t)hidden_size * num_tokens;
    p.period = hidden_size;
    const bool vec = hidden_size % 8 == 0 && aligned(x, 16) && aligned(bias, 16);
    return launch_ew<awo::Ew::Bias>(e, p, vec, (hipStream_t)stream);
}

int aw_ops_scale_f16(aw_engine* e, uint16_t* x, uint32_t count, float scale, void* stream) {
    int rc = enter(e);
    if (rc || count == 0) return rc;
    if (!x) return ei::fail(e, AW_E_INVALID_ARG, "scale_f16: null pointer");
    awo::EwArgs p{};
    p.a = x;
    p.out = x;
    p.n = count;
    p.s = scale;
    return launch_ew<awo::Ew::Scale>(e, p, aligned(x, 16), (hipStream_t)stream);
}

int aw_ops_causal_attention(aw_engine* e, const uint16_t* q, const uint16_t* k, const uint16_t* v, uint16_t* output,
                            uint32_t kv_len, uint32_t head_dim, uint64_t cache_tokens, void* stream) {
    if (!e) return AW_E_INVALID_ARG;
    return aw_multihead_attention_device(e, q, k, v, output, kv_len, head_dim, 1, 1, 1, cache_tokens, stream);
}

int aw_rotary_frequencies(const aw_rotary_scaling* s, double* inv_freq) {
    if (!s || !inv_freq || s->rotary_dim == 0 || s->rotary_dim % 2) return AW_E_INVALID_ARG;
    if (!(s->theta > 0.0 && std::isfinite(s->theta)) || s->kind > AW_ROTARY_SCALE_PARTS) return AW_E_INVALID_ARG;
    if (s->kind != AW_ROTARY_SCALE_NONE && !(s->factor > 0.0 && std::isfinite(s->factor))) return AW_E_INVALID_ARG;
    if (s->kind == AW_ROTARY_SCALE_NTK && s->rotary_dim == 2) return AW_E_INVALID_ARG;
    if (s->kind == AW_ROTARY_SCALE_PARTS && !(s->original_length > 0.0 && std::isfinite(s->original_length) &&
                                              s->low >= 0.0 && s->high > s->low && std::isfinite(s->high)))
        return AW_E_INVALID_ARG;
    const double n = (double)s->rotary_dim;
    const double theta = s->kind == AW_ROTARY_SCALE_NTK ? s->theta * std::pow(s->factor, n / (n - 2.0)) : s->theta;
    for (uint32_t p = 0; p < s->rotary_dim / 2; ++p) {
        double f = std::pow(theta, -2.0 * (double)p / n);
        if (s->kind == AW_ROTARY_SCALE_LINEAR) f /= s->factor;
        if (s->kind == AW_ROTARY_SCALE_PARTS) {
            const double turns = s->original_length * f / (2.0 * 3.14159265358979323846);
            const double keep = std::min(1.0, std::max(0.0, (turns - s->low) / (s->high - s->low)));
            f = (1.0 - keep) * f / s->factor + keep * f;
        }
        inv_freq[p] = f;
    }
    return AW_OK;
}

int aw_ops_check_rotary(const aw_rotary_desc* d, int norms, char* msg, size_t msg_len) {
    awo::RotaryArgs a;
    return rows_args(d, norms != 0, &a, msg, msg_len);
}

int aw_ops_check_append(const aw_append_desc* d, char* msg, size_t msg_len) {
    awo::RotaryArgs a;
    return append_args(d, &a, msg, msg_len);
}

int aw_ops_rotary(aw_engine* e, const aw_rotary_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::RotaryArgs a;
    char msg[256] = {0};
    if ((rc = rows_args(d, false, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    return d->num_tokens && d->q_heads + d->kv_heads ? launch_rotary<false>(e, a, (hipStream_t)stream) : AW_OK;
}

int aw_ops_qk_norm_rotary(aw_engine* e, const aw_rotary_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::RotaryArgs a;
    char msg[256] = {0};
    if ((rc = rows_args(d, true, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    return d->num_tokens && d->q_heads + d->kv_heads ? launch_rotary<false>(e, a, (hipStream_t)stream) : AW_OK;
}

int aw_ops_append_paged(aw_engine* e, const aw_append_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::RotaryArgs a;
    char msg[256] = {0};
    if ((rc = append_args(d, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    return d->rows.num_tokens && d->batch ? launch_rotary<true>(e, a, (hipStream_t)stream) : AW_OK;
}

void aw_abi_ops_desc_sizes(size_t sizes[3]) {
    sizes[0] = sizeof(aw_rotary_scaling);
    sizes[1] = sizeof(aw_rotary_desc);
    sizes[2] = sizeof(aw_append_desc);
}

int aw_ops_check_tables(const aw_tables_desc* d, char* msg, size_t msg_len) {
    awo::TablesArgs a;
    return tables_args(d, &a, msg, msg_len);
}

int aw_ops_check_logits(const aw_logits_desc* d, char* msg, size_t msg_len) {
    awo::LogitsArgs a;
    return logits_args(d, &a, msg, msg_len);
}

int aw_ops_check_accept(const aw_accept_desc* d, char* msg, size_t msg_len) {
    awo::AcceptArgs a;
    return accept_args(d, &a, msg, msg_len);
}

int aw_ops_page_tables(aw_engine* e, const aw_tables_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::TablesArgs a;
    char msg[256] = {0};
    if ((rc = tables_args(d, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    a.err = ei::error_word(e);
    const dim3 grid((uint32_t)std::max<uint64_t>(1, cdiv64(a.tokens, awo::kTablesRows)));
    if (a.parents)
        hipLaunchKernelGGL(awo::tables_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(awo::tables_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

int aw_ops_adjust_logits(aw_engine* e, const aw_logits_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::LogitsArgs a;
    char msg[256] = {0};
    if ((rc = logits_args(d, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    if (a.rows == 0) return AW_OK;
    a.err = ei::error_word(e);
    // Slices of one piece a thread while those fill the card's CUs at most once, 4096 tokens
    // from there on: 1 x 151936 f32 7.0 us (4096 tokens: 8.6), but 8 x 151936 f16 9.4 (short
    // slices 10.4), 64 x 128256 f32 26.1 (42.4): the history is counted for each slice.
    const bool half = d->flags & AW_LOGITS_F16;
    const bool few = cdiv64(a.vocab, half ? 2048 : 1024) * a.rows <= ei::compute_units(e);
    if (half) return few ? launch_logits<_Float16, 1>(e, a, (hipStream_t)stream) : launch_logits<_Float16, 2>(e, a, (hipStream_t)stream);
    return few ? launch_logits<float, 1>(e, a, (hipStream_t)stream) : launch_logits<float, 4>(e, a, (hipStream_t)stream);
}

int aw_ops_accept_tree(aw_engine* e, const aw_accept_desc* d, void* stream) {
    int rc = enter(e);
    if (rc) return rc;
    awo::AcceptArgs a;
    char msg[256] = {0};
    if ((rc = accept_args(d, &a, msg, sizeof msg))) return ei::fail(e, rc, "%s", msg);
    if (a.batch == 0) return AW_OK;
    a.err = ei::error_word(e);
    const dim3 grid(a.batch, std::max(a.layers, 1u));
    const bool vec = aligned(a.k, 16) && aligned(a.v, 16) && aligned(a.hot_k, 16) && aligned(a.hot_v, 16) &&
                     (a.row | a.k_stride | a.v_stride | a.k_layer | a.v_layer | a.hot_layer) % 8 == 0;
    if (vec)
        hipLaunchKernelGGL(awo::accept_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, a);
    else
        hipLaunchKernelGGL(awo::accept_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, a);
    OPS_HIP(e, hipGetLastError());
    return AW_OK;
}

void aw_abi_step_desc_sizes(size_t sizes[3]) {
    sizes[0] = sizeof(aw_tables_desc);
    sizes[1] = sizeof(aw_logits_desc);
    sizes[2] = sizeof(aw_accept_desc);
}

int aw_debug_product_tile(uint32_t compute_units, uint32_t m, const uint32_t* n, uint32_t products, uint32_t k,
                          uint32_t tile[3]) {
    if (!n || !tile || products < 1 || products > 3 || m <= 64 || !compute_units) return AW_E_INVALID_ARG;
    if (k % 8 || (uint64_t)k * 512 > awo::kTileBytesMax) return AW_E_UNSUPPORTED;
    awo::GemmArgs g{};
    g.M = m;
    g.K = k;
    for (uint32_t i = 0; i < products; ++i)
        if (n[i]) g.g[g.groups++].N = n[i];
    const bool ok = g.groups && with_tile(g, compute_units, [&](auto t) {
        using T = decltype(t);
        tile[0] = T::TM;
        tile[1] = T::TN;
        tile[2] = T::NB;
    });
    return ok ? AW_OK : AW_E_UNSUPPORTED;
}

} // extern "C"
