// engine_internal.hpp — what the library's other sources (ops.hip) use of an
// aw_engine, whose definition stays private to weaver_engine.hip.
#pragma once

#include <stddef.h>
#include <stdint.h>

#include "../../include/aether_weaver.h"

namespace aw_engine_internal {

// Bits of the engine's device error word (aw_engine_check_device_errors):
// 1 hot block ref, 2 cold block ref, 4 atom index (weaver_kernels.hpp), 8 token id,
// 16 token counts of a sequence, 32 a list of free pages.
constexpr uint32_t kErrTokenBit = 8u;
constexpr uint32_t kErrSeqBit = 16u;
constexpr uint32_t kErrFreeBit = 32u;

int device(const aw_engine* e);        // HIP device ordinal
uint32_t compute_units(const aw_engine* e);
uint32_t* error_word(const aw_engine* e); // device address of the error word
// Records the message as the engine's last error and returns `code`.
int fail(aw_engine* e, int code, const char* fmt, ...) __attribute__((format(printf, 3, 4)));
// The engine's workspace, at least `bytes` of it, for a call on `stream` (aw_decode_device).
int workspace(aw_engine* e, size_t bytes, void* stream, void** at);

// Lets the dense-ops kernels that stage more than 64 KiB of LDS use `max_lds`
// bytes (ops.hip); false when the runtime refuses.
bool ops_set_lds_limits(size_t max_lds);

// Rows [tokens][row] of a call, `stride` elements apart; none at a null address.
struct Rows {
    const uint16_t* at;
    uint64_t stride, row, tokens;
    bool none() const { return !at || row == 0 || tokens == 0; }
    uintptr_t begin() const { return (uintptr_t)at; }
    uintptr_t end() const { return (uintptr_t)at + 2 * ((tokens - 1) * stride + row); }
};

// Whether two such sets share an element: parts of one fused buffer, rows of the same
// stride, lie at a fixed distance within it; with strides of their own the whole
// stretches count.
inline bool rows_meet(const Rows& p, const Rows& o) {
    if (p.none() || o.none() || p.begin() >= o.end() || o.begin() >= p.end()) return false;
    if (p.stride != o.stride) return true;
    const Rows &lo = p.begin() < o.begin() ? p : o, &hi = p.begin() < o.begin() ? o : p;
    const uint64_t stride = 2 * p.stride, d = (hi.begin() - lo.begin()) % stride;
    return d < 2 * lo.row || d + 2 * hi.row > stride;
}
inline bool rows_same(const Rows& p, const Rows& o) { return p.at == o.at && (p.stride == o.stride || p.tokens == 1); }

} // namespace aw_engine_internal
