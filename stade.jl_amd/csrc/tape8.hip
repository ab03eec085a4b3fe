// tape8_store and tape8_load: rows to and from their 8-bit tape (tape8.hpp).
//
// Both are copies: a lane takes 8 values (one wide load), a quad of lanes a group, whose largest
// value goes round by two DPP moves.  Bound by HBM: 16384 x 2048 bf16 are stored in 26 us (3.9 TB/s), in calls one after the
// other on the same arrays, which the last-level cache holds, in 18.4 and read back in 17.1 (5.5 and 5.9 TB/s); 16384 x 4096
// in 33 and 31.
#include "tape8.hpp"

#include <algorithm>

namespace stade {
namespace {

using namespace tape8;

constexpr int NT = 256;

// a quad of lanes a group: lanes past the row's last group leave together
template <class T>
__global__ __launch_bounds__(NT) void store_kernel(const T* x, int64_t ldx, uint8_t* q, uint8_t* qs, int d, int64_t n) {
    const int64_t ng = groups(d), all = n * ng;
    const int part = threadIdx.x & 3;
    for (int64_t g = (int64_t)blockIdx.x * (NT / 4) + (threadIdx.x >> 2); g < all; g += (int64_t)gridDim.x * (NT / 4)) {
        const int64_t row = g / ng;
        const int col = (int)(g - row * ng) * kGroup + 8 * part;
        float v[8];
        rows::load_row(v, x + row * ldx + col, d - col);
        store_part<T>(q + row * ng * kGroup, qs + row * ng, v, col, ng);
    }
}

template <class T>
__global__ __launch_bounds__(NT) void load_kernel(const uint8_t* q, const uint8_t* qs, T* x, int64_t ldx, int d, int64_t n) {
    const int64_t ng = groups(d), all = n * ng;
    const int part = threadIdx.x & 3;
    for (int64_t g = (int64_t)blockIdx.x * (NT / 4) + (threadIdx.x >> 2); g < all; g += (int64_t)gridDim.x * (NT / 4)) {
        const int64_t row = g / ng;
        const int col = (int)(g - row * ng) * kGroup + 8 * part;
        float v[8];
        values(v, q + g * kGroup + 8 * part, unit(qs[g]));
        if (col < d) rows::store_row(x + row * ldx + col, v, d - col);
    }
}

int32_t check(const char* fn, int64_t type, const void* x, int64_t ldx, const void* q, const void* qs, int64_t i_d, int64_t i_n) {
    if (int32_t rc = rows::check_type(fn, "x", type)) return rc;
    if (int32_t rc = rows::check_extent(fn, "i_d", i_d, rows::kMostCols)) return rc;
    if (int32_t rc = rows::check_extent(fn, "i_n", i_n, rows::kMostRows)) return rc;
    if (int32_t rc = rows::check_ld(fn, "ldx", ldx, i_d)) return rc;
    if (i_d > 0 && i_n > 0) {
        if (!x || !q || !qs) return rows::bad(fn, "null pointer");
        if ((uintptr_t)q % 8) return rows::bad(fn, "q is not aligned to 8 bytes");
    }
    return 0;
}

unsigned grid_of(int64_t i_d, int64_t i_n) {
    return (unsigned)std::min<int64_t>((i_n * groups(i_d) + NT / 4 - 1) / (NT / 4), 1 << 16);
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_tape8_lengths(int64_t i_d, int64_t i_n, int64_t lengths[2]) {
    if (!lengths) return rows::bad("stade_hip_tape8_lengths", "null output");
    if (int32_t rc = rows::check_extent("stade_hip_tape8_lengths", "i_d", i_d, rows::kMostCols)) return rc;
    if (int32_t rc = rows::check_extent("stade_hip_tape8_lengths", "i_n", i_n, rows::kMostRows)) return rc;
    lengths[0] = tape8::groups(i_d) * tape8::kGroup * i_n;
    lengths[1] = tape8::groups(i_d) * i_n;
    return STADE_HIP_OK;
}

int32_t stade_hip_tape8_store(int64_t type, const void* x, int64_t ldx, int8_t* q, uint8_t* qs, int64_t i_d, int64_t i_n,
                              hipStream_t stream) {
    if (int32_t rc = check("stade_hip_tape8_store", type, x, ldx, q, qs, i_d, i_n)) return rc;
    if (i_d == 0 || i_n == 0) return STADE_HIP_OK;
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    return rows::with_type(type, [&](auto t) -> int32_t {
        using T = decltype(t);
        STADE_TIMED("tape8_store", stream,
                    store_kernel<T><<<grid_of(i_d, i_n), NT, 0, stream>>>((const T*)x, ldx, (uint8_t*)q, qs, (int)i_d, i_n));
        STADE_LAUNCHED("tape8 store_kernel");
        return STADE_HIP_OK;
    });
}

int32_t stade_hip_tape8_load(int64_t type, const int8_t* q, const uint8_t* qs, void* x, int64_t ldx, int64_t i_d, int64_t i_n,
                             hipStream_t stream) {
    if (int32_t rc = check("stade_hip_tape8_load", type, x, ldx, q, qs, i_d, i_n)) return rc;
    if (i_d == 0 || i_n == 0) return STADE_HIP_OK;
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    return rows::with_type(type, [&](auto t) -> int32_t {
        using T = decltype(t);
        STADE_TIMED("tape8_load", stream,
                    load_kernel<T><<<grid_of(i_d, i_n), NT, 0, stream>>>((const uint8_t*)q, qs, (T*)x, ldx, (int)i_d, i_n));
        STADE_LAUNCHED("tape8 load_kernel");
        return STADE_HIP_OK;
    });
}

}  // extern "C"
