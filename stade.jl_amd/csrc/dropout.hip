// Dropout on a residual branch and its adjoint, with a mask that is never stored:
//   y = r + m x / (1 - p),   xb (+)= m yb / (1 - p)
// m is a function of (seed, call, token, column) alone, so the reverse sweep forms it again, whatever the arrays'
// strides, types and the launch: Philox 4x32 with ten rounds (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", 2011), its key the 64 bits of `seed`, its counter (column / 8, token, the 64 bits of `call`).  A block
// of 128 bits serves eight columns, 16 bits each in the order of the words, low half first; a value stays
// where its 16 bits are at least round(65536 p), so p counts in steps of 2^-16 and the scale is that of the
// rounded p.  seed and call are read on the device: a captured graph can move on to another mask.
//
// One pass, HBM bound in 16 bits: the generator's 20 products of 32 bits a block, at a quarter of the rate, are shared by eight
// values (a block for four values made the generator, not the memory, the bound).  8192 x 4096 bf16: 41 us with a residual (4.9 TB/s), the
// adjoint 28 (4.8 TB/s).
#include "rows.hpp"

#include <algorithm>
#include <math.h>

namespace stade {
namespace {

using namespace rows;

constexpr int NT = 256;

struct Drop {
    void* y; int64_t ldy;
    const void* x; int64_t ldx;
    const void* r; int64_t ldr;
    const uint64_t* key;
    int d;
    int64_t n;
    uint32_t least;   // of the 16 bits, to stay
    float scale;
};

struct Philox {
    uint32_t k0, k1, c2, c3;
    __device__ __forceinline__ explicit Philox(const uint64_t* key)
        : k0((uint32_t)key[0]), k1((uint32_t)(key[0] >> 32)), c2((uint32_t)key[1]), c3((uint32_t)(key[1] >> 32)) {}
    __device__ __forceinline__ void block(uint32_t c0, uint32_t c1, uint32_t (&out)[4]) const {
        uint32_t a = c0, b = c1, c = c2, d = c3, ka = k0, kb = k1;
#pragma unroll
        for (int i = 0; i < 10; ++i) {
            const uint64_t p = (uint64_t)a * 0xD2511F53u, q = (uint64_t)c * 0xCD9E8D57u;
            a = (uint32_t)(q >> 32) ^ b ^ ka;
            b = (uint32_t)q;
            c = (uint32_t)(p >> 32) ^ d ^ kb;
            d = (uint32_t)p;
            ka += 0x9E3779B9u;
            kb += 0xBB67AE85u;
        }
        out[0] = a; out[1] = b; out[2] = c; out[3] = d;
    }
};

// eight columns a lane; the lanes go over the rows' vectors one after the other
template <class T, bool RES>
__global__ __launch_bounds__(NT) void drop_kernel(Drop p) {
    const Philox gen(p.key);
    const uint32_t vecs = ((uint32_t)p.d + 7) / 8;
    const int64_t all = p.n * vecs, step = (int64_t)gridDim.x * NT;
    for (int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x; i < all; i += step) {
        const int64_t row = all <= 0xffffffffll ? (int64_t)((uint32_t)i / vecs) : i / vecs;
        const uint32_t vec = (uint32_t)(i - row * vecs);
        const int col = (int)vec * 8, left = p.d - col;
        float x[8], r[8];
        load_row(x, (const T*)p.x + row * p.ldx + col, left);
        if constexpr (RES) load_row(r, (const T*)p.r + row * p.ldr + col, left);
        uint32_t bits[4];
        gen.block(vec, (uint32_t)row, bits);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t u = k & 1 ? bits[k >> 1] >> 16 : bits[k >> 1] & 0xffffu;
            const float v = u >= p.least ? x[k] * p.scale : 0.f;   // (chosen, not multiplied: what is dropped may be infinite)
            x[k] = RES ? r[k] + v : v;
        }
        store_row((T*)p.y + row * p.ldy + col, x, left);
    }
}

int32_t run(const char* fn, const char* what, int64_t tx, Drop q, double p, hipStream_t stream) {
    if (q.d == 0 || q.n == 0) return STADE_HIP_OK;
    if (!q.y || !q.x || !q.key) return bad(fn, "null pointer");
    q.least = (uint32_t)lrint(65536.0 * p);
    q.scale = (float)(65536.0 / (65536.0 - (double)q.least));
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    const int64_t vecs = q.n * ((q.d + 7) / 8);
    const unsigned grid = (unsigned)std::min<int64_t>((vecs + NT - 1) / NT, 1 << 20);
    return with_type(tx, [&](auto t) -> int32_t {
        using T = decltype(t);
        STADE_TIMED(what, stream, {
            if (q.r) drop_kernel<T, true><<<grid, NT, 0, stream>>>(q);
            else drop_kernel<T, false><<<grid, NT, 0, stream>>>(q);
        });
        STADE_LAUNCHED("dropout drop_kernel");
        return STADE_HIP_OK;
    });
}

int32_t check(const char* fn, int64_t tx, double p, int64_t i_d, int64_t i_n) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_n", i_n, kMostRows)) return rc;
    if (!(p >= 0.0) || lrint(65536.0 * std::min(p, 2.0)) >= 65536) return bad(fn, "p is not in 0 <= p < 1 (in steps of 2^-16)");
    return 0;
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_dropout(int64_t tx, void* y, int64_t ldy, const void* x, int64_t ldx, const void* r, int64_t ldr, const int64_t* key, double p,
                          int64_t i_d, int64_t i_n, hipStream_t stream) {
    const char* fn = "stade_hip_dropout";
    if (int32_t rc = check(fn, tx, p, i_d, i_n)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldx", ldx, i_d)) return rc;
    if (r)
        if (int32_t rc = check_ld(fn, "ldr", ldr, i_d)) return rc;
    return run(fn, "dropout", tx, Drop{y, ldy, x, ldx, r, ldr, (const uint64_t*)key, (int)i_d, i_n}, p, stream);
}

int32_t stade_hip_dropout_b(int64_t tx, const void* yb, int64_t ldyb, void* xb, int64_t ldxb, const int64_t* key, double p, int64_t i_d,
                            int64_t i_n, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_dropout_b";
    if (int32_t rc = check(fn, tx, p, i_d, i_n)) return rc;
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldxb", ldxb, i_d)) return rc;
    // (accumulated: what xb holds is the residual)
    return run(fn, "dropout_b", tx, Drop{xb, ldxb, yb, ldyb, add ? xb : nullptr, ldxb, (const uint64_t*)key, (int)i_d, i_n}, p, stream);
}

}  // extern "C"
