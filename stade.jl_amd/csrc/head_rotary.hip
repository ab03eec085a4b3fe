// Queries and keys, head by head: a norm over the head and the rotation by the token's position, in one
// pass, and the adjoint.  With rs = 1 / sqrt(mean(x^2) + eps) and h = x rs g over a head's i_d values (without
// the norm h = x), the pairs (a, b) among the head's first i_r values turn by the angle pos * freq[j]:
//   y_a = s (a cos - b sin),  y_b = s (b cos + a sin);   values behind the first i_r stay h.
// The adjoint turns yb back, hb, and with xh = x rs, a = hb g:
//   gb (+)= sum over tokens and heads of hb xh,   xb (+)= rs (a - xh mean(a xh)).
// rs is formed again from x, which the adjoint reads anyway: nothing is kept between the sweeps.
//
// Angles are formed in fp64 as turns, pos * (freq / 2 pi), and only the fraction of a turn goes on to fp32, in two parts (an
// fp32 angle of position 10^5 is off by 10^-2).  A block forms its tokens' cosines and sines once, in LDS, for all
// heads.  Sums are fp32.
//
// Bound by HBM.  A group of lanes takes a head of a token: a lane has two vectors of it that belong together (the
// two parts of its pairs), so a pair never crosses lanes, and the sums over a head are a few DPP moves.
// The adjoint's lanes keep gb of their columns in registers over all of the block's tokens; blocks leave
// partial sums that a second launch adds in a fixed order (no atomics: the same call gives the same bits).
// 8192 tokens of 20 heads of 128, bf16: forward 23.5 us (3.6 TB/s), adjoint 31.8 (3.9 TB/s) and the weights' sums 4.6.
#include "rows.hpp"

#include <algorithm>
#include <math.h>

namespace stade {
namespace {

using namespace rows;

constexpr int NT = 256;
constexpr int64_t kMostHead = 256, kMostHeads = 4096;
constexpr int kTable = 2048;      // pairs' cosines and sines in LDS (16 KB)
constexpr int64_t kSumParts = 1024;    // blocks that leave partial sums, at most

struct Rot {
    const void* x; int64_t ldx;
    void* y; int64_t ldy;               // the results: y, or xb
    const void* yb; int64_t ldyb;       // (the adjoint)
    const void* gq; const void* gk; int gtype;
    const int64_t* pos; const double* freq;
    float* part;                        // (the adjoint) a block's sums of its weights' shadow; null without them
    int d, nq, nk, r;
    int64_t t;
    int tile;                           // tokens of a block at a time
    int log_lanes;                      // lanes of a head
    float eps, s;
    int add;
    int q_blocks;                       // blocks for queries; the rest are for keys
};

__device__ __forceinline__ float weight(const void* g, int type, int i) {
    if (!g) return 1.f;
    return type == STADE_HIP_F32 ? ((const float*)g)[i] : type == STADE_HIP_BF16 ? (float)((const bf16*)g)[i] : (float)((const f16*)g)[i];
}

// the sum over the 2^log lanes of a head, in each of them
constexpr int kDppHalfMirror = 0x141, kDppMirror = 0x140;
__device__ __forceinline__ float head_sum(float v, int log) {
    if (log > 0) v += dpp_f32<kDppQuadSwap1>(v);
    if (log > 1) v += dpp_f32<kDppQuadSwap2>(v);
    if (log > 2) v += dpp_f32<kDppHalfMirror>(v);
    if (log > 3) v += dpp_f32<kDppMirror>(v);
    if (log > 4) v += __shfl_xor(v, 16, 64);
    if (log > 5) v += __shfl_xor(v, 32, 64);
    return v;
}

// A lane's two vectors of a head: `a` and `b` the first columns, `na` and `nb` how many values there are
// (0 and less: none); `turn`: rotated, with the pairs' angles from `pair` on.
struct Cols {
    int a, b, na, nb, pair;
    bool turn;
};
template <bool HALF, int V>
__device__ __forceinline__ Cols my_cols(int lane, int d, int r) {
    const int turned = (r / 2 + V - 1) / V;
    Cols c;
    c.turn = lane < turned;
    c.pair = lane * V;
    if (c.turn && HALF) {
        c.a = lane * V;
        c.b = r / 2 + c.a;
        c.na = c.nb = r / 2 - c.a;
    } else {
        c.a = c.turn ? 2 * V * lane : r + 2 * V * (lane - turned);
        c.b = c.a + V;
        c.na = (c.turn ? r : d) - c.a;
        c.nb = c.na - V;
    }
    return c;
}

// (a, b) turned by the angles of cs; BACK: by their negatives
template <bool HALF, bool BACK, int V>
__device__ __forceinline__ void turn(float (&a)[V], float (&b)[V], const float2* cs) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        const float c = cs[i].x, s = BACK ? -cs[i].y : cs[i].y;
        // (the i-th pair: of the two vectors, or neighbours in the 2 V values that they make)
        float& u = HALF ? a[i] : 2 * i < V ? a[2 * i % V] : b[2 * i % V];
        float& w = HALF ? b[i] : 2 * i < V ? a[(2 * i + 1) % V] : b[(2 * i + 1) % V];
        const float p = u, q = w;
        u = fmaf(p, c, -(q * s));
        w = fmaf(q, c, p * s);
    }
}

// the cosines and sines of a tile's tokens, times s; `stride` pairs a token
__device__ __forceinline__ void fill_table(const Rot& p, int64_t first, int tokens, int stride, float2* table) {
    for (int i = threadIdx.x; i < tokens * stride; i += NT) {
        const int k = i / stride, j = i - k * stride;
        float2 cs = {0.f, 0.f};
        if (j < p.r / 2) {
            const double turns = (double)p.pos[first + k] * (p.freq[j] * 0.15915494309189533577);   // 1 / 2 pi
            const double whole = 2.0 * (turns - rint(turns));
            // (what its rounding leaves out, to the first order: a sine near half a turn is as small as that)
            const float f = (float)whole, rest = 3.14159265358979f * (float)(whole - (double)f);
            float sn, c;
            sincospif(f, &sn, &c);
            cs = {fmaf(-rest, sn, c) * p.s, fmaf(rest, c, sn) * p.s};
        }
        table[i] = cs;
    }
}

// A lane's two vectors of a head as they come from memory, so that the next head's are on their way while this one's
// are worked on.  WHOLE: vectors are full or empty.
template <class T, int V, bool WHOLE>
struct Raw {
    typedef typename Pack<T, V>::vec vec;
    vec a, b;
    static __device__ __forceinline__ void get(vec& v, const T* at, int left) {
        v = vec{};
        if (WHOLE ? left > 0 : left >= V) {
            v = *reinterpret_cast<const typename Pack<T, V>::loose*>(at);
        } else if constexpr (!WHOLE) {
            if (left > 0) {
#pragma unroll
                for (int i = 0; i < V; ++i) v[i] = i < left ? at[i] : (T)0.f;
            }
        }
    }
    __device__ __forceinline__ void load(const void* x, int64_t at, const Cols& c) {
        get(a, (const T*)x + at + c.a, c.na);
        get(b, (const T*)x + at + c.b, c.nb);
    }
    __device__ __forceinline__ void values(float (&u)[V], float (&w)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u[i] = (float)a[i];
            w[i] = (float)b[i];
        }
    }
};

// What a block works on: queries' heads, or keys' (the last blocks), which have weights of their own
struct Part {
    int first, heads;       // of the heads
    const void* g;
    int64_t block, blocks;  // among those of its kind
};
__device__ __forceinline__ Part my_part(const Rot& p) {
    if ((int)blockIdx.x < p.q_blocks) return Part{0, p.nq, p.gq, blockIdx.x, p.q_blocks};
    return Part{p.nq, p.nk, p.gk, blockIdx.x - p.q_blocks, gridDim.x - p.q_blocks};
}

template <class T, int V, bool HALF, bool NORM, bool WHOLE>
__global__ __launch_bounds__(NT) void forward_kernel(Rot p) {
    __shared__ float2 table[kTable];
    const Part part = my_part(p);
    const int log = p.log_lanes, lane = threadIdx.x & ((1 << log) - 1), heads = part.heads, step = gridDim.y * (NT >> log);
    const Cols c = my_cols<HALF, V>(lane, p.d, p.r);
    const int stride = (p.r / 2 + V - 1) / V * V;
    float g[2][V];
    if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[0][i] = i < c.na ? weight(part.g, p.gtype, c.a + i) : 0.f;
            g[1][i] = i < c.nb ? weight(part.g, p.gtype, c.b + i) : 0.f;
        }
    }
    for (int64_t first = part.block * p.tile; first < p.t; first += part.blocks * p.tile) {
        const int tokens = (int)min((int64_t)p.tile, p.t - first), units = tokens * heads;
        Raw<T, V, WHOLE> next;
        auto fetch = [&](int u) __attribute__((always_inline)) {
            const int k = u / heads, h = u - k * heads;
            if (u < units) next.load(p.x, (first + k) * p.ldx + (int64_t)(part.first + h) * p.d, c);
        };
        int u = (blockIdx.y * NT + threadIdx.x) >> log;
        fetch(u);
        __syncthreads();
        fill_table(p, first, tokens, stride, table);
        __syncthreads();
        for (; u < units; u += step) {
            const int k = u / heads, h = u - k * heads;
            float a[V], b[V];
            next.values(a, b);
            fetch(u + step);
            if constexpr (NORM) {
                float sq = 0.f;
#pragma unroll
                for (int i = 0; i < V; ++i) sq = fmaf(a[i], a[i], fmaf(b[i], b[i], sq));
                sq = head_sum(sq, log);
                const float rs = 1.0f / sqrtf(sq / (float)p.d + p.eps);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    a[i] = a[i] * rs * g[0][i];
                    b[i] = b[i] * rs * g[1][i];
                }
            }
            if (c.turn) turn<HALF, false>(a, b, table + k * stride + c.pair);
            T* y = (T*)p.y + (first + k) * p.ldy + (int64_t)(part.first + h) * p.d;
            store_row<WHOLE>(y + c.a, a, c.na);
            store_row<WHOLE>(y + c.b, b, c.nb);
        }
    }
}

template <class T, int V, bool HALF, bool NORM, bool WHOLE>
__global__ __launch_bounds__(NT) void backward_kernel(Rot p) {
    __shared__ float2 table[kTable];
    __shared__ float sums[kMostHead];
    const Part part = my_part(p);
    const int log = p.log_lanes, lane = threadIdx.x & ((1 << log) - 1), heads = part.heads, step = NT >> log;
    const Cols c = my_cols<HALF, V>(lane, p.d, p.r);
    const int stride = (p.r / 2 + V - 1) / V * V;
    float g[2][V], acc[2][V];
    if constexpr (NORM) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            g[0][i] = i < c.na ? weight(part.g, p.gtype, c.a + i) : 0.f;
            g[1][i] = i < c.nb ? weight(part.g, p.gtype, c.b + i) : 0.f;
            acc[0][i] = acc[1][i] = 0.f;
        }
    }
    for (int64_t first = part.block * p.tile; first < p.t; first += part.blocks * p.tile) {
        const int tokens = (int)min((int64_t)p.tile, p.t - first), units = tokens * heads;
        Raw<T, V, WHOLE> next, next_x;
        auto fetch = [&](int u) __attribute__((always_inline)) {
            const int k = u / heads, h = u - k * heads;
            const int64_t col = (int64_t)(part.first + h) * p.d;
            if (u < units) {
                next.load(p.yb, (first + k) * p.ldyb + col, c);
                if constexpr (NORM) next_x.load(p.x, (first + k) * p.ldx + col, c);
            }
        };
        int u = threadIdx.x >> log;
        fetch(u);
        __syncthreads();
        fill_table(p, first, tokens, stride, table);
        __syncthreads();
        for (; u < units; u += step) {
            const int k = u / heads, h = u - k * heads;
            float a[V], b[V], xa[V], xb[V];
            next.values(a, b);
            if constexpr (NORM) next_x.values(xa, xb);
            fetch(u + step);
            if (c.turn) turn<HALF, true>(a, b, table + k * stride + c.pair);
            if constexpr (NORM) {
                float sq = 0.f, dot = 0.f, ga[V], gb[V];
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    ga[i] = a[i] * g[0][i];
                    gb[i] = b[i] * g[1][i];
                    sq = fmaf(xa[i], xa[i], fmaf(xb[i], xb[i], sq));
                    dot = fmaf(ga[i], xa[i], fmaf(gb[i], xb[i], dot));
                }
                sq = head_sum(sq, log);
                dot = head_sum(dot, log);
                const float rs = 1.0f / sqrtf(sq / (float)p.d + p.eps), m = dot * rs / (float)p.d;
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float ha = xa[i] * rs, hb = xb[i] * rs;
                    acc[0][i] = fmaf(a[i], ha, acc[0][i]);
                    acc[1][i] = fmaf(b[i], hb, acc[1][i]);
                    a[i] = rs * fmaf(-ha, m, ga[i]);
                    b[i] = rs * fmaf(-hb, m, gb[i]);
                }
            }
            if (p.y) {
                T* y = (T*)p.y + (first + k) * p.ldy + (int64_t)(part.first + h) * p.d;
                if (p.add) {
                    float oa[V], ob[V];
                    load_row<WHOLE>(oa, y + c.a, c.na);
                    load_row<WHOLE>(ob, y + c.b, c.nb);
#pragma unroll
                    for (int i = 0; i < V; ++i) {
                        a[i] += oa[i];
                        b[i] += ob[i];
                    }
                }
                store_row<WHOLE>(y + c.a, a, c.na);
                store_row<WHOLE>(y + c.b, b, c.nb);
            }
        }
    }
    if constexpr (NORM) {
        if (!p.part) return;
        // the block's groups of lanes joined: those of a wave by steps of twice as many, then the waves one after the other
        for (int o = 1 << log; o < 64; o <<= 1)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                acc[0][i] += __shfl_xor(acc[0][i], o, 64);
                acc[1][i] += __shfl_xor(acc[1][i], o, 64);
            }
        for (int k = 0; k < NT / 64; ++k) {
            __syncthreads();
            if ((int)(threadIdx.x >> 6) == k && (int)(threadIdx.x & 63) == lane) {
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    if (i < c.na) sums[c.a + i] = (k ? sums[c.a + i] : 0.f) + acc[0][i];
                    if (i < c.nb) sums[c.b + i] = (k ? sums[c.b + i] : 0.f) + acc[1][i];
                }
            }
        }
        __syncthreads();
        for (int i = threadIdx.x; i < p.d; i += NT) p.part[(int64_t)blockIdx.x * p.d + i] = sums[i];
    }
}

// gqb and gkb (blockIdx.y) from their blocks' sums, in order: 16 columns a block, 16 strips of the blocks each
__global__ __launch_bounds__(NT) void weight_sum_kernel(const float* part, int q_blocks, int blocks, int d, float* gqb, float* gkb, int add) {
    __shared__ float lds[16][17];
    const int c = threadIdx.x & 15, strip = threadIdx.x >> 4, i = blockIdx.x * 16 + c;
    const int from = blockIdx.y ? q_blocks : 0, to = blockIdx.y ? blocks : q_blocks;
    float v = 0.f;
    if (i < d)
#pragma unroll 8
        for (int b = from + strip; b < to; b += 16) v += part[(int64_t)b * d + i];
    lds[strip][c] = v;
    __syncthreads();
    if (strip == 0 && i < d) {
        for (int k = 1; k < 16; ++k) v += lds[k][c];
        float* out = blockIdx.y ? gkb : gqb;
        if (out) out[i] = add ? out[i] + v : v;
    }
}

int32_t check(const char* fn, int64_t tx, int64_t tg, const void* gq, const void* gk, int64_t i_d, int64_t i_q, int64_t i_k, int64_t i_r,
              int64_t i_t, int64_t norm, double eps, double s) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_type(fn, "g", tg)) return rc;
    if (tg != STADE_HIP_F32 && tg != tx) return bad(fn, "the weights are neither Float32 nor of x's type");
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostHead)) return rc;
    if (int32_t rc = check_extent(fn, "i_q", i_q, kMostHeads)) return rc;
    if (int32_t rc = check_extent(fn, "i_k", i_k, kMostHeads)) return rc;
    if (int32_t rc = check_extent(fn, "i_r", i_r, i_d)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (i_r % 2) return bad(fn, "i_r is odd");
    if (!norm && (gq || gk)) return bad(fn, "weights without the norm");
    // (both are taken in Float32)
    if (norm && !(eps >= 0.0 && (float)eps < INFINITY)) return bad(fn, "eps is negative or not finite in Float32");
    if (!(fabsf((float)s) < INFINITY)) return bad(fn, "s is not finite in Float32");
    return 0;
}

template <class F>
int32_t with_form(int64_t tx, int64_t half, int64_t norm, bool whole, F&& f) {
    return with_type(tx, [&](auto t) -> int32_t {
        auto with_whole = [&](auto h, auto n) -> int32_t { return whole ? f(t, h, n, std::true_type{}) : f(t, h, n, std::false_type{}); };
        if (half) return norm ? with_whole(std::true_type{}, std::true_type{}) : with_whole(std::true_type{}, std::false_type{});
        return norm ? with_whole(std::false_type{}, std::true_type{}) : with_whole(std::false_type{}, std::false_type{});
    });
}

// a lane's vectors: 16 bytes
inline int values_of(int64_t type) { return type == STADE_HIP_F32 ? 4 : 8; }
inline int log_lanes(int64_t type, int64_t d, int64_t r) {
    const int v = values_of(type), lanes = (int)((r / 2 + v - 1) / v + (d - r + 2 * v - 1) / (2 * v));
    int log = 0;
    while ((1 << log) < lanes) ++log;
    return log;
}
// (two vectors of a lane are full or empty together, in both layouts)
inline bool whole_vectors(int64_t type, int64_t d, int64_t r) {
    const int v = values_of(type);
    return r % (2 * v) == 0 && (d - r) % (2 * v) == 0;
}
// tokens of a block at a time: some eight rounds of its lanes, and a table that fits
inline int tile_of(const Rot& p, int v) {
    const int stride = std::max(1, (p.r / 2 + v - 1) / v * v), lanes = std::max(p.nq, p.nk) << p.log_lanes;
    return std::max(1, std::min({kTable / stride, 8 * NT / lanes, 64}));
}
// `blocks` of them for all heads, as many for queries as they have of the heads
inline void share(Rot& p, int64_t blocks, int64_t tiles, unsigned& grid) {
    blocks = std::min<int64_t>(blocks, 1 << 20);   // (a launch's threads are counted in 32 bits)
    const int64_t heads = p.nq + p.nk, q = p.nq ? std::max<int64_t>(1, std::min(tiles, (blocks * p.nq + heads / 2) / heads)) : 0;
    const int64_t k = p.nk ? std::max<int64_t>(1, std::min(tiles, blocks - q)) : 0;
    p.q_blocks = (int)q;
    grid = (unsigned)(q + k);
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_rotary_freq(int64_t i_r, double base, double factor, double length, double low, double high, double* freq) {
    const char* fn = "stade_hip_rotary_freq";
    if (int32_t rc = check_extent(fn, "i_r", i_r, kMostHead)) return rc;
    if (i_r % 2) return bad(fn, "i_r is odd");
    if (!(base > 0.0) || !(base < INFINITY) || !(factor > 0.0) || !(factor < INFINITY)) return bad(fn, "base and factor must be positive and finite");
    if (!(length >= 0.0) || !(length < INFINITY)) return bad(fn, "length is negative or not finite");
    if (length > 0.0 && !(low < high)) return bad(fn, "low must be below high");
    if (i_r == 0) return STADE_HIP_OK;
    if (!freq) return bad(fn, "null output");
    for (int64_t j = 0; j < i_r / 2; ++j) {
        const double f = pow(base, -2.0 * (double)j / (double)i_r);
        double keep = 0.0;   // how much of the pair's own frequency stays
        if (length > 0.0) keep = std::min(1.0, std::max(0.0, (length * f / 6.283185307179586477 - low) / (high - low)));
        freq[j] = f * (keep + (1.0 - keep) / factor);
    }
    return STADE_HIP_OK;
}

int32_t stade_hip_head_rotary(int64_t tx, int64_t tg, void* y, int64_t ldy, const void* x, int64_t ldx, const void* gq, const void* gk,
                              const int64_t* pos, const double* freq, int64_t i_d, int64_t i_q, int64_t i_k, int64_t i_r, int64_t i_t,
                              int64_t half, int64_t norm, double eps, double s, hipStream_t stream) {
    const char* fn = "stade_hip_head_rotary";
    if (int32_t rc = check(fn, tx, tg, gq, gk, i_d, i_q, i_k, i_r, i_t, norm, eps, s)) return rc;
    const int64_t width = i_d * (i_q + i_k);
    if (int32_t rc = check_ld(fn, "ldy", ldy, width)) return rc;
    if (int32_t rc = check_ld(fn, "ldx", ldx, width)) return rc;
    if (width == 0 || i_t == 0) return STADE_HIP_OK;
    if (!y || !x || (i_r > 0 && (!pos || !freq))) return bad(fn, "null pointer");
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    Rot p{x, ldx, y, ldy, nullptr, 0, gq, gk, (int)tg, pos, freq, nullptr, (int)i_d, (int)i_q, (int)i_k, (int)i_r, i_t, 1, log_lanes(tx, i_d, i_r),
          (float)eps, (float)s, 0, 0};
    // (Few tokens: a block for each, and its heads over as many blocks as have work for their lanes.)
    const int64_t lanes = std::max(i_q, i_k) << p.log_lanes;
    const bool few = i_t <= 256;
    p.tile = few ? 1 : tile_of(p, values_of(tx));
    const unsigned parts = few ? (unsigned)std::min<int64_t>((lanes + NT - 1) / NT, 64) : 1;
    const int64_t tiles = (i_t + p.tile - 1) / p.tile;
    unsigned grid;
    share(p, 2 * tiles, tiles, grid);
    return with_form(tx, half, norm, whole_vectors(tx, i_d, i_r), [&](auto t, auto h, auto n, auto w) -> int32_t {
        using T = decltype(t);
        STADE_TIMED("head_rotary", stream,
                    forward_kernel<T, 16 / sizeof(T), decltype(h)::value, decltype(n)::value, decltype(w)::value>
                        <<<dim3(grid, parts), NT, 0, stream>>>(p));
        STADE_LAUNCHED("head_rotary forward_kernel");
        return STADE_HIP_OK;
    });
}

int32_t stade_hip_head_rotary_b(int64_t tx, int64_t tg, const void* yb, int64_t ldyb, const void* x, int64_t ldx, void* xb, int64_t ldxb,
                                const void* gq, float* gqb, const void* gk, float* gkb, const int64_t* pos, const double* freq, int64_t i_d,
                                int64_t i_q, int64_t i_k, int64_t i_r, int64_t i_t, int64_t half, int64_t norm, double eps, double s,
                                int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_head_rotary_b";
    if (int32_t rc = check(fn, tx, tg, gq, gk, i_d, i_q, i_k, i_r, i_t, norm, eps, s)) return rc;
    const int64_t width = i_d * (i_q + i_k);
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, width)) return rc;
    if (norm)
        if (int32_t rc = check_ld(fn, "ldx", ldx, width)) return rc;
    if (xb)
        if (int32_t rc = check_ld(fn, "ldxb", ldxb, width)) return rc;
    if (!norm && (gqb || gkb)) return bad(fn, "weights' shadows without the norm");
    if (i_d == 0) return STADE_HIP_OK;
    const bool some = i_t > 0 && width > 0, sums = gqb || gkb;
    if (some && (!yb || (norm && !x) || (i_r > 0 && (!pos || !freq)))) return bad(fn, "null pointer");
    if (!sums && (!some || !xb)) return STADE_HIP_OK;
    if (!some && add) return STADE_HIP_OK;
    WsCall call(stream, sums);   // (the workspace for the partial sums only)
    if (!call.ok()) return call.error();
    Rot p{x, ldx, xb, ldxb, yb, ldyb, gq, gk, (int)tg, pos, freq, nullptr, (int)i_d, (int)i_q, (int)i_k, (int)i_r, i_t, 1, log_lanes(tx, i_d, i_r),
          (float)eps, (float)s, add != 0, 0};
    p.tile = some ? tile_of(p, values_of(tx)) : 1;
    const int64_t tiles = (i_t + p.tile - 1) / p.tile;
    unsigned grid = 0;
    // (with sums not more blocks than they are added up fast; queries' and keys' shadows each have blocks of their own)
    if (some) share(p, sums ? std::min<int64_t>(2 * tiles, kSumParts) : 2 * tiles, tiles, grid);
    // (as much as the largest call takes, so that any call is captured after an eager one)
    if (sums && !(p.part = (float*)scratch((size_t)(kSumParts + 2) * kMostHead * sizeof(float)))) return scratch_error();
    if (some) {
        const int32_t rc = with_form(tx, half, norm, whole_vectors(tx, i_d, i_r), [&](auto t, auto h, auto n, auto w) -> int32_t {
            using T = decltype(t);
            STADE_TIMED("head_rotary_b", stream,
                        backward_kernel<T, 16 / sizeof(T), decltype(h)::value, decltype(n)::value, decltype(w)::value><<<grid, NT, 0, stream>>>(p));
            STADE_LAUNCHED("head_rotary backward_kernel");
            return STADE_HIP_OK;
        });
        if (rc) return rc;
    }
    if (sums) {
        STADE_TIMED("head_rotary_sum", stream,
                    weight_sum_kernel<<<dim3((unsigned)((i_d + 15) / 16), 2), NT, 0, stream>>>(p.part, some ? p.q_blocks : 0, (int)grid, (int)i_d, gqb, gkb,
                                                                                              add != 0));
        STADE_LAUNCHED("head_rotary weight_sum_kernel");
    }
    return STADE_HIP_OK;
}

}  // extern "C"
