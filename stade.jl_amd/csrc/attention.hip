// Attention over ragged sequences with heads in groups, a sliding window and sinks:
//   y = sum over the seen keys of softmax(s q . k) v,   lse = log sum exp(s q . k)
// One pass over the keys with the running maximum m and sum l of a row's exponentials: a tile of keys whose scores go
// up to m' > m scales what was summed before by exp(m - m').  (The sums are scaled only where some row's maximum grows by
// more than 8 in the exponent of 2; until then exponentials are up to 2^8, which every type holds.  f16 has few exponents below 1, and
// many small weights may make up a row: its exponentials and their sum are 2^7 times as large, so that 2^-31 of a row's largest counts.)
//
// Scores are formed as K Q^T, keys along the registers: a lane has one query and half of a tile's keys, so
// maxima and sums are lane by lane and one exchange of the half waves.  Exponentials are rounded to the
// type (to nearest: like v, they are one factor of a product, whose sum is fp32) and are, as they lie in registers, the other operand of
// V^T P, whose V^T comes from the row-major tile by the transposing LDS read: they never go through LDS.
//
// A block has 128 rows, four waves of 32, which share tiles of 64 keys and values in two buffers.  Where the rows do not make two
// blocks a CU (single tokens, chunks behind a long context) the keys of each go over several blocks, whose maxima, sums and values a
// second launch joins in order.
//
// bf16, heads of 128: 5 sequences of 3300, 32 heads of queries and 8 of keys, a window of 1024: 320 us, 733 TFLOP/s of what is seen; causal
// without a window 952 (the clock then falls to 1.6 GHz).  64 single tokens of 4096 keys, 8 key heads: 228 us, 4.7 TB/s.
#include "attention.hpp"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace stade {
namespace {

using namespace attn;

struct Att {
    void* y; int64_t ldy;
    float* lse;
    const void* q; int64_t ldq;
    const void* k; int64_t ldk;
    const void* v; int64_t ldv;
    Seqs seqs;
    int d, heads;          // of the keys
    float s;               // the scores' factor, made positive (`negate`: q's sign is turned)
    int negate;
    int64_t slots;         // tiles of rows
    int splits;            // blocks that share a tile's keys
    float* part;           // their sums, where there are several: by block and row, d values, the maximum and the sum
};

constexpr float kGrow = 8.f;     // of the maximum, in the exponent of 2, before sums are scaled
// what is added to the exponents (of 2): the largest exponential, 2^(kGrow + kLift), is below f16's 65504
template <class T> constexpr float kLift = std::is_same<T, f16>::value ? 7.f : 0.f;

// a lane's query
struct Row {
    bool here;
    int64_t t;      // column
    int head;
    int pos;        // its key
};
__device__ __forceinline__ Row head_row(const Seq& q, const Seqs& s, int kvh, int r) {
    Row w;
    const int j = r / s.group;
    w.here = j < q.nq;
    w.t = q.q0 + j;
    w.head = kvh * s.group + r - j * s.group;
    w.pos = w.here ? j + q.shift() : -1;
    return w;
}

// The running softmax and the sums of a wave's 32 rows
template <class T, int DT, int NB>
struct Sums {
    static constexpr int DP = DT > 2 ? 128 : 64, FR = DT * 32 / (2 * kCE<T>);
    struct Scores { floatx16 x[NB]; };   // of 32 NB keys
    float m, l;          // of the lane's row: the maximum (raw scores), the lane's share of the sum
    floatx16 o[DT];      // values 32 i + .. of the head by rows of registers, the row by lane
    v4u q[FR];

    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int j = 0; j < 16; ++j) o[i][j] = 0.f;
    }

    __device__ __forceinline__ void scores(Scores& s, const char* kt) const {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s.x[b][j] = 0.f;
#pragma unroll
            for (int f = 0; f < FR; ++f) s.x[b] = multiply<T>(along_head<T, DP>(kt, 32 * b, f), q[f], s.x[b]);
        }
    }

    // what the row at `pos` does not see of the keys from `key` on; p0, p1: the positions of all rows (tiles that every row
    // sees whole need no tests)
    __device__ __forceinline__ void hide(Scores& v, int key, const Seqs& s, int pos, int p0, int p1) const {
        if (!(key + 32 * NB - 1 > p0 || (p1 - key >= s.window && key + 32 * NB > s.sinks))) return;
        const int h = (threadIdx.x & 63) >> 5, high = pos - key - 4 * h, low = high - s.window, sink = s.sinks - key - 4 * h;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int e = 32 * b + 8 * (j >> 2) + (j & 3);
                if (!(e <= high && (e > low || e < sink))) v.x[b][j] = -INFINITY;
            }
    }

    // the maximum with these scores; c = s log2(e)
    __device__ __forceinline__ void raise(const Scores& s, float c) {
        float top = s.x[0][0];
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int j = 0; j < 16; ++j) top = fmaxf(top, s.x[b][j]);
        top = fmaxf(top, other_half(top));
        if (__any((top - m) * c > kGrow)) {   // (m = -Inf, of rows that saw nothing so far, too; NaN: no)
            const float to = fmaxf(m, top), f = to == -INFINITY ? 1.f : __builtin_amdgcn_exp2f((m - to) * c);
            m = to;
            l *= f;
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[i][j] *= f;
        }
    }

    // the order of scores() and add() together, as the compiler is to issue them
    static __device__ __forceinline__ void order() {
        ORDER(kRead, 4);
        ORDER(kValu, 6);
        ORDER(kTrans, 2);
        static_for<NB * FR>([&](auto i) INLINE {
            ORDER(kMfma, 1);
            ORDER(kRead, decltype(i)::value + 4 < NB * FR ? 1 : 2);
            ORDER(kValu, 3);
            ORDER(kTrans, 2);
            ORDER(kValu, 2);
        });
        static_for<NB * kParts<T> * DT>([&](auto) INLINE {
            ORDER(kMfma, 1);
            ORDER(kRead, 2);
            ORDER(kValu, 2);
        });
    }

    // the scores' weights, and the values by them
    __device__ __forceinline__ void add(Scores& s, const char* vt, float c) {
        const float base = (m == -INFINITY ? 0.f : -m * c) + kLift<T>;
        float sum = 0.f;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                s.x[b][j] = __builtin_amdgcn_exp2f(fmaf(s.x[b][j], c, base));
                sum += s.x[b][j];
            }
#pragma unroll
            for (int u = 0; u < kParts<T>; ++u) {
                const v4u p = part_of<T>(s.x[b], u);
#pragma unroll
                for (int i = 0; i < DT; ++i) o[i] = multiply<T>(along_rows<T, DP>(vt, 32 * b + u * 2 * kCE<T>, 32 * i), p, o[i]);
            }
        }
        l += sum;
    }
};

template <class T>
__device__ __forceinline__ void negate_all(v4u* f, int n) {
    const uint32_t bits = sizeof(T) == 4 ? 0x80000000u : 0x80008000u;
    for (int i = 0; i < n; ++i) f[i] ^= bits;
}

// a wave's finished rows: y and lse
template <class T, int DT>
__device__ __forceinline__ void store_rows(const Att& p, const floatx16 (&o)[DT], const Row& w, float m, float l) {
    if (!w.here) return;
    const int h = (threadIdx.x & 63) >> 5;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    T* y = (T*)p.y + w.t * p.ldy + (int64_t)w.head * p.d;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int col = 32 * i + 8 * g + 4 * h;
            store4(y + col, o[i][4 * g] * inv, o[i][4 * g + 1] * inv, o[i][4 * g + 2] * inv, o[i][4 * g + 3] * inv, p.d - col);
        }
    if (p.lse && h == 0) p.lse[w.t * (p.heads * p.seqs.group) + w.head] = l > 0.f ? m * p.s + kLn2 * (__builtin_amdgcn_logf(l) - kLift<T>) : -INFINITY;
}

// One row after the other, from the keys of [from, to) that it sees: done(row, m, l, its two values of the sum).
template <class T, class F>
__device__ __forceinline__ void exact_rows(const Att& p, const Seq& q, int kvh, int r0, int from, int to, F&& done) {
    const float s = p.negate ? -p.s : p.s;
    for (int r = r0; r < r0 + 32; ++r) {
        const Row w = head_row(q, p.seqs, kvh, r);
        if (!w.here) break;
        const Range range = seen_by(p.seqs, w.pos, w.pos);
        const Two x = load_two((const T*)p.q + w.t * p.ldq + (int64_t)w.head * p.d, p.d);
        float m = -INFINITY, l = 0.f;
        Two o{0.f, 0.f};
        for (int part = 0; part < 2; ++part) {
            const int end = min(part ? range.high : range.sinks, to);
            for (int i = max(part ? range.low : 0, from); i < end; ++i) {
                const Two k = load_two((const T*)p.k + (q.k0 + i) * p.ldk + (int64_t)kvh * p.d, p.d);
                const Two v = load_two((const T*)p.v + (q.k0 + i) * p.ldv + (int64_t)kvh * p.d, p.d);
                const float score = dot(x, k) * s;
                if (score == -INFINITY) continue;
                const float top = fmaxf(m, score), f = m == -INFINITY ? 0.f : exp2f((m - top) * kLog2e), e = exp2f((score - top) * kLog2e);
                m = top;
                l = fmaf(l, f, e);
                o.a = fmaf(o.a, f, e * v.a);
                o.b = fmaf(o.b, f, e * v.b);
            }
        }
        done(w, m, l, o);
    }
}

// columns of no sequence: zeros and -Inf
template <class T>
__device__ __forceinline__ void store_nothing(const Att& p, const Seq& q, int kvh, int r0, int rows) {
    for (int r = r0 + threadIdx.x; r < r0 + rows; r += blockDim.x) {
        const Row w = head_row(q, p.seqs, kvh, r);
        if (!w.here) continue;
        for (int i = 0; i < p.d; ++i) ((T*)p.y)[w.t * p.ldy + (int64_t)w.head * p.d + i] = (T)0.f;
        if (p.lse) p.lse[w.t * (p.heads * p.seqs.group) + w.head] = -INFINITY;
    }
}

constexpr int kWideRows = 128, kWideKeys = 64;
constexpr int64_t kSplitBlocks = 1024;

template <class T, int DT, bool DIRECT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void wide_kernel(Att p) {
    constexpr int DP = DT > 2 ? 128 : 64, BN = kWideKeys, TILE = kTile<T, DP, BN>;
    using S = Stage<T, DP, BN, 256, DIRECT>;
    using R = Sums<T, DT, BN / 32>;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];   // two tiles of keys, two of values
    const Seqs& s = p.seqs;
    if (blockIdx.y == 0) check_offsets(s, blockIdx.x, gridDim.x);
    int64_t slot, tile;
    int kvh;
    place_of(blockIdx.x, p.slots, p.heads, slot, kvh);
    // (the last tiles of a sequence, which see the most, first)
    const int j = find_range(s.qstart, s.t, s.group, kWideRows, s.n + 1, slot, tile);
    const Seq q = sequence(s, j - 1);
    const int rows = q.nq * s.group;
    const int tiles = (rows + kWideRows - 1) / kWideRows;
    if (tile >= tiles) return;
    const int r0 = uniform((int)(tiles - 1 - tile) * kWideRows);
    if (!q.real) {
        if (blockIdx.y == 0) store_nothing<T>(p, q, kvh, r0, kWideRows);
        return;
    }
    const int wave = uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63;
    const Row w = head_row(q, s, kvh, r0 + 32 * wave + (lane & 31));
    const int p0 = r0 / s.group + q.shift(), p1 = min(r0 + kWideRows - 1, rows - 1) / s.group + q.shift();
    // this wave's rows
    const int w0 = uniform((r0 + 32 * wave) / s.group + q.shift()), w1 = uniform(min(r0 + 32 * wave + 31, rows - 1) / s.group + q.shift());
    const bool working = r0 + 32 * wave < rows;
    R sums;
    sums.clear();
    row_fragments<T, DT, DIRECT>(sums.q, (const T*)p.q + w.t * p.ldq + (int64_t)w.head * p.d, w.here, p.d);
    if (p.negate) negate_all<T>(sums.q, sums.FR);
    const Range range = seen_by(s, p0, p1);
    const KeyTiles<BN> all(range);
    // this block's share of the tiles of keys
    const int share = (all.count + p.splits - 1) / p.splits, i_first = min((int)blockIdx.y * share, all.count), count = min(share, all.count - i_first);
    if (blockIdx.y > 0 && count <= 0) return;
    const T* k = (const T*)p.k + q.k0 * p.ldk + (int64_t)kvh * p.d;
    const T* v = (const T*)p.v + q.k0 * p.ldv + (int64_t)kvh * p.d;
    const float c = p.s * kLog2e;
    S sk(p.ldk, p.d, threadIdx.x), sv(p.ldv, p.d, threadIdx.x);
    auto load = [&](S& st, const T* from_row, int64_t ld, int i, char* at) INLINE {
        const int key = all.key(i_first + i);
        int from, to;
        tile_rows<BN>(range, key, from, to);
        st.load(from_row + key * ld, from, to, at);
    };
    // Tile i's weights are formed while the matrix cores form tile i + 1's scores (two waves of a SIMD alone do not fill them):
    // keys lie two tiles ahead of the values' sums, values one.
    char* const kt[2] = {lds, lds + TILE};
    char* const vt[2] = {lds + 2 * TILE, lds + 3 * TILE};
    if (count > 0) {
        load(sk, k, p.ldk, 0, kt[0]);
        load(sv, v, p.ldv, 0, vt[0]);
        sk.store(kt[0]);
        sv.store(vt[0]);
        if (count > 1) {
            load(sk, k, p.ldk, 1, kt[1]);
            sk.store(kt[1]);
        }
        if constexpr (DIRECT) wait_loads<0>();
    }
    settle_loads();
    __syncthreads();
    typename R::Scores a, b;
    if (count > 0 && working) sums.scores(a, kt[0]);
    __syncthreads();
    auto step = [&](auto parity, typename R::Scores& now, typename R::Scores& next, int i) INLINE {
        constexpr int P = decltype(parity)::value;
        if (i + 2 < count) load(sk, k, p.ldk, i + 2, kt[P]);
        if (i + 1 < count) load(sv, v, p.ldv, i + 1, vt[1 - P]);
        if (working) {
            sums.hide(now, all.key(i_first + i), s, w.pos, w0, w1);
            sums.raise(now, c);
            sums.scores(next, kt[1 - P]);      // (behind the last tile: of what lies there, for nothing)
            sums.add(now, vt[P], c);
            if constexpr (sizeof(T) == 2) R::order();
        }
        if (i + 2 < count) sk.store(kt[P]);
        if (i + 1 < count) sv.store(vt[1 - P]);
        if constexpr (DIRECT) wait_loads<0>();
        __syncthreads();
    };
    for (int i = 0; i < count; i += 2) {
        step(std::integral_constant<int, 0>{}, a, b, i);
        if (i + 1 < count) step(std::integral_constant<int, 1>{}, b, a, i + 1);
    }
    const float l = sums.l + other_half(sums.l);
    const bool odd = any_not_finite<DT>(sums.o);
    if (p.splits > 1) {
        float* part = p.part + (((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * kWideRows + 32 * wave) * (p.d + 2);
        if (odd) {   // (no row sees a key between the tiles of sinks and those of the window)
            const int from = all.key(i_first), to = all.key(i_first + count - 1) + BN;
            exact_rows<T>(p, q, kvh, r0 + 32 * wave, from, to, [&](const Row& x, float m, float sum, Two o) INLINE {
                float* at = part + (int64_t)((int)(x.t - q.q0) * s.group + x.head - kvh * s.group - (r0 + 32 * wave)) * (p.d + 2);
                store_two(at, o.a, o.b, p.d, false);
                if (lane == 0) {
                    at[p.d] = m;
                    at[p.d + 1] = sum;
                }
            });
            return;
        }
        if (!w.here) return;
        const int h = lane >> 5;
        part += (lane & 31) * (p.d + 2);
#pragma unroll
        for (int i = 0; i < DT; ++i)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = 32 * i + 8 * g + 4 * h;
                store4(part + col, sums.o[i][4 * g], sums.o[i][4 * g + 1], sums.o[i][4 * g + 2], sums.o[i][4 * g + 3], p.d - col);
            }
        if (h == 0) {
            part[p.d] = sums.m == -INFINITY ? sums.m : sums.m * p.s - kLn2 * kLift<T>;
            part[p.d + 1] = l;
        }
        return;
    }
    if (odd) {
        exact_rows<T>(p, q, kvh, r0 + 32 * wave, 0, q.nk, [&](const Row& x, float m, float sum, Two o) INLINE {
            const float inv = sum != 0.f ? 1.f / sum : 0.f;     // (rows that see nothing; a NaN stays one)
            store_two((T*)p.y + x.t * p.ldy + (int64_t)x.head * p.d, o.a * inv, o.b * inv, p.d, false);
            if (p.lse && lane == 0) p.lse[x.t * (p.heads * s.group) + x.head] = sum != 0.f ? m + logf(sum) : -INFINITY;
        });
        return;
    }
    store_rows<T, DT>(p, sums.o, w, sums.m, l);
}

// The blocks' sums of a row joined in order: a wave has four rows, one after the other (eight, in half as many blocks: 16 us for 11 of 240
// blocks' sums)
constexpr int kJoinRows = 16;
template <class T>
__global__ __launch_bounds__(256) void join_kernel(Att p, int64_t blocks) {
    const Seqs& s = p.seqs;
    const int lane = threadIdx.x & 63, wave = uniform((int)(threadIdx.x >> 6));
    const int64_t block = blockIdx.x / (kWideRows / kJoinRows);
    const int first = (int)(blockIdx.x % (kWideRows / kJoinRows)) * kJoinRows + wave;
    int64_t slot, tile;
    int kvh;
    place_of(block, p.slots, p.heads, slot, kvh);
    const int j = find_range(s.qstart, s.t, s.group, kWideRows, s.n + 1, slot, tile);
    const Seq q = sequence(s, j - 1);
    const int rows = q.nq * s.group, tiles = (rows + kWideRows - 1) / kWideRows;
    if (tile >= tiles || !q.real) return;
    const int r0 = (int)(tiles - 1 - tile) * kWideRows;
    // (as the blocks counted them)
    const KeyTiles<kWideKeys> keys(seen_by(s, r0 / s.group + q.shift(), min(r0 + kWideRows - 1, rows - 1) / s.group + q.shift()));
    const int share = (keys.count + p.splits - 1) / p.splits, parts = max(1, share ? (keys.count + share - 1) / share : 1);
    const int64_t next = blocks * kWideRows * (p.d + 2);
    for (int in = first; in < first + kJoinRows; in += 4) {
        const Row w = head_row(q, s, kvh, r0 + in);
        if (!w.here) return;
        const float* part = p.part + (block * kWideRows + in) * (p.d + 2);
        float m = -INFINITY, l = 0.f;
        Two o{0.f, 0.f};
#pragma unroll 4
        for (int n = 0; n < parts; ++n) {
            const float* at = part + n * next;
            const Two v = load_two(at, p.d);
            const float mn = at[p.d], ln = at[p.d + 1], top = fmaxf(m, mn);
            const float f = m == -INFINITY ? 0.f : exp2f((m - top) * kLog2e), e = mn == -INFINITY ? 0.f : exp2f((mn - top) * kLog2e);
            m = top;
            l = fmaf(l, f, ln * e);
            o.a = fmaf(o.a, f, v.a * e);
            o.b = fmaf(o.b, f, v.b * e);
        }
        const float inv = l != 0.f ? 1.f / l : 0.f;     // (a NaN stays one)
        store_two((T*)p.y + w.t * p.ldy + (int64_t)w.head * p.d, o.a * inv, o.b * inv, p.d, false);
        if (p.lse && lane == 0) p.lse[w.t * (p.heads * s.group) + w.head] = l != 0.f ? m + logf(l) : -INFINITY;
    }
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_attention(int64_t tx, void* y, int64_t ldy, float* lse, const void* q, int64_t ldq, const void* k, int64_t ldk, const void* v,
                            int64_t ldv, const int64_t* qstart, const int64_t* kstart, double s, int64_t i_d, int64_t i_q, int64_t i_k,
                            int64_t i_t, int64_t i_tk, int64_t i_n, int64_t window, int64_t sinks, hipStream_t stream) {
    const char* fn = "stade_hip_attention";
    Seqs seqs;
    if (int32_t rc = check_attention(fn, tx, s, i_d, i_q, i_k, i_t, i_tk, i_n, window, sinks, qstart, kstart, seqs)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d * i_q)) return rc;
    if (int32_t rc = check_ld(fn, "ldq", ldq, i_d * i_q)) return rc;
    if (int32_t rc = check_ld(fn, "ldk", ldk, i_d * i_k)) return rc;
    if (int32_t rc = check_ld(fn, "ldv", ldv, i_d * i_k)) return rc;
    const int64_t slots = slots_of(i_t, seqs.group, kWideRows, i_n + 1), blocks = slots * i_k;
    if (int32_t rc = check_extent(fn, "blocks of 128 rows of a key head", blocks, kMostBlocks)) return rc;
    if (i_d == 0 || i_q == 0 || i_t == 0) return STADE_HIP_OK;
    if (!y || !q || (i_tk > 0 && (!k || !v))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    Att p{y, ldy, lse, q, ldq, k, ldk, v, ldv, seqs, (int)i_d, (int)i_k, fabsf(factor(s)), s < 0.0};
    p.seqs.flag = error_flag(call.ws);
    p.slots = slots;
    // Blocks for two rounds of two a CU, eight tiles of keys each (a tile takes a microsecond, the second launch with what it reads
    // some ten; fp32: two tiles, which take twelve each), and no more than 32 (which the second launch reads one after the other).
    // A sequence is taken to be up to twice as long as the mean (one of 131072 keys among 63 of 1000, a token each, is not split: 2360 us,
    // where it alone takes 130 and they 45).  One token of 8192 keys, 8 key heads: 135 us alone, 22 by 16
    // blocks; of 65536: 1167 and 75 by 32; 4 chunks of 512 behind 8192, 4 key heads: 319 and 229 by three; 2 prompts of 300, 2 key
    // heads: 17, and 25 by two; in fp32 3 of 500, 2 key heads, a window of 300: 82 and 43 + 11 by three.
    // (Two slots more than sequences, for columns of none, usually are empty.)
    const int64_t full = std::max<int64_t>(1, (p.slots - 2) * i_k);
    const int64_t longest = std::min({i_tk, 2 * i_tk / std::max<int64_t>(i_n, 1) + 1, (int64_t)seqs.window + kMostSinks + kWideRows});
    p.splits = (int)std::max<int64_t>(1, std::min({kSplitBlocks / full, 2 * kSplitBlocks / blocks, longest / ((tx == STADE_HIP_F32 ? 2 : 8) * kWideKeys), (int64_t)32}));
    // (as much as any call takes, and by each, so that every other is captured after it)
    if (!(p.part = (float*)scratch((size_t)2 * kSplitBlocks * kWideRows * (kMostHead + 2) * 4))) return scratch_error();
    return with_type(tx, [&](auto t) -> int32_t {
        return with_width(i_d, [&](auto dt) -> int32_t {
            using T = decltype(t);
            constexpr int DT = decltype(dt)::value;
            const int64_t size = sizeof(T);
            const bool direct = straight(q, ldq, i_d, size) && straight(k, ldk, i_d, size) && straight(v, ldv, i_d, size);
            STADE_TIMED("attention", stream, {
                if (direct) wide_kernel<T, DT, true><<<dim3((unsigned)blocks, p.splits), 256, 0, stream>>>(p);
                else wide_kernel<T, DT, false><<<dim3((unsigned)blocks, p.splits), 256, 0, stream>>>(p);
            });
            STADE_LAUNCHED("attention wide_kernel");
            if (p.splits > 1) {
                STADE_TIMED("attention_join", stream, join_kernel<T><<<(unsigned)(blocks * (kWideRows / kJoinRows)), 256, 0, stream>>>(p, blocks));
                STADE_LAUNCHED("attention join_kernel");
            }
            return STADE_HIP_OK;
        });
    });
}

}  // extern "C"
