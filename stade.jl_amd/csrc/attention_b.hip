// The adjoint of attention.  With P = exp(s q . k - lse) over the seen keys, the rows as in the forward sweep (query after query
// with the heads of a group side by side), and delta = yb . y for each row:
//   vb (+)= P^T yb,   S = P (yb v^T - delta),   qb (+)= s S k,   kb (+)= s S^T q
// P is formed again from lse; nothing of the size of the scores is kept.  Two launches, and up to three more (below):
//   rows_kernel   a block has 128 rows and goes over their keys: qb, and delta as the sum of P (yb v^T).  Scores as keys x rows, so that
//                 lse and delta are one value a lane, and S, rounded, is the operand of K^T S as it lies.
//   keys_kernel   a block has 128 keys and goes over the rows that see them, all heads of the group: kb and vb.  Scores as
//                 rows x keys; P and S are the operands of yb^T P and q^T S as they lie.
// That forms the scores and yb v^T twice, 7 products for 5, and needs no atomics: each result has one writer, its
// sums go in a fixed order, and the same call gives the same bits.
// Sinks are seen by every later row: rows past the window of the first tile of keys go over blocks of their own (a launch), which leave
// partial sums; far_kernel joins them, and the tile's block adds them.  Tiles of keys that fill no round of the CUs go over several
// blocks, which join_kernel joins.
// 4 sequences of 2048, 16 heads of 128 and 4 of keys, a window of 1024, 4 sinks, bf16: rows 121 us, keys 194, sinks 31, joins 9: some 590
// TFLOP/s of the products formed for what is seen.  f16 pays for the powers of two (below) with some 15 us of the rows', 7 of the
// keys' and 2 of the sinks'.
// Sums are fp32; P and S are rounded to the type as factors of products (to nearest), as the values they meet are; in f16 times powers of two.
#include "attention.hpp"

#include <algorithm>
#include <math.h>
#include <type_traits>

namespace stade {
namespace {

using namespace attn;

struct Back {
    const void* yb; int64_t ldyb;
    const void* y; int64_t ldy;
    const float* lse;
    const void* q; int64_t ldq;
    void* qb; int64_t ldqb;
    const void* k; int64_t ldk;
    void* kb; int64_t ldkb;
    const void* v; int64_t ldv;
    void* vb; int64_t ldvb;
    float* delta;          // by (head, column), as lse
    Seqs seqs;
    int d, heads;          // of the keys
    float s;
    int add;
    float factor;          // of the scores: s, not 0
    int64_t slots;
    uint32_t magic;        // ceil(2^31 / group)
    float* far;            // partial sums of the sinks; null: none
    int far_parts;
    int64_t whole;         // tiles of keys that a block has alone; the others go over `splits` blocks each
    int splits;
    float* part;           // those blocks' sums
    float* most;           // f16: what the S of each 32 rows are below
};

constexpr int kRows = 128, kKeys = 128;
constexpr int kFewTiles = 4;      // of keys, where delta is formed from the weights

// ------------------------------------------------------------------------------------------
// factors in f16
// ------------------------------------------------------------------------------------------
// f16 holds 2^-24 to 65504.  P is 1 / keys and S = P (yb v^T - delta) a shadow's size of that, or far above 65504: rounded as they are, they
// vanish or overflow where the results, sums of thousands of them, do not.  So for kb and vb P stands for P 2^14, by its exponent, and S
// for that by 2^k, k from the largest S of the block's rows, which rows_kernel leaves; and for qb S stands for S 2^k, k of each row by
// itself: its largest S so far is below 2^15, and sums are scaled where a larger one comes, as the forward sweep's are.  S of
// 2^-36 of the largest and more counts, and any of 2^-55 (which no sum of f16's values makes a value of).
template <class T> constexpr bool kNarrow = std::is_same<T, f16>::value;
template <class T> constexpr int kWeightLift = kNarrow<T> ? 14 : 0;
constexpr int kMostLift = 32;     // of a row whose S are all below 2^-17 so far
__device__ __forceinline__ float power(int k) { return __builtin_amdgcn_ldexpf(1.f, k); }

// where what the S of the 32 rows from r on of a key head are below is (sequence i): as many places as rows_kernel's waves have
__device__ __forceinline__ int64_t most_at(const Seqs& s, int i, int r, int heads, int kvh) {
    return ((first_slot(s.qstart, s.t, s.group, kRows, i + 1) + r / kRows) * heads + kvh) * (kRows / 32) + r % kRows / 32;
}
// k for the rows [r, end): their S are below 2^14 (and yb v^T - delta, rounded another way here, may be larger where it is next
// to 0), times 2^kWeightLift as P has it
template <class T>
__device__ __forceinline__ int lift_of(const float* most, const Seqs& s, int i, int r, int end, int heads, int kvh) {
    float top = 0.f;
    for (int w = r / 32 + (int)(threadIdx.x & 63); 32 * w < end; w += 64) {
        const float v = most[most_at(s, i, 32 * w, heads, kvh)];
        if (v < INFINITY) top = fmaxf(top, v);     // (what is not finite makes sums that are formed again)
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor(top, o, 64));
    return uniform(14 - __builtin_amdgcn_frexp_expf(top) - kWeightLift<T>);
}

// ------------------------------------------------------------------------------------------
// qb, and delta
// ------------------------------------------------------------------------------------------
template <class T, int DT, bool DIRECT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void rows_kernel(Back p) {
    constexpr int DP = DT > 2 ? 128 : 64, BN = sizeof(T) == 2 ? 64 : 32, NB = BN / 32, TILE = kTile<T, DP, BN>, FR = DT * 32 / (2 * kCE<T>);
    using S = Stage<T, DP, BN, 256, DIRECT>;
    __shared__ __attribute__((aligned(1024))) char lds[4 * TILE];
    const Seqs& s = p.seqs;
    check_offsets(s, blockIdx.x, gridDim.x);
    int64_t slot, tile;
    int kvh;
    place_of(blockIdx.x, p.slots, p.heads, slot, kvh);
    const int j = find_range(s.qstart, s.t, s.group, kRows, s.n + 1, slot, tile);
    const Seq q = sequence(s, j - 1);
    const int rows = q.nq * s.group, tiles = (rows + kRows - 1) / kRows;
    if (tile >= tiles) return;
    const int r0 = uniform((int)(tiles - 1 - tile) * kRows);
    const int wave = uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, h = lane >> 5;
    const int r = r0 + 32 * wave + (lane & 31), jq = r / s.group, head = kvh * s.group + r - jq * s.group;
    const bool here = jq < q.nq, working = r0 + 32 * wave < rows;
    const int64_t t = q.q0 + jq, col = (int64_t)head * p.d;
    const int pos = here && q.real ? jq + q.shift() : -1;
    v4u qf[FR], of[FR];
    float lse = here ? p.lse[t * (p.heads * s.group) + head] : 0.f, delta = 0.f;
    {
        v4u yf[FR];
        row_fragments<T, DT, DIRECT>(of, (const T*)p.yb + t * p.ldyb + col, here, p.d);
        row_fragments<T, DT, DIRECT>(yf, (const T*)p.y + t * p.ldy + col, here, p.d);
        typedef T vec __attribute__((ext_vector_type(kCE<T>)));
#pragma unroll
        for (int f = 0; f < FR; ++f) {
            const vec a = __builtin_bit_cast(vec, of[f]), b = __builtin_bit_cast(vec, yf[f]);
#pragma unroll
            for (int i = 0; i < kCE<T>; ++i) delta = fmaf((float)a[i], (float)b[i], delta);
        }
        delta += other_half(delta);
    }
    row_fragments<T, DT, DIRECT>(qf, (const T*)p.q + t * p.ldq + col, here, p.d);
    const int p0 = r0 / s.group + q.shift(), p1 = min(r0 + kRows - 1, rows - 1) / s.group + q.shift();
    const int w0 = uniform((r0 + 32 * wave) / s.group + q.shift()), w1 = uniform(min(r0 + 32 * wave + 31, rows - 1) / s.group + q.shift());
    Range range = seen_by(s, p0, p1), mine = seen_by(s, w0, w1);
    if (!q.real) range = mine = Range{0, 0, 0};
    const KeyTiles<BN> keys(range);
    const T* k = (const T*)p.k + q.k0 * p.ldk + (int64_t)kvh * p.d;
    const T* v = (const T*)p.v + q.k0 * p.ldv + (int64_t)kvh * p.d;
    const float c = p.factor * kLog2e, base = -lse * kLog2e;
    int lift = kMostLift;
    floatx16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    S sk(p.ldk, p.d, threadIdx.x), sv(p.ldv, p.d, threadIdx.x);
    auto load = [&](int i, char* at) INLINE {
        const int key = keys.key(i);
        int from, to;
        tile_rows<BN>(range, key, from, to);
        sk.load(k + key * p.ldk, from, to, at);
        sv.load(v + key * p.ldv, from, to, at + TILE);
    };
    // yb . y is delta but for y's rounding, which few keys do not make small beside the differences yb v^T - delta (y is as large as they
    // are: qb of 16-bit types would be off by 1.7 of the plain form's error, not 1.4).  There a pass before forms it from P and yb v^T;
    // kb gets it so in any case.
    const bool exact = sizeof(T) == 2 && keys.count <= kFewTiles;
    float sum = 0.f;
    for (int pass = exact ? 0 : 1; pass < 2; ++pass) {
        if (keys.count > 0) {
            load(0, lds);
            sk.store(lds);
            sv.store(lds + TILE);
            if constexpr (DIRECT) wait_loads<0>();
        }
        settle_loads();
        __syncthreads();
        for (int i = 0; i < keys.count; ++i) {
            char* now = lds + (i & 1) * 2 * TILE;
            char* next = lds + (~i & 1) * 2 * TILE;
            if (i + 1 < keys.count) load(i + 1, next);
            const int key = keys.key(i);
            if (working && ((key < mine.high && key + BN > mine.low) || key < mine.sinks)) {
                const bool whole = key + BN - 1 <= w0 && (w1 - key < s.window || key + BN <= s.sinks);
                const int high = pos - key - 4 * h, low = high - s.window, sink = s.sinks - key - 4 * h;
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const float lift_by = power(lift);
                    floatx16 x, g;
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = g[e] = 0.f;
#pragma unroll
                    for (int f = 0; f < FR; ++f) x = multiply<T>(along_head<T, DP>(now, 32 * b, f), qf[f], x);
#pragma unroll
                    for (int f = 0; f < FR; ++f) g = multiply<T>(along_head<T, DP>(now + TILE, 32 * b, f), of[f], g);
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, base));
                    if (!whole) {
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int at = 32 * b + 8 * (e >> 2) + (e & 3);
                            if (!(at <= high && (at > low || at < sink))) x[e] = 0.f;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        sum = fmaf(x[e], g[e], sum);
                        x[e] *= kNarrow<T> ? fmaf(g[e], lift_by, -delta * lift_by) : g[e] - delta;
                    }
                    if (pass) {
                        if constexpr (kNarrow<T>) {
                            float top = 0.f;
#pragma unroll
                            for (int e = 0; e < 16; ++e) top = fmaxf(top, fabsf(x[e]));    // (NaN and Inf make sums that are formed again)
                            top = fmaxf(top, other_half(top));
                            if (__any(top > 0x1p15f)) {
                                const int less = top > 0x1p15f ? max(__builtin_amdgcn_frexp_expf(top) - 14, 0) : 0;   // (to 2^13 .. 2^14)
                                const float f = power(-less);
                                lift -= less;
#pragma unroll
                                for (int e = 0; e < 16; ++e) x[e] *= f;
#pragma unroll
                                for (int m = 0; m < DT; ++m)
#pragma unroll
                                    for (int e = 0; e < 16; ++e) acc[m][e] *= f;
                            }
                        }
#pragma unroll
                        for (int u = 0; u < kParts<T>; ++u) {
                            const v4u part = part_of<T>(x, u);
#pragma unroll
                            for (int m = 0; m < DT; ++m) acc[m] = multiply<T>(along_rows<T, DP>(now, 32 * b + u * 2 * kCE<T>, 32 * m), part, acc[m]);
                        }
                    }
                }
            }
            if (i + 1 < keys.count) {
                sk.store(next);
                sv.store(next + TILE);
                if constexpr (DIRECT) wait_loads<0>();
            }
            __syncthreads();
        }
        if (!pass) {
            delta = sum + other_half(sum);
            sum = 0.f;
        }
    }
    sum += other_half(sum);
    float most = 0.f;
    if constexpr (kNarrow<T>) {
        const float moved = fabsf(sum - delta);      // (keys_kernel has the sum)
        most = power(15 - lift) + (moved < INFINITY ? moved : 0.f);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) most = fmaxf(most, __shfl_xor(most, o, 64));
    }
    auto leave_most = [&]() INLINE {
        if constexpr (kNarrow<T>)
            if (working && q.real && lane == 0) p.most[most_at(s, j - 1, r0 + 32 * wave, p.heads, kvh)] = most;
    };
    if (here && h == 0) p.delta[t * (p.heads * s.group) + head] = sum;
    // (what is not finite: products with what is not seen among it.  Of what is seen, it reaches the other keys by y alone.)
    if (any_not_finite<DT>(acc) || __any(here && sum * 0.f != 0.f)) {
        for (int i = 0; i < 32; ++i) {
            const int ri = r0 + 32 * wave + i, ji = ri / s.group, hi = kvh * s.group + ri - ji * s.group;
            if (ji >= q.nq) break;
            const Range seen = seen_by(s, ji + q.shift(), ji + q.shift());
            const int64_t ti = q.q0 + ji, ci = (int64_t)hi * p.d, at = ti * (p.heads * s.group) + hi;
            const Two x = load_two((const T*)p.q + ti * p.ldq + ci, p.d), g = load_two((const T*)p.yb + ti * p.ldyb + ci, p.d);
            const float li = p.lse[at];
            float di = 0.f, a = 0.f, b = 0.f;
            for (int step = 0; step < 2; ++step) {
                if (step == 1 && di * 0.f != 0.f) di = dot(g, load_two((const T*)p.y + ti * p.ldy + ci, p.d));
                for (int part = 0; part < 2; ++part) {
                    const int end = part ? seen.high : seen.sinks;
                    for (int n = part ? seen.low : 0; n < end; ++n) {
                        const Two kn = load_two(k + n * p.ldk, p.d), vn = load_two(v + n * p.ldv, p.d);
                        const float w = exp2f((dot(x, kn) * p.s - li) * kLog2e), gv = dot(g, vn);
                        if (step == 0) {
                            di = fmaf(w, gv, di);
                        } else {
                            a = fmaf(w * (gv - di), kn.a, a);
                            b = fmaf(w * (gv - di), kn.b, b);
                            if (kNarrow<T> && fabsf(w * (gv - di)) < INFINITY) most = fmaxf(most, fabsf(w * (gv - di)));
                        }
                    }
                }
            }
            if (lane == 0) p.delta[at] = di;
            if (!p.qb) continue;
            store_two((T*)p.qb + ti * p.ldqb + ci, a * p.s, b * p.s, p.d, p.add);
        }
        leave_most();
        return;
    }
    leave_most();
    if (!here || !p.qb) return;
    T* out = (T*)p.qb + t * p.ldqb + col;
    const float by = power(-lift);     // (of f16: what the factors were multiplied by)
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * m + 8 * g + 4 * h;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = (kNarrow<T> ? acc[m][4 * g + e] * by : acc[m][4 * g + e]) * p.s;
            store4(out + at, v[0], v[1], v[2], v[3], p.d - at, p.add);
        }
}

// ------------------------------------------------------------------------------------------
// kb and vb
// ------------------------------------------------------------------------------------------
// A block's waves: kGroups of 32 keys by kRowWaves, each with kBlocks of 32 rows of a tile.  16-bit types: four by one with two
// blocks side by side, one wave a SIMD, whose 512 registers hold its keys and values, the sums and both blocks' scores; one
// block's exponentials lie between the other's products.  (Two waves a SIMD, one block each, have no room for the values, and read LDS half
// as often again.)  fp32: four by one, a block.  FAR: one by four (fp32 two), a block, see below.
template <class T, bool FAR> constexpr int kGroups = FAR ? 1 : 4;
template <class T, bool FAR> constexpr int kRowWaves = FAR ? (sizeof(T) == 2 ? 4 : 2) : 1;
template <class T, bool FAR> constexpr int kBlocks = FAR ? 1 : sizeof(T) == 2 ? 2 : 1;
template <class T, bool FAR> constexpr int kTileRows = 32 * kRowWaves<T, FAR> * kBlocks<T, FAR>;

// x / group for small x, by the reciprocal (off by less than x 2^-31: exact for x below 2^31 / group, and here x is
// below group + 64)
__device__ __forceinline__ uint32_t by_group(uint32_t x, uint32_t magic) { return __umulhi(2 * x, magic); }

// Rows of a sequence in LDS: q or yb of the (query, head) pairs from one on, heads side by side.  Which of its values a thread
// loads depends on the first row's head, and not on that where a tile has whole queries.  Their addresses grow row by
// row: the rows behind the last lie past the buffer's end, and become zeros.
template <class T, int DP, int ROWS, int NT, bool DIRECT>
struct RowStage {
    static constexpr int CPR = kRow<T, DP> / 16, PER = ROWS * CPR / NT;
    static_assert(ROWS * CPR % NT == 0, "whole chunks a thread");
    uint32_t off[DIRECT ? PER : 1];
    v4u held[DIRECT ? 1 : PER];
    const T* p;      // the tile's first row's query, head 0 of the group
    uint32_t bytes;  // from there to the last row's end
    int rem, rows;   // the first row's head; rows

    // the chunks' places for a first row of head `rem_`
    __device__ __forceinline__ void places(int64_t ld, int d, int group, uint32_t magic, int rem_) {
        rem = rem_;
        if constexpr (DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int place = i * NT + threadIdx.x, o = place / CPR, c = (place % CPR) ^ turn<T, DP>(o);
                const uint32_t x = rem + o, jq = by_group(x, magic), hd = x - jq * group;
                off[i] = c * kCE<T> < d ? (jq * (uint32_t)ld + hd * d + c * kCE<T>) * (uint32_t)sizeof(T) : 0x80000000u;
            }
        }
    }
    __device__ __forceinline__ void tile(const T* p_, int64_t ld, int d, int group, uint32_t magic, int rows_) {
        p = p_;
        rows = rows_;
        const uint32_t x = rem + max(rows - 1, 0), jq = by_group(x, magic), hd = x - jq * group;
        bytes = rows > 0 ? (uint32_t)uniform((int)((jq * (uint32_t)ld + hd * d + d) * (uint32_t)sizeof(T))) : 0;
    }
    template <int I>
    __device__ __forceinline__ void load(int64_t ld, int d, int group, uint32_t magic, const char* lds) {
        if constexpr (DIRECT) {
            const uint64_t base = (uint64_t)p;
            const v4u r = {(uint32_t)uniform((int)(uint32_t)base), (uint32_t)uniform((int)((uint32_t)(base >> 32) & 0xffffu)), bytes, 0x00020000u};
            const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds + uniform((int)(threadIdx.x >> 6)) * (1024 + kPad<T>);
            load_to_lds(r, off[I], at + I * (NT / 64) * (1024 + kPad<T>));
        } else {
            const int place = I * NT + threadIdx.x, o = place / CPR, c = (place % CPR) ^ turn<T, DP>(o);
            const uint32_t x = rem + o, jq = by_group(x, magic), hd = x - jq * group;
            held[I] = load_chunk(p + (int64_t)jq * ld + hd * d + c * kCE<T>, o < rows ? d - c * kCE<T> : 0);
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) *reinterpret_cast<v4u*>(lds + place_at<T>(i * NT + threadIdx.x)) = held[i];
        }
    }
};

// What a block of keys_kernel works on, and where the rows' range is cut
struct KeyTile {
    Seq q;
    int64_t first;       // of the sequence's (or of no sequence's) key columns
    int keys, key0;      // how many they are; the tile's first
    int r_first, r_end;  // the rows that see it, without those past the window of a first tile
    int far_rows;        // those
};
__device__ __forceinline__ KeyTile key_tile(const Seqs& s, int j, int64_t tile) {
    KeyTile k;
    k.first = j == 0 ? 0 : clamped(s.kstart[j - 1], s.tk);
    k.keys = (int)max((j > s.n ? s.tk : clamped(s.kstart[j], s.tk)) - k.first, (int64_t)0);
    k.key0 = (int)min(tile * kKeys, (int64_t)k.keys);
    k.q = sequence(s, j - 1);
    const int64_t last = (int64_t)k.key0 + kKeys - 1 + s.window - 1;    // the last position whose window has a key of the tile
    const int j0 = max(k.key0 - k.q.shift(), 0), j1 = k.q.real ? (int)min((int64_t)k.q.nq, max(last + 1 - k.q.shift(), (int64_t)0)) : 0;
    k.r_first = j0 * s.group;
    k.r_end = max(j1, j0) * s.group;
    k.far_rows = k.q.real ? (k.q.nq - j1) * s.group : 0;
    return k;
}
// rows of a part, of `parts` that a range is cut into: whole tiles of BM
__device__ __forceinline__ int part_rows(int rows, int parts, int BM) { return (rows / parts / BM + 1) * BM; }

// A split block's sums, and a far block's: (kb, vb) of its keys, d values each, one key after the other
template <bool SCALED, int DT>
__device__ __forceinline__ void store_part(float* out, int d, const floatx16 (&a)[DT], float by) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * m + 8 * g + 4 * h;
            float v[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = SCALED ? a[m][4 * g + e] * by : a[m][4 * g + e];
            store_row(out + at, v, d - at);
        }
}

// FAR: rows past the first tile's window, which see its sinks only; block (part, sequence, head, 32 of the sinks).  Its waves have
// the same keys and other rows.
template <class T, int DT, bool DIRECT, bool FAR>
__global__ __launch_bounds__((64 * kGroups<T, FAR> * kRowWaves<T, FAR>), (sizeof(T) == 2 && DT == 2 && !FAR ? 2 : 1)) void keys_kernel(Back p) {
    constexpr int DP = DT > 2 ? 128 : 64, KG = kGroups<T, FAR>, RG = kRowWaves<T, FAR>, RB = kBlocks<T, FAR>, NT = 64 * KG * RG, BM = kTileRows<T, FAR>;
    constexpr int TILE = kTile<T, DP, BM>, FR = DT * 32 / (2 * kCE<T>), STATS = 2 * BM * 4, BUF = 2 * TILE;
    static_assert(FAR || KG * 32 == kKeys, "the waves' keys make a tile");
    using S = RowStage<T, DP, BM, NT, DIRECT>;
    // two tiles of rows of q and of yb, and the rows' lse and delta
    __shared__ __attribute__((aligned(1024))) char lds[2 * BUF + 2 * STATS];
    char* const st = lds + 2 * BUF;
    const Seqs& s = p.seqs;
    int64_t slot, tile;
    int kvh, j, split = -1, far32 = 0;
    if constexpr (FAR) {
        const int64_t b = blockIdx.x / p.far_parts;
        tile = blockIdx.x % p.far_parts;
        kvh = (int)(b % p.heads);
        j = (int)(b / p.heads) + 1;
        far32 = 32 * blockIdx.y;
    } else {
        int64_t unit = blockIdx.x;
        if (unit >= p.whole) {
            split = (int)((unit - p.whole) % p.splits);
            unit = p.whole + (unit - p.whole) / p.splits;
        }
        place_of(unit, p.slots, p.heads, slot, kvh);
        j = find_range(s.kstart, s.tk, 1, kKeys, s.n + 1, slot, tile);
    }
    const int wave = uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, h = lane >> 5;
    const KeyTile kt = key_tile(s, j, FAR ? 0 : tile);
    const Seq& q = kt.q;
    const int keys = kt.keys, key0 = kt.key0, shift = q.shift();
    if (key0 >= keys) return;
    int r_first = kt.r_first, r_end = kt.r_end;
    const int far_step = p.far_parts ? part_rows(kt.far_rows, p.far_parts, BM) : 0;
    if constexpr (FAR) {
        r_first = r_end + (int)tile * far_step;
        r_end = min(r_first + far_step, q.nq * s.group);
        if (!q.real || r_first >= r_end) return;
    } else if (split >= 0) {
        const int step = part_rows(r_end - r_first, p.splits, BM);
        r_first += split * step;
        r_end = min(r_first + step, r_end);
        if (r_first >= r_end) return;
    }
    const int group = wave % KG, first_row = 32 * RB * (wave / KG);                     // the wave's rows of a tile
    const int own = FAR ? far32 : key0 + 32 * group, key = own + (lane & 31);      // its keys, and the lane's
    const int64_t kcol = kt.first + key, hcol = (int64_t)kvh * p.d;
    const bool here = key < keys, working = own < keys && (!FAR || own < s.sinks);
    v4u kf[FR], vf[FR];
    row_fragments<T, DT, DIRECT>(kf, (const T*)p.k + kcol * p.ldk + hcol, here, p.d);
    row_fragments<T, DT, DIRECT>(vf, (const T*)p.v + kcol * p.ldv + hcol, here, p.d);
    floatx16 ka[DT], va[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) ka[i][e] = va[i][e] = 0.f;
    const float c = p.factor * kLog2e;
    const int lift = kNarrow<T> && q.real ? lift_of<T>(p.most, s, j - 1, r_first, r_end, p.heads, kvh) : 0;
    const float lift_by = power(lift);
    const int heads = p.heads * s.group, tiles = r_end > r_first ? (r_end - r_first + BM - 1) / BM : 0;
    // (the query and the head in its group of a tile's first row: of the one at work and of the one on its way)
    int now_j = uniform(r_first / s.group), now_h = uniform(r_first - now_j * s.group), next_j = now_j, next_h = now_h;
    S sq, so;
    float stat = 0.f;
    sq.places(p.ldq, p.d, s.group, p.magic, now_h);
    so.places(p.ldyb, p.d, s.group, p.magic, now_h);
    const bool fixed = BM % s.group == 0;      // (tiles of whole queries)
    const float per_s = -1.f / p.factor;
    auto aim = [&](int i) INLINE {             // at tile i (behind the last: no rows)
        const int64_t t = q.q0 + next_j, head = (int64_t)kvh * s.group;
        const int rows = min(BM, r_end - (r_first + i * BM));
        if (!fixed) {
            sq.places(p.ldq, p.d, s.group, p.magic, next_h);
            so.places(p.ldyb, p.d, s.group, p.magic, next_h);
        }
        sq.tile((const T*)p.q + t * p.ldq + head * p.d, p.ldq, p.d, s.group, p.magic, rows);
        so.tile((const T*)p.yb + t * p.ldyb + head * p.d, p.ldyb, p.d, s.group, p.magic, rows);
        if (threadIdx.x < 2 * BM) {            // lse and delta, one a thread (rows that are not: no weight)
            const int o = threadIdx.x % BM;
            const uint32_t x = next_h + o, jo = by_group(x, p.magic);
            const int64_t at = (t + jo) * heads + head + (x - jo * s.group);
            const bool first = threadIdx.x < BM;
            stat = first ? INFINITY : 0.f;
            if (o < rows) stat = first ? p.lse[at] : p.delta[at];
        }
    };
    constexpr int CHUNKS = 2 * S::PER;         // of a thread, q's and yb's
    auto load = [&](auto piece, char* at) INLINE {
        constexpr int N = decltype(piece)::value;
        if constexpr (N < S::PER) sq.template load<N>(p.ldq, p.d, s.group, p.magic, at);
        else so.template load<N - S::PER>(p.ldyb, p.d, s.group, p.magic, at + TILE);
    };
    auto load_all = [&](char* at) INLINE { static_for<CHUNKS>([&](auto n) INLINE { load(n, at); }); };
    // The products start from what belongs to a row: yb v^T from -delta, scores of 16-bit types from -lse / s (in fp32 the sum would lose by
    // it: they start from zero, and -lse comes behind).
    constexpr bool FROM_LSE = sizeof(T) == 2;
    auto keep = [&](int i, char* at) INLINE {
        sq.store(at);
        so.store(at + TILE);
        if (threadIdx.x < 2 * BM)
            reinterpret_cast<float*>(st + (i & 1) * STATS)[threadIdx.x] =
                threadIdx.x < BM ? (stat - kLn2 * kWeightLift<T>) * (FROM_LSE ? per_s : -kLog2e) : -stat;
        if constexpr (DIRECT) wait_loads<0>();
    };
    if (tiles > 0) {
        aim(0);
        load_all(lds);
        keep(0, lds);
    }
    settle_loads();
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
        const char* now = lds + (i & 1) * BUF;
        char* next = lds + (~i & 1) * BUF;
        const int step = (int)by_group(now_h + BM, p.magic);
        next_j = now_j + step;
        next_h = now_h + BM - step * s.group;
        aim(i + 1);
        const int end = min(first_row + 32 * RB, r_end - (r_first + i * BM)) - 1;
        const int pa = uniform(now_j + (int)by_group(now_h + first_row, p.magic) + shift), pb = uniform(now_j + (int)by_group(now_h + max(end, 0), p.magic) + shift);
        const bool whole = (own + 31 <= pa) & ((pb - own < s.window) | (own + 31 < s.sinks));
        if (working && end >= first_row && pb >= own && (pa - (own + 31) < s.window || own < s.sinks)) {
            const float* stats = reinterpret_cast<const float*>(st + (i & 1) * STATS) + first_row;
            const char* qt = now + row_at<T, DP>(first_row);
            const char* yt = qt + TILE;
            constexpr int PU = kParts<T>, PER = PU * DT;      // parts of a result; products by them
            floatx16 x[RB], g[RB];
            auto start = [&](floatx16& v, int at) INLINE {
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                    const v4f a = *reinterpret_cast<const v4f*>(stats + at + 8 * m + 4 * h);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[4 * m + e] = a[e];
                }
            };
            // The scores block by block, then yb v^T.  Between the first block's products go the loads of the next tile, between all that
            // follow the exponentials, none before its scores are there.
            if constexpr (FROM_LSE) {
                start(x[0], 0);
            } else {
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) x[b][e] = 0.f;
            }
            products<2 * RB * FR, 6>(
                [&](auto n) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / FR;
                    return along_head<T, DP>(PH < RB ? qt : yt, 32 * (PH % RB), N % FR);
                },
                [&](auto n, const v4u& f) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / FR;
                    if constexpr (PH < RB) x[PH] = multiply<T>(f, kf[N % FR], x[PH]);
                    else g[PH - RB] = multiply<T>(f, vf[N % FR], g[PH - RB]);
                },
                [&](auto n) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / FR, F = N % FR;
                    if constexpr (PH == 0) {
                        constexpr int FROM = F * CHUNKS / FR;
                        static_for<(F + 1) * CHUNKS / FR - FROM>([&](auto k) INLINE { load(std::integral_constant<int, FROM + decltype(k)::value>{}, next); });
                    }
                    if constexpr (F == FR - 3 && PH + 1 < 2 * RB) {
                        if constexpr (PH + 1 >= RB) start(g[PH + 1 - RB], BM + 32 * (PH + 1 - RB));
                        else if constexpr (FROM_LSE) start(x[PH + 1], 32 * (PH + 1));
                    }
                    if constexpr (N > FR) {
                        constexpr int STEPS = (2 * RB - 1) * FR - 1, FROM = (N - FR - 1) * 16 * RB / STEPS;
                        static_for<(N - FR) * 16 * RB / STEPS - FROM>([&](auto k) INLINE {
                            constexpr int E = FROM + decltype(k)::value;
                            const float l = FROM_LSE ? 0.f : stats[32 * (E / 16) + 8 * (E % 16 / 4) + 4 * h + E % 4];
                            x[E / 16][E % 16] = __builtin_amdgcn_exp2f(FROM_LSE ? x[E / 16][E % 16] * c : fmaf(x[E / 16][E % 16], c, l));
                        });
                    }
                });
            if (!whole) {
#pragma unroll
                for (int b = 0; b < RB; ++b)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int pos = now_j + (int)by_group(now_h + first_row + 32 * b + 4 * h + 8 * (e >> 2) + (e & 3), p.magic) + shift;
                        if (!((key <= pos) & ((pos - key < s.window) | (key < s.sinks)))) x[b][e] = g[b][e] = 0.f;
                    }
            }
            // vb's products block by block, and between them S = P (yb v^T - delta); then kb's
            v4u w[RB * PU];
#pragma unroll
            for (int b = 0; b < RB; ++b)
#pragma unroll
                for (int u = 0; u < PU; ++u) w[b * PU + u] = part_of<T>(x[b], u);
            products<2 * RB * PER, 4>(
                [&](auto n) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / PER, U = N % PER / DT, M = N % DT;
                    return along_rows<T, DP>(PH < RB ? yt : qt, 32 * (PH % RB) + U * 2 * kCE<T>, 32 * M);
                },
                [&](auto n, const v4u& f) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / PER, U = N % PER / DT, M = N % DT;
                    if constexpr (PH < RB) va[M] = multiply<T>(f, w[PH * PU + U], va[M]);
                    else ka[M] = multiply<T>(f, w[(PH - RB) * PU + U], ka[M]);
                },
                [&](auto n) INLINE {
                    constexpr int N = decltype(n)::value, PH = N / PER, F = N % PER, FROM = F * 16 / PER;
                    if constexpr (PH < RB) {
                        static_for<(F + 1) * 16 / PER - FROM>([&](auto k) INLINE {
                            constexpr int E = FROM + decltype(k)::value;
                            x[PH][E] *= kNarrow<T> ? g[PH][E] * lift_by : g[PH][E];
                        });
                        if constexpr (F == PER - 1) {
#pragma unroll
                            for (int u = 0; u < PU; ++u) w[PH * PU + u] = part_of<T>(x[PH], u);
                        }
                    }
                });
        } else {
            load_all(next);
        }
        keep(i + 1, next);
        now_j = next_j;
        now_h = next_h;
        __syncthreads();
    }
    if (working && (any_not_finite<DT>(ka) || any_not_finite<DT>(va))) {
        for (int n = 0; n < 32 && own + n < keys; ++n) {
            const int kn = own + n;
            const Two kv = load_two((const T*)p.k + (kt.first + kn) * p.ldk + hcol, p.d), vv = load_two((const T*)p.v + (kt.first + kn) * p.ldv + hcol, p.d);
            Two a{0.f, 0.f}, b{0.f, 0.f};
            for (int r = r_first + first_row; r < r_end; r += (r - r_first) % (32 * RB) == 32 * RB - 1 ? BM - 32 * RB + 1 : 1) {
                const int ji = r / s.group, hi = kvh * s.group + r - ji * s.group, pos = ji + shift;
                if (!(kn <= pos && (pos - kn < s.window || kn < s.sinks))) continue;
                const int64_t ti = q.q0 + ji, ci = (int64_t)hi * p.d, at = ti * heads + hi;
                const Two x = load_two((const T*)p.q + ti * p.ldq + ci, p.d), g = load_two((const T*)p.yb + ti * p.ldyb + ci, p.d);
                const float w = exp2f((dot(x, kv) * p.s - p.lse[at]) * kLog2e), ds = w * (dot(g, vv) - p.delta[at]);
                a.a = fmaf(ds, x.a, a.a);
                a.b = fmaf(ds, x.b, a.b);
                b.a = fmaf(w, g.a, b.a);
                b.b = fmaf(w, g.b, b.b);
            }
            // to where the sums of products have them
#pragma unroll
            for (int m = 0; m < DT; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int from = (32 * m + 8 * (e >> 2) + 4 * h + (e & 3)) & 63;
                    const float x = __shfl(m < 2 ? a.a : a.b, from, 64), y = __shfl(m < 2 ? b.a : b.b, from, 64);
                    if ((lane & 31) == n) {
                        ka[m][e] = kNarrow<T> ? x * power(lift + kWeightLift<T>) : x;
                        va[m][e] = kNarrow<T> ? y * power(kWeightLift<T>) : y;
                    }
                }
        }
    }
    if constexpr (RG > 1) {     // the sums of the waves with the same keys, one after the other
        static_assert(KG * DT * 4096 <= 2 * BUF, "the sums fit the tiles' memory");
        float* sums = reinterpret_cast<float*>(lds) + group * DT * 1024 + lane;
        auto join = [&](floatx16 (&v)[DT]) INLINE {
            for (int n = 1; n < RG; ++n) {
                __syncthreads();
                if (first_row == 32 * RB * n) {
#pragma unroll
                    for (int m = 0; m < DT; ++m)
#pragma unroll
                        for (int e = 0; e < 16; ++e) sums[(m * 16 + e) * 64] = v[m][e];
                }
                __syncthreads();
                if (first_row == 0) {
#pragma unroll
                    for (int m = 0; m < DT; ++m)
#pragma unroll
                        for (int e = 0; e < 16; ++e) v[m][e] += sums[(m * 16 + e) * 64];
                }
            }
        };
        join(ka);
        join(va);
        if (first_row != 0) return;
    }
    if (!here) return;
    // (of f16: what the factors were multiplied by)
    float ka_by = kNarrow<T> ? power(-lift - kWeightLift<T>) : 1.f, va_by = kNarrow<T> ? power(-kWeightLift<T>) : 1.f;
    // partial sums of the sinks: (sequence, head), part, sink, kb and vb, the head's values
    const int64_t far_at = ((int64_t)(j - 1) * p.heads + kvh) * p.far_parts * s.sinks * 2 * p.d, far_next = (int64_t)s.sinks * 2 * p.d;
    if constexpr (FAR) {
        if (key >= s.sinks) return;
        float* out = p.far + far_at + tile * far_next + (int64_t)key * 2 * p.d;
        store_part<kNarrow<T>>(out, p.d, ka, ka_by);
        store_part<kNarrow<T>>(out + p.d, p.d, va, va_by);
        return;
    }
    if (split >= 0) {
        float* out = p.part + ((int64_t)(blockIdx.x - p.whole) * kKeys + key - key0) * 2 * p.d;
        store_part<kNarrow<T>>(out, p.d, ka, ka_by);
        store_part<kNarrow<T>>(out + p.d, p.d, va, va_by);
        return;
    }
    if (p.far && q.real && key0 == 0 && key < s.sinks && kt.far_rows > 0) {
        const float* in = p.far + far_at + (int64_t)key * 2 * p.d;   // (far_kernel has added the parts to the first)
#pragma unroll
        for (int m = 0; m < DT; ++m)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int at = 32 * m + 8 * g + 4 * h;
                float a[4], b[4];
                load_row(a, in + at, p.d - at);
                load_row(b, in + p.d + at, p.d - at);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    ka[m][4 * g + e] = kNarrow<T> ? fmaf(ka[m][4 * g + e], ka_by, a[e]) : ka[m][4 * g + e] + a[e];
                    va[m][4 * g + e] = kNarrow<T> ? fmaf(va[m][4 * g + e], va_by, b[e]) : va[m][4 * g + e] + b[e];
                }
            }
        ka_by = va_by = 1.f;
    }
    T* kb = p.kb ? (T*)p.kb + kcol * p.ldkb + hcol : nullptr;
    T* vb = p.vb ? (T*)p.vb + kcol * p.ldvb + hcol : nullptr;
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * m + 8 * g + 4 * h;
            const floatx16 &x = ka[m], &y = va[m];
            const int i = 4 * g;
            if constexpr (kNarrow<T>) {
                if (kb) store4(kb + at, x[i] * ka_by * p.s, x[i + 1] * ka_by * p.s, x[i + 2] * ka_by * p.s, x[i + 3] * ka_by * p.s, p.d - at, p.add);
                if (vb) store4(vb + at, y[i] * va_by, y[i + 1] * va_by, y[i + 2] * va_by, y[i + 3] * va_by, p.d - at, p.add);
            } else {
                if (kb) store4(kb + at, x[i] * p.s, x[i + 1] * p.s, x[i + 2] * p.s, x[i + 3] * p.s, p.d - at, p.add);
                if (vb) store4(vb + at, y[i], y[i + 1], y[i + 2], y[i + 3], p.d - at, p.add);
            }
        }
}

// The far parts' sums of a sequence's sinks added to the first, in order: a block has a strip of (kb, vb) of a (sequence, head)
__global__ __launch_bounds__(256) void far_kernel(Back p, int BM) {
    const int strips = (p.seqs.sinks * 2 * p.d + 255) / 256, at = (blockIdx.x % strips) * 256 + threadIdx.x;
    const int64_t pair = blockIdx.x / strips, next = (int64_t)p.seqs.sinks * 2 * p.d;
    const KeyTile kt = key_tile(p.seqs, (int)(pair / p.heads) + 1, 0);
    const int key = at / (2 * p.d), step = part_rows(kt.far_rows, p.far_parts, BM), parts = min(p.far_parts, (kt.far_rows + step - 1) / step);
    if (key >= p.seqs.sinks || key >= kt.keys || !kt.q.real) return;
    float* out = p.far + pair * p.far_parts * next + at;
    float sum = 0.f;
#pragma unroll 8
    for (int f = 0; f < parts; ++f) sum += out[f * next];
    if (parts > 1) *out = sum;
}

// The split tiles' sums added in order, and the sinks': a block has four of a tile's keys
template <class T>
__global__ __launch_bounds__(256) void join_kernel(Back p, int BM) {
    const Seqs& s = p.seqs;
    int64_t slot, tile;
    int kvh;
    const int64_t nth = blockIdx.x >> 5;
    place_of(p.whole + nth, p.slots, p.heads, slot, kvh);
    const int j = find_range(s.kstart, s.tk, 1, kKeys, s.n + 1, slot, tile);
    const KeyTile kt = key_tile(s, j, tile);
    const int rows = kt.r_end - kt.r_first, step = part_rows(rows, p.splits, BM);
    const int64_t next = (int64_t)kKeys * 2 * p.d;
    const int vecs = (2 * p.d + 3) / 4;
    for (int i = threadIdx.x; i < 4 * vecs; i += 256) {
        const int in_tile = (blockIdx.x & 31) * 4 + i / vecs, at = (i % vecs) * 4, key = kt.key0 + in_tile;
        if (key >= kt.keys) continue;
        float sum[4] = {0.f, 0.f, 0.f, 0.f}, v[4];
        const float* in = p.part + nth * p.splits * next + (int64_t)in_tile * 2 * p.d + at;
        const int parts = min(p.splits, (rows + step - 1) / step);
#pragma unroll 8
        for (int n = 0; n < parts; ++n) {
            load_row(v, in + n * next, 2 * p.d - at);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[e];
        }
        if (p.far && kt.q.real && kt.key0 == 0 && key < s.sinks && kt.far_rows > 0) {
            load_row(v, p.far + (((int64_t)(j - 1) * p.heads + kvh) * p.far_parts * s.sinks + key) * 2 * p.d + at, 2 * p.d - at);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int x = at + e;
            if (x >= 2 * p.d) break;
            T* out = (T*)(x < p.d ? p.kb : p.vb);
            if (!out) continue;
            out += (kt.first + key) * (x < p.d ? p.ldkb : p.ldvb) + (int64_t)kvh * p.d + (x < p.d ? x : x - p.d);
            const float w = x < p.d ? sum[e] * p.s : sum[e];
            *out = (T)(p.add ? (float)*out + w : w);
        }
    }
}

int cu_count() {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
    return cus > 0 ? cus : 256;
}

// blocks of far rows for each key head of a sequence: about one a CU in all
constexpr int64_t kFarBlocks = 256;

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_attention_b(int64_t tx, const void* yb, int64_t ldyb, const void* y, int64_t ldy, const float* lse, const void* q, int64_t ldq,
                              void* qb, int64_t ldqb, const void* k, int64_t ldk, void* kb, int64_t ldkb, const void* v, int64_t ldv, void* vb,
                              int64_t ldvb, const int64_t* qstart, const int64_t* kstart, double s, int64_t i_d, int64_t i_q, int64_t i_k,
                              int64_t i_t, int64_t i_tk, int64_t i_n, int64_t window, int64_t sinks, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_attention_b";
    Seqs seqs;
    if (int32_t rc = check_attention(fn, tx, s, i_d, i_q, i_k, i_t, i_tk, i_n, window, sinks, qstart, kstart, seqs)) return rc;
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_d * i_q)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d * i_q)) return rc;
    if (int32_t rc = check_ld(fn, "ldq", ldq, i_d * i_q)) return rc;
    if (int32_t rc = check_ld(fn, "ldk", ldk, i_d * i_k)) return rc;
    if (int32_t rc = check_ld(fn, "ldv", ldv, i_d * i_k)) return rc;
    if (qb)
        if (int32_t rc = check_ld(fn, "ldqb", ldqb, i_d * i_q)) return rc;
    if (kb)
        if (int32_t rc = check_ld(fn, "ldkb", ldkb, i_d * i_k)) return rc;
    if (vb)
        if (int32_t rc = check_ld(fn, "ldvb", ldvb, i_d * i_k)) return rc;
    const int64_t row_slots = slots_of(i_t, seqs.group, kRows, i_n + 1), slots = slots_of(i_tk, 1, kKeys, i_n + 1), units = slots * i_k;
    if (int32_t rc = check_extent(fn, "blocks of 128 rows of a key head", row_slots * i_k, kMostBlocks)) return rc;
    if (int32_t rc = check_extent(fn, "blocks of 128 keys of a key head", units, kMostBlocks)) return rc;
    const bool far = sinks > 0 && window >= 0 && window < i_tk && (kb || vb);
    const int64_t pairs = i_n * i_k, far_blocks = pairs * ((sinks * 2 * i_d + 255) / 256);
    if (far)
        if (int32_t rc = check_extent(fn, "i_n * i_k with sinks", far_blocks, kMostBlocks)) return rc;
    if (i_q == 0 && i_k > 0) return bad(fn, "i_q is zero");
    if (i_d == 0 || i_k == 0 || (i_t == 0 && (add || i_tk == 0)) || (!qb && !kb && !vb)) return STADE_HIP_OK;
    if ((i_t > 0 && (!yb || !y || !lse || !q)) || (i_tk > 0 && (!k || !v))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    Back p{yb, ldyb, y, ldy, lse, q, ldq, qb, ldqb, k, ldk, kb, ldkb, v, ldv, vb, ldvb, nullptr, seqs, (int)i_d, (int)i_k, (float)s, add != 0, factor(s)};
    p.seqs.flag = error_flag(call.ws);
    p.magic = (uint32_t)((((uint64_t)1 << 31) + seqs.group - 1) / seqs.group);
    const size_t deltas = ((size_t)i_t * i_q * 4 + 256) / 256 * 256;
    const int64_t sink_bytes = (int64_t)std::max<int64_t>(sinks, 1) * 2 * i_d * 4;
    // (what any call of up to kFarBlocks pairs takes is taken by each, so that every smaller one is captured after an eager one)
    const size_t fars = std::max((size_t)kFarBlocks * kMostSinks * 2 * kMostHead * 4, far ? (size_t)(pairs * sink_bytes) : 0);
    // Tiles of keys that fill no whole round of the CUs go over as many blocks as make two rounds (a block has a CU to itself), or
    // as have six tiles of rows each (fp32, whose products take eight times as long: four of half the size.  3 sequences of 500, 2
    // key heads: 111 us by three blocks a tile, 50 by ten).
    const int64_t cus = cu_count();
    p.whole = units / cus * cus;
    const int64_t rest = units - p.whole, longest = std::min<int64_t>(i_t, (int64_t)seqs.window + kKeys) * seqs.group;
    p.splits = rest ? (int)std::min<int64_t>(2 * cus / rest, std::max<int64_t>(1, longest / (tx == STADE_HIP_F32 ? 4 * 32 : 6 * 64))) : 1;
    if (p.splits <= 1) p.whole = units;
    const size_t parts = (size_t)(2 * cus) * kKeys * 2 * kMostHead * 4;
    const size_t mosts = ((size_t)row_slots * i_k * (kRows / 32) * 4 + 256) / 256 * 256;
    char* work = (char*)scratch(deltas + mosts + fars + parts);
    if (!work) return scratch_error();
    p.delta = (float*)work;
    work += deltas;
    p.most = (float*)work;
    work += mosts;
    if (far) {
        p.far = (float*)work;
        p.far_parts = (int)std::max<int64_t>(1, kFarBlocks / std::max<int64_t>(pairs, 1));
    }
    p.part = (float*)(work + fars);
    return with_type(tx, [&](auto t) -> int32_t {
        return with_width(i_d, [&](auto dt) -> int32_t {
            using T = decltype(t);
            constexpr int DT = decltype(dt)::value;
            const int64_t size = sizeof(T);
            const bool direct = straight(q, ldq, i_d, size) && straight(k, ldk, i_d, size) && straight(v, ldv, i_d, size) &&
                                straight(yb, ldyb, i_d, size) && straight(y, ldy, i_d, size);
            if (i_t > 0) {
                Back r = p;
                r.slots = row_slots;
                STADE_TIMED("attention_b_rows", stream, {
                    if (direct) rows_kernel<T, DT, true><<<(unsigned)(r.slots * i_k), 256, 0, stream>>>(r);
                    else rows_kernel<T, DT, false><<<(unsigned)(r.slots * i_k), 256, 0, stream>>>(r);
                });
                STADE_LAUNCHED("attention rows_kernel");
            }
            if ((kb || vb) && i_tk > 0) {
                constexpr unsigned NT = 64 * kGroups<T, false> * kRowWaves<T, false>, NTF = 64 * kGroups<T, true> * kRowWaves<T, true>;
                if (far) {
                    STADE_TIMED("attention_b_sinks", stream, {
                        if (direct) keys_kernel<T, DT, true, true><<<dim3((unsigned)(pairs * p.far_parts), sinks > 32 ? 2 : 1), NTF, 0, stream>>>(p);
                        else keys_kernel<T, DT, false, true><<<dim3((unsigned)(pairs * p.far_parts), sinks > 32 ? 2 : 1), NTF, 0, stream>>>(p);
                    });
                    STADE_LAUNCHED("attention keys_kernel (sinks)");
                    STADE_TIMED("attention_b_sinks", stream, far_kernel<<<(unsigned)far_blocks, 256, 0, stream>>>(p, (kTileRows<T, true>)));
                    STADE_LAUNCHED("attention far_kernel");
                }
                p.slots = slots;
                const unsigned grid = (unsigned)(p.whole + (units - p.whole) * p.splits);
                STADE_TIMED("attention_b_keys", stream, {
                    if (direct) keys_kernel<T, DT, true, false><<<grid, NT, 0, stream>>>(p);
                    else keys_kernel<T, DT, false, false><<<grid, NT, 0, stream>>>(p);
                });
                STADE_LAUNCHED("attention keys_kernel");
                if (p.whole < units) {
                    STADE_TIMED("attention_b_join", stream, join_kernel<T><<<(unsigned)(32 * (units - p.whole)), 256, 0, stream>>>(p, (kTileRows<T, false>)));
                    STADE_LAUNCHED("attention join_kernel");
                }
            }
            return STADE_HIP_OK;
        });
    });
}

}  // extern "C"
