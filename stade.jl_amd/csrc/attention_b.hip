// The adjoint of attention.  With P = exp(s q . k - lse) over the seen keys, the rows as in the forward sweep (query after query
// with the heads of a group side by side), and delta = yb . y for each row:
//   vb (+)= P^T yb,   S = P (yb v^T - delta),   qb (+)= s S k,   kb (+)= s S^T q
// P is formed again from lse; nothing of the size of the scores is kept.  Two launches (three with sinks):
//   rows_kernel   a block has 128 rows and goes over their keys: delta, and qb.  Scores as keys x rows, so that lse and
//                 delta are one value a lane, and S, rounded, is the operand of K^T S as it lies.
//   keys_kernel   a block has 128 keys and goes over the rows that see them, all heads of the group: kb and vb.  Scores as
//                 rows x keys; P and S are the operands of yb^T P and q^T S as they lie.
// That forms the scores and yb v^T twice, 7 products for 5, and needs no atomics: each result has one writer, its
// sums go in a fixed order, and the same call gives the same bits.
// Sinks are seen by every later row: rows past the window of the first tile of keys go over blocks of their own, which leave
// partial sums that the tile's block adds.
// Sums are fp32; P and S are rounded to the type as factors of products (to nearest), as the values they meet are.
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
    int64_t slots;
    uint32_t magic;        // ceil(2^32 / group)
    float* far;            // partial sums of the sinks; null: none
    int far_parts;
};

constexpr int kRows = 128, kKeys = 128;

template <class T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float e, int left, bool add) {
    float v[4] = {a, b, c, e};
    if (add) {
        float o[4];
        load_row(o, p, left);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += o[i];
    }
    store_row(p, v, left);
}

// blocks of one key head go to one XCD, or a key head's blocks go round the XCDs that have it
__device__ __forceinline__ void place_of(int64_t block, int64_t slots, int heads, int64_t& slot, int& kvh) {
    if (heads % 8 == 0) {
        const int64_t in = block >> 3;
        kvh = (int)(block & 7) + 8 * (int)(in / slots);
        slot = in % slots;
    } else if (8 % heads == 0) {
        kvh = (int)(block % heads);
        slot = block / heads;
    } else {
        kvh = (int)(block / slots);
        slot = block % slots;
    }
}

// ------------------------------------------------------------------------------------------
// qb, and delta
// ------------------------------------------------------------------------------------------
template <class T, int DT, bool DIRECT>
__global__ __launch_bounds__(256, sizeof(T) == 2 ? 2 : 1) void rows_kernel(Back p) {
    constexpr int DP = DT > 2 ? 128 : 64, BN = sizeof(T) == 2 ? 64 : 32, NB = BN / 32, TILE = BN * kRow<T, DP>, FR = DT * 32 / (2 * kCE<T>);
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
        if (here && h == 0) p.delta[t * (p.heads * s.group) + head] = delta;
    }
    if (!p.qb) return;
    row_fragments<T, DT, DIRECT>(qf, (const T*)p.q + t * p.ldq + col, here, p.d);
    const int p0 = r0 / s.group + q.shift(), p1 = min(r0 + kRows - 1, rows - 1) / s.group + q.shift();
    const int w0 = uniform((r0 + 32 * wave) / s.group + q.shift()), w1 = uniform(min(r0 + 32 * wave + 31, rows - 1) / s.group + q.shift());
    Range range = seen_by(s, p0, p1), mine = seen_by(s, w0, w1);
    if (!q.real) range = mine = Range{0, 0, 0};
    const KeyTiles<BN> keys(range);
    const T* k = (const T*)p.k + q.k0 * p.ldk + (int64_t)kvh * p.d;
    const T* v = (const T*)p.v + q.k0 * p.ldv + (int64_t)kvh * p.d;
    const float c = p.s * kLog2e, base = -lse * kLog2e;
    floatx16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][e] = 0.f;
    typename S::Held hk, hv;
    auto load = [&](int i, char* at) {
        const int key = keys.key(i);
        int from, to;
        tile_rows<BN>(range, key, from, to);
        S::load(hk, k + key * p.ldk, p.ldk, p.d, from, to, at, threadIdx.x);
        S::load(hv, v + key * p.ldv, p.ldv, p.d, from, to, at + TILE, threadIdx.x);
    };
    if (keys.count > 0) {
        load(0, lds);
        S::store(hk, lds, threadIdx.x);
        S::store(hv, lds + TILE, threadIdx.x);
        if constexpr (DIRECT) wait_loads<0>();
    }
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
                floatx16 x, g;
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = g[e] = 0.f;
#pragma unroll
                for (int f = 0; f < FR; ++f) x = multiply<T>(along_head<T, DP>(now, 32 * b, f), qf[f], x);
#pragma unroll
                for (int f = 0; f < FR; ++f) g = multiply<T>(along_head<T, DP>(now + TILE, 32 * b, f), of[f], g);
#pragma unroll
                for (int e = 0; e < 16; ++e) x[e] = __builtin_amdgcn_exp2f(fmaf(x[e], c, base)) * (g[e] - delta);
                if (!whole) {
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        const int at = 32 * b + 8 * (e >> 2) + (e & 3);
                        if (!(at <= high && (at > low || at < sink))) x[e] = 0.f;
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
        if (i + 1 < keys.count) {
            S::store(hk, next, threadIdx.x);
            S::store(hv, next + TILE, threadIdx.x);
            if constexpr (DIRECT) wait_loads<0>();
        }
        __syncthreads();
    }
    if (any_not_finite<DT>(acc)) {
        for (int i = 0; i < 32; ++i) {
            const int ri = r0 + 32 * wave + i, ji = ri / s.group, hi = kvh * s.group + ri - ji * s.group;
            if (ji >= q.nq) break;
            const Range seen = seen_by(s, ji + q.shift(), ji + q.shift());
            const int64_t ti = q.q0 + ji, ci = (int64_t)hi * p.d, at = ti * (p.heads * s.group) + hi;
            const Two x = load_two((const T*)p.q + ti * p.ldq + ci, p.d), g = load_two((const T*)p.yb + ti * p.ldyb + ci, p.d);
            const float li = p.lse[at], di = dot(g, load_two((const T*)p.y + ti * p.ldy + ci, p.d));
            float a = 0.f, b = 0.f;
            for (int part = 0; part < 2; ++part) {
                const int end = part ? seen.high : seen.sinks;
                for (int n = part ? seen.low : 0; n < end; ++n) {
                    const Two kn = load_two(k + n * p.ldk, p.d), vn = load_two(v + n * p.ldv, p.d);
                    const float w = exp2f((dot(x, kn) * p.s - li) * kLog2e) * (dot(g, vn) - di);
                    a = fmaf(w, kn.a, a);
                    b = fmaf(w, kn.b, b);
                }
            }
            store_two((T*)p.qb + ti * p.ldqb + ci, a * p.s, b * p.s, p.d, p.add);
        }
        return;
    }
    if (!here) return;
    T* out = (T*)p.qb + t * p.ldqb + col;
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * m + 8 * g + 4 * h;
            store4(out + at, acc[m][4 * g] * p.s, acc[m][4 * g + 1] * p.s, acc[m][4 * g + 2] * p.s, acc[m][4 * g + 3] * p.s, p.d - at, p.add);
        }
}

// ------------------------------------------------------------------------------------------
// kb and vb
// ------------------------------------------------------------------------------------------
// The block's waves: four of 32 keys each; for 16-bit types twice, for the two halves of a tile's rows (two waves a SIMD:
// one's exponentials beside the other's products), whose sums are joined at the end.
template <class T> constexpr int kHalves = sizeof(T) == 2 ? 2 : 1;

// rows r0 .. of a sequence in LDS: a row's q, yb, lse and delta.  A row's column and head by a product with the
// group's reciprocal (exact for less than 2^32 / group).
template <class T, int DP, int ROWS, int NT, bool DIRECT>
struct RowStage {
    static constexpr int CPR = kRow<T, DP> / 16, PER = ROWS * CPR / NT;
    struct Held { v4u v[DIRECT ? 1 : PER]; };

    static __device__ __forceinline__ void load(Held& held, const T* p, int64_t ld, int d, int group, uint32_t magic, int rem, int rows, const char* lds) {
        // (p: the head 0 of the group of row r0's query; rem: r0's head)
        const uint64_t base = (uint64_t)p;
        const v4u r = {(uint32_t)uniform((int)(uint32_t)base), (uint32_t)uniform((int)((uint32_t)(base >> 32) & 0xffffu)), 0x7fffffffu, 0x00020000u};
        const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds + uniform((int)(threadIdx.x >> 6)) * 1024;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int place = i * NT + threadIdx.x, o = place / CPR, c = (place % CPR) ^ turn<T, DP>(o);
            const uint32_t x = rem + o, jq = group == 1 ? x : __umulhi(x, magic), hd = x - jq * group;
            if constexpr (DIRECT)
                load_to_lds(r, o < rows && c * kCE<T> < d ? (jq * (uint32_t)ld + hd * d + c * kCE<T>) * (uint32_t)sizeof(T) : 0x80000000u, at + i * NT * 16);
            else
                held.v[i] = load_chunk(p + (int64_t)jq * ld + hd * d + c * kCE<T>, o < rows ? d - c * kCE<T> : 0);
        }
    }
    static __device__ __forceinline__ void store(const Held& held, char* lds) {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) *reinterpret_cast<v4u*>(lds + (i * NT + threadIdx.x) * 16) = held.v[i];
        }
    }
};

// FAR: rows past the first tile's window, which see its sinks only; block (part, sequence, head)
template <class T, int DT, bool DIRECT, bool FAR>
__global__ __launch_bounds__(256 * kHalves<T>, kHalves<T>) void keys_kernel(Back p) {
    constexpr int DP = DT > 2 ? 128 : 64, HALVES = kHalves<T>, NT = 256 * HALVES, BM = 32 * HALVES, TILE = BM * kRow<T, DP>;
    constexpr int FR = DT * 32 / (2 * kCE<T>), STATS = 2 * BM * 4, BUF = 2 * TILE;
    using S = RowStage<T, DP, BM, NT, DIRECT>;
    __shared__ __attribute__((aligned(1024))) char lds[2 * BUF + 2 * STATS];
    const Seqs& s = p.seqs;
    int64_t slot, tile;
    int kvh, j;
    if constexpr (FAR) {
        const int64_t b = blockIdx.x / p.far_parts;
        tile = blockIdx.x % p.far_parts;
        kvh = (int)(b % p.heads);
        j = (int)(b / p.heads) + 1;
    } else {
        place_of(blockIdx.x, p.slots, p.heads, slot, kvh);
        j = find_range(s.kstart, s.tk, 1, kKeys, s.n + 1, slot, tile);
    }
    const int wave = uniform((int)(threadIdx.x >> 6)), lane = threadIdx.x & 63, h = lane >> 5, part = wave & 3, half = wave >> 2;
    const int64_t k_first = j == 0 ? 0 : clamped(s.kstart[j - 1], s.tk);
    const int keys = (int)max((j > s.n ? s.tk : clamped(s.kstart[j], s.tk)) - k_first, (int64_t)0);
    const int key0 = FAR ? 0 : (int)min(tile * kKeys, (int64_t)keys);
    if (key0 >= keys) return;
    const Seq q = sequence(s, j - 1);
    // the rows that see the tile's keys, without what the far blocks do
    const int shift = q.shift();
    const int64_t last = (int64_t)key0 + kKeys - 1 + s.window - 1;    // the last position whose window has a key of the tile
    const int j0 = max(key0 - shift, 0), j1 = q.real ? (int)min((int64_t)q.nq, max(last + 1 - shift, (int64_t)0)) : 0;
    int r_first = j0 * s.group, r_end = j1 * s.group;
    const int far_rows = max(q.nq - max(j1, 0), 0) * s.group;         // (of the first tile)
    const int far_step = p.far_parts ? (far_rows / p.far_parts / BM + 1) * BM : 0;
    if constexpr (FAR) {
        r_first = r_end + (int)tile * far_step;
        r_end = min(r_first + far_step, q.nq * s.group);
        if (!q.real || r_first >= r_end) return;
    }
    const int own = key0 + 32 * part;      // this wave's keys
    const int64_t kcol = k_first + own + (lane & 31), hcol = (int64_t)kvh * p.d;
    const bool here = own + (lane & 31) < keys, working = own < keys && (!FAR || own < s.sinks);
    v4u kf[FR], vf[FR];
    row_fragments<T, DT, DIRECT>(kf, (const T*)p.k + kcol * p.ldk + hcol, here, p.d);
    row_fragments<T, DT, DIRECT>(vf, (const T*)p.v + kcol * p.ldv + hcol, here, p.d);
    floatx16 ka[DT], va[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int e = 0; e < 16; ++e) ka[i][e] = va[i][e] = 0.f;
    const float c = p.s * kLog2e;
    const int heads = p.heads * s.group, tiles = r_end > r_first ? (r_end - r_first + BM - 1) / BM : 0;
    typename S::Held hq, ho;
    float stat = 0.f;
    auto load = [&](int i, char* at) {
        const int r0 = r_first + i * BM, jq = r0 / s.group, rem = r0 - jq * s.group, rows = min(BM, r_end - r0);
        const int64_t t = q.q0 + jq, head = (int64_t)kvh * s.group;
        S::load(hq, (const T*)p.q + t * p.ldq + head * p.d, p.ldq, p.d, s.group, p.magic, rem, rows, at);
        S::load(ho, (const T*)p.yb + t * p.ldyb + head * p.d, p.ldyb, p.d, s.group, p.magic, rem, rows, at + TILE);
        if (threadIdx.x < 2 * BM) {     // lse and delta, one a thread (rows that are not: no weight)
            const int o = threadIdx.x % BM;
            const uint32_t x = rem + o, jo = s.group == 1 ? x : __umulhi(x, p.magic);
            const int64_t at1 = (t + jo) * heads + head + (x - jo * s.group);
            const bool first = threadIdx.x < BM;
            stat = first ? INFINITY : 0.f;
            if (o < rows) stat = first ? p.lse[at1] : p.delta[at1];
            if (first) stat *= -kLog2e;
        }
    };
    auto keep = [&](int i, char* at) {
        S::store(hq, at);
        S::store(ho, at + TILE);
        if (threadIdx.x < 2 * BM) reinterpret_cast<float*>(lds + 2 * BUF + (i & 1) * STATS)[threadIdx.x] = stat;
        if constexpr (DIRECT) wait_loads<0>();
    };
    if (tiles > 0) {
        load(0, lds);
        keep(0, lds);
    }
    __syncthreads();
    for (int i = 0; i < tiles; ++i) {
        const char* now = lds + (i & 1) * BUF;
        char* next = lds + (~i & 1) * BUF;
        if (i + 1 < tiles) load(i + 1, next);
        const int r0 = r_first + i * BM + 32 * half, end = min(r0 + 31, r_end - 1);
        const int pa = uniform(r0 / s.group + shift), pb = uniform(end / s.group + shift);
        const int own_to = own + 31;
        if (working && r0 < r_end && pb >= own && (pa - own_to < s.window || own < s.sinks)) {
            const float* stats = reinterpret_cast<const float*>(lds + 2 * BUF + (i & 1) * STATS) + 32 * half;
            floatx16 x, g;
#pragma unroll
            for (int e = 0; e < 16; ++e) x[e] = g[e] = 0.f;
#pragma unroll
            for (int f = 0; f < FR; ++f) x = multiply<T>(along_head<T, DP>(now, 32 * half, f), kf[f], x);
#pragma unroll
            for (int f = 0; f < FR; ++f) g = multiply<T>(along_head<T, DP>(now + TILE, 32 * half, f), vf[f], g);
            const bool whole = own_to <= pa && (pb - own < s.window || own_to < s.sinks);
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const v4f l = *reinterpret_cast<const v4f*>(stats + 8 * m + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * m + e] = __builtin_amdgcn_exp2f(fmaf(x[4 * m + e], c, l[e]));
            }
            if (!whole) {
                const int key = own + (lane & 31), rr = r0 + 4 * h;
                const int rem = rr % s.group, jq = rr / s.group;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const uint32_t xo = rem + 8 * (e >> 2) + (e & 3), jo = s.group == 1 ? xo : __umulhi(xo, p.magic);
                    const int pos = jq + (int)jo + shift;
                    if (!(key <= pos && (pos - key < s.window || key < s.sinks))) x[e] = g[e] = 0.f;
                }
            }
#pragma unroll
            for (int u = 0; u < kParts<T>; ++u) {
                const v4u w = part_of<T>(x, u);
#pragma unroll
                for (int m = 0; m < DT; ++m) va[m] = multiply<T>(along_rows<T, DP>(now + TILE, 32 * half + u * 2 * kCE<T>, 32 * m), w, va[m]);
            }
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const v4f dl = *reinterpret_cast<const v4f*>(stats + BM + 8 * m + 4 * h);
#pragma unroll
                for (int e = 0; e < 4; ++e) x[4 * m + e] *= g[4 * m + e] - dl[e];
            }
#pragma unroll
            for (int u = 0; u < kParts<T>; ++u) {
                const v4u w = part_of<T>(x, u);
#pragma unroll
                for (int m = 0; m < DT; ++m) ka[m] = multiply<T>(along_rows<T, DP>(now, 32 * half + u * 2 * kCE<T>, 32 * m), w, ka[m]);
            }
        }
        if (i + 1 < tiles) keep(i + 1, next);
        __syncthreads();
    }
    if (working && (any_not_finite<DT>(ka) || any_not_finite<DT>(va))) {
        for (int n = 0; n < 32 && own + n < keys; ++n) {
            const int key = own + n;
            const Two kn = load_two((const T*)p.k + (k_first + key) * p.ldk + hcol, p.d), vn = load_two((const T*)p.v + (k_first + key) * p.ldv + hcol, p.d);
            Two a{0.f, 0.f}, b{0.f, 0.f};
            for (int r = r_first + 32 * half; r < r_end; r += (r - r_first) % 32 == 31 ? BM - 31 : 1) {
                const int ji = r / s.group, hi = kvh * s.group + r - ji * s.group, pos = ji + shift;
                if (!(key <= pos && (pos - key < s.window || key < s.sinks))) continue;
                const int64_t ti = q.q0 + ji, ci = (int64_t)hi * p.d, at = ti * heads + hi;
                const Two x = load_two((const T*)p.q + ti * p.ldq + ci, p.d), g = load_two((const T*)p.yb + ti * p.ldyb + ci, p.d);
                const float w = exp2f((dot(x, kn) * p.s - p.lse[at]) * kLog2e), ds = w * (dot(g, vn) - p.delta[at]);
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
                        ka[m][e] = x;
                        va[m][e] = y;
                    }
                }
        }
    }
    if constexpr (HALVES > 1) {   // the second half's sums, one array after the other
        static_assert(4 * DT * 4096 <= 2 * BUF, "the sums fit the tiles' memory");
        float* sums = reinterpret_cast<float*>(lds) + part * DT * 1024 + lane;
        for (int a = 0; a < 2; ++a) {
            __syncthreads();
            if (half == 1) {
#pragma unroll
                for (int m = 0; m < DT; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e) sums[(m * 16 + e) * 64] = a ? va[m][e] : ka[m][e];
            }
            __syncthreads();
            if (half == 0) {
#pragma unroll
                for (int m = 0; m < DT; ++m)
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        if (a) va[m][e] += sums[(m * 16 + e) * 64];
                        else ka[m][e] += sums[(m * 16 + e) * 64];
                    }
            }
        }
        if (half == 1) return;
    }
    if (!here) return;
    const int key = own + (lane & 31);
    // partial sums of the sinks: (sequence, head), part, sink, kb and vb, the head's values
    const int64_t far_at = (((int64_t)(j - 1) * p.heads + kvh) * p.far_parts * s.sinks + key) * 2 * p.d, far_next = (int64_t)s.sinks * 2 * p.d;
    if constexpr (FAR) {
        if (key >= s.sinks) return;
        float* out = p.far + far_at + tile * far_next;
#pragma unroll
        for (int m = 0; m < DT; ++m)
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const int at = 32 * m + 8 * (e >> 2) + 4 * h + (e & 3);
                if (at < p.d) {
                    out[at] = ka[m][e];
                    out[p.d + at] = va[m][e];
                }
            }
        return;
    }
    if (p.far && q.real && key < s.sinks && key0 == 0) {
        for (int f = 0; f < p.far_parts && f * far_step < far_rows; ++f) {
            const float* in = p.far + far_at + f * far_next;
#pragma unroll
            for (int m = 0; m < DT; ++m)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int at = 32 * m + 8 * (e >> 2) + 4 * h + (e & 3);
                    if (at < p.d) {
                        ka[m][e] += in[at];
                        va[m][e] += in[p.d + at];
                    }
                }
        }
    }
    T* kb = p.kb ? (T*)p.kb + kcol * p.ldkb + hcol : nullptr;
    T* vb = p.vb ? (T*)p.vb + kcol * p.ldvb + hcol : nullptr;
#pragma unroll
    for (int m = 0; m < DT; ++m)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const int at = 32 * m + 8 * g + 4 * h;
            if (kb) store4(kb + at, ka[m][4 * g] * p.s, ka[m][4 * g + 1] * p.s, ka[m][4 * g + 2] * p.s, ka[m][4 * g + 3] * p.s, p.d - at, p.add);
            if (vb) store4(vb + at, va[m][4 * g], va[m][4 * g + 1], va[m][4 * g + 2], va[m][4 * g + 3], p.d - at, p.add);
        }
}

int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

template <class F>
int32_t with_width(int64_t d, F&& f) {
    if (d <= 64) return f(std::integral_constant<int, 2>{});
    if (d <= 96) return f(std::integral_constant<int, 3>{});
    return f(std::integral_constant<int, 4>{});
}

// blocks of far rows for each key head of a sequence: about two a CU in all
constexpr int64_t kFarBlocks = 512;

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
    if (i_d == 0 || i_q == 0 || (i_t == 0 && (add || i_tk == 0)) || (!qb && !kb && !vb)) return STADE_HIP_OK;
    if ((i_t > 0 && (!yb || !y || !lse || !q)) || (i_tk > 0 && (!k || !v))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    Back p{yb, ldyb, y, ldy, lse, q, ldq, qb, ldqb, k, ldk, kb, ldkb, v, ldv, vb, ldvb, nullptr, seqs, (int)i_d, (int)i_k, (float)s, add != 0};
    p.seqs.flag = error_flag(call.ws);
    p.magic = seqs.group > 1 ? (uint32_t)(((uint64_t)1 << 32) / seqs.group + 1) : 0;
    const bool far = sinks > 0 && window >= 0 && window < i_tk && (kb || vb);
    const size_t deltas = ((size_t)i_t * i_q * 4 + 256) / 256 * 256;
    const int64_t pairs = i_n * i_k, sink_bytes = (int64_t)std::max<int64_t>(sinks, 1) * 2 * i_d * 4;
    char* work = (char*)scratch(deltas + (far ? (size_t)(std::max(pairs, kFarBlocks) * sink_bytes) : 0));
    if (!work) return scratch_error();
    p.delta = (float*)work;
    if (far) {
        p.far = (float*)(work + deltas);
        p.far_parts = (int)std::max<int64_t>(1, kFarBlocks / std::max<int64_t>(pairs, 1));
    }
    return with_type(tx, [&](auto t) -> int32_t {
        return with_width(i_d, [&](auto dt) -> int32_t {
            using T = decltype(t);
            constexpr int DT = decltype(dt)::value;
            const int64_t size = sizeof(T);
            const bool direct = straight(q, ldq, i_d, size) && straight(k, ldk, i_d, size) && straight(v, ldv, i_d, size) &&
                                straight(yb, ldyb, i_d, size) && straight(y, ldy, i_d, size);
            if (i_t > 0) {
                Back r = p;
                r.slots = slots_of(i_t, seqs.group, kRows, i_n + 1);
                STADE_TIMED("attention_b_rows", stream, {
                    if (direct) rows_kernel<T, DT, true><<<(unsigned)(r.slots * i_k), 256, 0, stream>>>(r);
                    else rows_kernel<T, DT, false><<<(unsigned)(r.slots * i_k), 256, 0, stream>>>(r);
                });
                STADE_LAUNCHED("attention rows_kernel");
            }
            if ((kb || vb) && i_tk > 0) {
                constexpr unsigned NT = 256 * kHalves<T>;
                if (far) {
                    STADE_TIMED("attention_b_sinks", stream, {
                        if (direct) keys_kernel<T, DT, true, true><<<(unsigned)(pairs * p.far_parts), NT, 0, stream>>>(p);
                        else keys_kernel<T, DT, false, true><<<(unsigned)(pairs * p.far_parts), NT, 0, stream>>>(p);
                    });
                    STADE_LAUNCHED("attention keys_kernel (sinks)");
                }
                p.slots = slots_of(i_tk, 1, kKeys, i_n + 1);
                STADE_TIMED("attention_b_keys", stream, {
                    if (direct) keys_kernel<T, DT, true, false><<<(unsigned)(p.slots * i_k), NT, 0, stream>>>(p);
                    else keys_kernel<T, DT, false, false><<<(unsigned)(p.slots * i_k), NT, 0, stream>>>(p);
                });
                STADE_LAUNCHED("attention keys_kernel");
            }
            return STADE_HIP_OK;
        });
    });
}

}  // extern "C"
