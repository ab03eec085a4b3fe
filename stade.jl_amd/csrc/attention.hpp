// What attention and its adjoint share: the sequences' tiles, the operands' tiles in LDS and their
// fragments, and which keys a query sees.
//
// The rows that a tile works on are the (query, head) pairs that go with one key head, query after query with its `group` heads
// side by side: row r of a sequence is query r / group and head r % group.  One tile of keys and values then serves all heads of
// a group, a tile of rows spans few positions (a window's edges are cut finely), and single tokens
// still make rows of a tile.
#pragma once

#include "rows.hpp"

#include <type_traits>

namespace stade {
namespace attn {

using namespace rows;

// (a launch's threads are counted in 32 bits, and blocks have up to 512)
constexpr int64_t kMostBlocks = (1 << 23) - 1;
constexpr int64_t kMostHead = 128, kMostHeads = 4096, kMostSeqs = 1 << 20, kMostSinks = 64;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));

// of a lambda in a kernel: what it captures stays in registers only where it is inlined
#define INLINE __attribute__((always_inline))

// the same value in every lane, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}

// the other half wave's value
__device__ __forceinline__ float other_half(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float((threadIdx.x & 32) ? r[0] : r[1]);
}

// ------------------------------------------------------------------------------------------
// sequences
// ------------------------------------------------------------------------------------------
struct Seqs {
    const int64_t* qstart;
    const int64_t* kstart;
    int n;
    int64_t t, tk;
    int group;
    int window, sinks;   // window: at most 2^30, which is all
    int32_t* flag;
};

// Every offset of both kinds is looked at by some block; those out of order or range raise the flag.
__device__ __forceinline__ void check_offsets(const Seqs& s, int64_t block, int64_t blocks) {
    for (int64_t i = block * blockDim.x + threadIdx.x; i <= s.n; i += blocks * blockDim.x) {
        const int64_t q = s.qstart[i], k = s.kstart[i], q0 = i ? s.qstart[i - 1] : 0, k0 = i ? s.kstart[i - 1] : 0;
        if (q < q0 || q > s.t || k < k0 || k > s.tk) *s.flag = kErrIndex;
    }
}

__device__ __forceinline__ int64_t clamped(int64_t v, int64_t most) { return min(max(v, (int64_t)0), most); }

// One sequence, or columns of none (i < 0 or i >= n: those before the first and behind the last)
struct Seq {
    bool real;
    int64_t q0, k0;   // first query and key
    int nq, nk;
    __device__ __forceinline__ int shift() const { return nk - nq; }   // query j stands at key j + shift
};
__device__ __forceinline__ Seq sequence(const Seqs& s, int i) {
    Seq r;
    r.real = i >= 0 && i < s.n;
    r.q0 = i < 0 ? 0 : clamped(s.qstart[min(i, s.n)], s.t);
    const int64_t q1 = i >= s.n ? s.t : clamped(s.qstart[i + 1], s.t);
    r.nq = (int)max(q1 - r.q0, (int64_t)0);
    r.k0 = 0;
    r.nk = 0;
    if (r.real) {
        r.k0 = clamped(s.kstart[i], s.tk);
        r.nk = (int)max(clamped(s.kstart[i + 1], s.tk) - r.k0, (int64_t)0);
    }
    return r;
}

// Ranges of columns cut into tiles of `size` units, `per` units a column, without a count of the tiles before:
// range j (from 0, columns at[j - 1] .. at[j], with at[-1] = 0 and at[m] = t) has the slots from at[j - 1] * per / size + j on.
// That is room for its tiles, as one range's part of the quotient and one more are never fewer than the tiles it
// takes, and it grows with j, so a slot's range is found by a search, 64 offsets a step.
// m + 1 ranges; slots in all: slots_of().
__device__ __forceinline__ int64_t first_slot(const int64_t* at, int64_t t, int per, int size, int j) {
    return (j ? clamped(at[j - 1], t) * per / size : 0) + j;
}
inline int64_t slots_of(int64_t t, int per, int size, int64_t m) { return t * per / size + m + 1; }
__device__ __forceinline__ int find_range(const int64_t* at, int64_t t, int per, int size, int m, int64_t slot, int64_t& tile) {
    int lo = 0, hi = m + 1;
    while (hi - lo > 1) {
        const int step = (hi - lo + 63) / 64, c = lo + (int)(threadIdx.x & 63) * step;
        const uint64_t hit = __ballot(c < hi && first_slot(at, t, per, size, c) <= slot);
        const int top = hit ? 63 - __builtin_clzll(hit) : 0;
        lo += top * step;
        hi = min(hi, lo + step);
    }
    tile = slot - first_slot(at, t, per, size, lo);
    return lo;
}

// The keys that rows at positions p0 .. p1 of a sequence see: [0, sinks) and [low, high)
struct Range {
    int sinks, low, high;
};
__device__ __forceinline__ Range seen_by(const Seqs& s, int p0, int p1) {
    Range r;
    r.high = max(p1 + 1, 0);
    r.low = min(max(p0 - s.window + 1, 0), r.high);
    r.sinks = min(min(s.sinks, r.high), r.low);
    return r;
}

// The tiles of BN keys that hold a range: `sink` of them from 0 on, then those from `first` on
template <int BN>
struct KeyTiles {
    int sink, first, count;
    __device__ __forceinline__ explicit KeyTiles(const Range& r) {
        first = r.low / BN;
        const int end = r.high > r.low ? (r.high + BN - 1) / BN : first;
        sink = min((r.sinks + BN - 1) / BN, first);
        count = sink + end - first;
    }
    __device__ __forceinline__ int key(int i) const { return (i < sink ? i : first + i - sink) * BN; }
};

// the keys of [key, key + BN) that a range has: rows [from, to) of the tile (what lies between sinks and window comes along)
template <int BN>
__device__ __forceinline__ void tile_rows(const Range& r, int key, int& from, int& to) {
    from = key < r.sinks ? 0 : max(r.low - key, 0);
    to = r.high > key && key + BN > r.low ? min(r.high - key, BN) : r.sinks - key;
}

// ------------------------------------------------------------------------------------------
// operand tiles in LDS
// ------------------------------------------------------------------------------------------
// A tile holds rows of DP values (64 or 128: the head's values and zeros), in 16-byte chunks, 1024 bytes (what a wave loads
// straight to LDS at a time) one after the other, each kPad further.  Row r has its chunk c at place c ^ turn(r).  It is read in two
// ways: sixteen rows' chunk c (fragments along the head), and, by the transposing read for 16-bit types, four rows' 64
// bytes (fragments along the rows); turn and pad together let both meet all the banks.  For 16-bit types the turn
// moves whole 64 bytes (two rows a pass over the banks: and 32), so that few addresses serve all fragments, the rest being constants.
template <class T> constexpr int kCE = 16 / (int)sizeof(T);
template <class T, int DP> constexpr int kRow = DP * (int)sizeof(T);
template <class T> constexpr int kPad = sizeof(T) == 2 ? 16 : 0;
template <class T, int DP, int ROWS> constexpr int kTile = ROWS * kRow<T, DP> / 1024 * (1024 + kPad<T>);

template <class T, int DP>
__device__ __forceinline__ int turn(int r) {
    if constexpr (sizeof(T) == 4) return (r >> 2 & 1) << 3 | (r & 3) << 1 | (r >> 3 & 1);   // (its rows are read 128 bytes at a time, two rows four apart)
    else if constexpr (DP == 128) return (r & 3) << 2;
    else return (r >> 1 & 1) << 2 | (r >> 2 & 1) << 1;
}
// the start of a row
template <class T, int DP>
__device__ __forceinline__ int row_at(int r) {
    constexpr int PER = 1024 / kRow<T, DP>;
    return r / PER * (1024 + kPad<T>) + r % PER * kRow<T, DP>;
}
template <class T, int DP>
__device__ __forceinline__ int chunk_at(int r, int c) {
    return row_at<T, DP>(r) + ((c ^ turn<T, DP>(r)) << 4);
}

// 16 bytes a lane from the buffer `r` at `off` to LDS, the wave's lanes from `at` on.  In assembly because
// of the waits: for the builtin the compiler waits for all loads before the next LDS read of any kind, as it
// cannot tell the buffers apart.  It has no output register; wait_loads counts it.
__device__ __forceinline__ void load_to_lds(v4u r, uint32_t off, uint32_t at) {
    at = (uint32_t)uniform((int)at);
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(at) : "memory");
}
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}
// Before a loop that counts its own loads: what the compiler's loads brought into registers is there, in a form that the
// compiler sees.  Without it the compiler waits for them at their first use inside the loop, in every round, and with them
// for all that is under way to LDS.
__device__ __forceinline__ void settle_loads() { __builtin_amdgcn_s_waitcnt(0x0f70); }   // vmcnt(0)

// 16 bytes at any alignment: the first `left` values, and zeros
template <class T>
__device__ __forceinline__ v4u load_chunk(const T* p, int left) {
    typedef T vec __attribute__((ext_vector_type(kCE<T>)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    vec v = {};
    if (left >= kCE<T>) {
        v = *reinterpret_cast<const loose*>(p);
    } else if (left > 0) {
#pragma unroll
        for (int i = 0; i < kCE<T>; ++i) v[i] = i < left ? p[i] : (T)0.f;
    }
    return __builtin_bit_cast(v4u, v);
}

// where the chunk that is the place'th of a tile lies
template <class T>
__device__ __forceinline__ int place_at(int place) {
    return (place >> 6) * (1024 + kPad<T>) + (place & 63) * 16;
}

// Staging of a tile of ROWS rows by NT threads (`tid`: this thread's number among them): straight to LDS (DIRECT:
// 16-byte aligned rows and whole chunks), or through registers.  Rows outside [from, to) become zeros.
template <class T, int DP, int ROWS, int NT, bool DIRECT>
struct Stage {
    static constexpr int CPR = kRow<T, DP> / 16, PER = ROWS * CPR / NT;
    static_assert(ROWS * CPR % NT == 0, "whole chunks a thread");
    uint32_t off[DIRECT ? PER : 1];   // a thread's chunks from the first row's start (past any buffer: none)
    v4u held[DIRECT ? 1 : PER];
    int64_t ld;
    int d, tid;

    __device__ __forceinline__ Stage(int64_t ld_, int d_, int tid_) : ld(ld_), d(d_), tid(tid_) {
        if constexpr (DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int place = i * NT + tid, o = place / CPR, c = (place % CPR) ^ turn<T, DP>(o);
                off[i] = c * kCE<T> < d ? (uint32_t)o * ((uint32_t)ld * sizeof(T)) + c * 16 : 0x80000000u;
            }
        }
    }
    // (`p`: the tile's first row)
    __device__ __forceinline__ void load(const T* p, int from, int to, const char* lds) {
        if constexpr (DIRECT) {
            const uint64_t base = (uint64_t)(p + (int64_t)from * ld);
            const uint32_t row = (uint32_t)ld * sizeof(T), bytes = to > from ? (uint32_t)(to - from - 1) * row + (uint32_t)d * sizeof(T) : 0;
            const uint32_t less = (uint32_t)uniform((int)(from * row));   // (rows before `from` have offsets past the buffer too: they wrap)
            const v4u r = {(uint32_t)uniform((int)(uint32_t)base), (uint32_t)uniform((int)((uint32_t)(base >> 32) & 0xffffu)), (uint32_t)uniform((int)bytes),
                           0x00020000u};
            const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds + uniform(tid >> 6) * (1024 + kPad<T>);
#pragma unroll
            for (int i = 0; i < PER; ++i) load_to_lds(r, off[i] - less, at + i * (NT / 64) * (1024 + kPad<T>));
        } else {
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int place = i * NT + tid, o = place / CPR, c = (place % CPR) ^ turn<T, DP>(o);
                held[i] = load_chunk(p + (int64_t)o * ld + c * kCE<T>, o >= from && o < to ? d - c * kCE<T> : 0);
            }
        }
    }
    __device__ __forceinline__ void store(char* lds) const {
        if constexpr (!DIRECT) {
#pragma unroll
            for (int i = 0; i < PER; ++i) *reinterpret_cast<v4u*>(lds + place_at<T>(i * NT + tid)) = held[i];
        }
    }
};

// ------------------------------------------------------------------------------------------
// fragments and products: 32 x 32 tiles, v_mfma 32x32x16 (16-bit types) or 32x32x2 (fp32)
// ------------------------------------------------------------------------------------------
// A fragment is 16 bytes a lane.  Along the head: 32 rows' values of head chunk 2 s + h, h = lane / 32 (16 values
// of the head for 16-bit types, 8 for fp32).
template <class T, int DP>
__device__ __forceinline__ v4u along_head(const char* lds, int row0, int s) {
    const int lane = threadIdx.x & 63, h = lane >> 5, r = lane & 31, t = turn<T, DP>(r);
    // (row0 is a multiple of 32, which the turn does not see)
    if constexpr (sizeof(T) == 2 && DP == 128) {
        return *reinterpret_cast<const v4u*>(lds + (row_at<T, DP>(r) + h * 16 + ((4 * (s >> 1) ^ t) << 4)) + (row_at<T, DP>(row0) + 32 * (s & 1)));
    } else {
        return *reinterpret_cast<const v4u*>(lds + (row_at<T, DP>(r) + (((2 * s + h) ^ t) << 4)) + row_at<T, DP>(row0));
    }
}
// Along the rows: 32 values of the head from `col` on, for as many rows from row0 on as a fragment has (16, fp32: 8).
// The rows come in the order in which a 32 x 32 result holds its rows in registers (lane half h, register i: row
// 8 (i / 4) + 4 h + i % 4), so that a result, rounded, is the other operand as it lies.
template <class T, int DP>
__device__ __forceinline__ v4u along_rows(const char* lds, int row0, int col) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
        // (row0 is a multiple of 16, col of 32: of a chunk's number the turn moves the fours, and the two where it does, by lane)
        const int i = lane & 15, r = 4 * h + (i >> 2), c = 2 * ((lane >> 4) & 1) + ((i & 3) >> 1), t = turn<T, DP>(r);
        const char* at = lds + (row_at<T, DP>(r) + (((c ^ (t & 3)) + (col / 8 ^ (t & ~3))) << 4) + (i & 1) * 8) + row_at<T, DP>(row0);
        typedef __attribute__((address_space(3))) v4s* lp;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at));
        const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at + row_at<T, DP>(8)));
        return __builtin_bit_cast(v4u, (v8s){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    } else {
        const int x = col + (lane & 31);
        v4f v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(lds + chunk_at<T, DP>(row0 + 4 * h + j, x >> 2) + (x & 3) * 4);
        return __builtin_bit_cast(v4u, v);
    }
}
template <class T>
__device__ __forceinline__ floatx16 multiply(v4u a, v4u b, floatx16 c) {
    if constexpr (sizeof(T) == 4) {
        const v4f x = __builtin_bit_cast(v4f, a), y = __builtin_bit_cast(v4f, b);
#pragma unroll
        for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[j], y[j], c, 0, 0, 0);
        return c;
    } else if constexpr (Code<T>::value == STADE_HIP_BF16) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
}
// fragments that a 32-row result makes, as an operand along its rows
template <class T> constexpr int kParts = 32 / (2 * kCE<T>);
template <class T>
__device__ __forceinline__ v4u part_of(const floatx16& v, int u) {
    typedef T vec __attribute__((ext_vector_type(kCE<T>)));
    vec p;
#pragma unroll
    for (int i = 0; i < kCE<T>; ++i) p[i] = (T)v[u * kCE<T> + i];
    return __builtin_bit_cast(v4u, p);
}

// The order in which the compiler is to issue a stretch of code: so many instructions of a kind next.  (Left alone it reads a
// fragment just before its product and waits for LDS each time.)
constexpr int kValu = 2, kMfma = 8, kRead = 0x100, kTrans = 0x400;
#define ORDER(kind, n) __builtin_amdgcn_sched_group_barrier(kind, n, 0)

// N products one after the other, in the order written, each step fenced off: product(i, fragment i), the read of the
// fragment AHEAD products later (so that LDS is never waited for), and what else there is to do meanwhile, rest(i).
template <int N, int AHEAD, class L, class M, class F>
__device__ __forceinline__ void products(L&& fragment, M&& product, F&& rest) {
    decltype(fragment(std::integral_constant<int, 0>{})) r[AHEAD];
    static_for<AHEAD>([&](auto i) INLINE {
        if constexpr (decltype(i)::value < N) r[decltype(i)::value] = fragment(i);
    });
    __builtin_amdgcn_sched_barrier(0);
    static_for<N>([&](auto i) INLINE {
        constexpr int I = decltype(i)::value;
        product(i, r[I % AHEAD]);
        if constexpr (I + AHEAD < N) r[I % AHEAD] = fragment(std::integral_constant<int, I + AHEAD>{});
        rest(i);
        __builtin_amdgcn_sched_barrier(0);
    });
}

// ------------------------------------------------------------------------------------------
// values that are not finite
// ------------------------------------------------------------------------------------------
// A tile's product multiplies what a row does not see by zero, which infinities and NaN do not mind.  So a wave whose sums
// are not all finite forms them again one row (or key) after the other, from what is seen alone: a lane has two
// values of the head.  That is slow (some 500 cycles a pair) and costs nothing where all values are finite but the look at the sums.
template <int DT>
__device__ __forceinline__ bool any_not_finite(const floatx16 (&o)[DT]) {
    float z = 0.f;
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) z = fmaf(o[i][j], 0.f, z);
    return __any(z != 0.f);
}
struct Two {
    float a, b;
};
template <class T>
__device__ __forceinline__ Two load_two(const T* row, int d) {
    const int lane = threadIdx.x & 63;
    return Two{lane < d ? (float)row[lane] : 0.f, lane + 64 < d ? (float)row[lane + 64] : 0.f};
}
__device__ __forceinline__ float dot(Two x, Two y) { return wave_sum(fmaf(x.a, y.a, x.b * y.b)); }
template <class T>
__device__ __forceinline__ void store_two(T* row, float a, float b, int d, bool add) {
    const int lane = threadIdx.x & 63;
    if (lane < d) row[lane] = (T)(add ? (float)row[lane] + a : a);
    if (lane + 64 < d) row[lane + 64] = (T)(add ? (float)row[lane + 64] + b : b);
}

// a row's fragments along the head from memory: one row a lane (its half's chunks), zeros past d
template <class T, int DT, bool DIRECT>
__device__ __forceinline__ void row_fragments(v4u (&f)[DT * 32 / (2 * kCE<T>)], const T* row, bool here, int d) {
    const int h = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int s = 0; s < DT * 32 / (2 * kCE<T>); ++s) {
        const int c = (2 * s + h) * kCE<T>;
        if constexpr (DIRECT) {
            f[s] = (v4u){0, 0, 0, 0};
            if (here && c < d) f[s] = *reinterpret_cast<const v4u*>(row + c);
        } else {
            f[s] = load_chunk(row + c, here ? d - c : 0);
        }
    }
}

// a block's place: blocks go round the 8 XCDs, each with an L2 of its own; blocks of one key head
// go to one XCD, or a key head's blocks go round the XCDs that have it
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

// four consecutive values of the head
template <class T>
__device__ __forceinline__ void store4(T* p, float a, float b, float c, float e, int left, bool add = false) {
    float v[4] = {a, b, c, e};
    if (add) {
        float o[4];
        load_row(o, p, left);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] += o[i];
    }
    store_row(p, v, left);
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------
// rows that go straight to LDS: 16-byte aligned, whole chunks, and a tile's offsets within 31 bits
inline bool straight(const void* p, int64_t ld, int64_t d, int64_t size) {
    return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0 && d * size % 16 == 0 && ld * size < (int64_t)1 << 23;
}

inline int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

template <class F>
inline int32_t with_width(int64_t d, F&& f) {
    if (d <= 64) return f(std::integral_constant<int, 2>{});
    if (d <= 96) return f(std::integral_constant<int, 3>{});
    return f(std::integral_constant<int, 4>{});
}

// The scores' factor as the kernels divide by it and multiply -Inf with it: not below 2^-100 in size (in place of 0 it moves weights by less
// than a rounding while q . k is below 2^76)
inline float factor(double s) {
    const float f = (float)s;
    return fabsf(f) >= 0x1p-100f ? f : f < 0.f ? -0x1p-100f : 0x1p-100f;
}

// the checks of both functions; the sequences with everything but the flag
inline int32_t check_attention(const char* fn, int64_t tx, double s, int64_t i_d, int64_t i_q, int64_t i_k, int64_t i_t, int64_t i_tk, int64_t i_n,
                               int64_t window, int64_t sinks, const int64_t* qstart, const int64_t* kstart, Seqs& seqs) {
    if (int32_t rc = check_type(fn, "q", tx)) return rc;
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostHead)) return rc;
    if (int32_t rc = check_extent(fn, "i_q", i_q, kMostHeads)) return rc;
    if (int32_t rc = check_extent(fn, "i_k", i_k, kMostHeads)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (int32_t rc = check_extent(fn, "i_tk", i_tk, kMostRows)) return rc;
    if (int32_t rc = check_extent(fn, "i_n", i_n, kMostSeqs)) return rc;
    if (int32_t rc = check_extent(fn, "sinks", sinks, kMostSinks)) return rc;
    if (i_k == 0 ? i_q != 0 : i_q % i_k != 0) return bad(fn, "i_q is not a multiple of i_k");
    // (rows of a sequence are counted in 32 bits)
    const int64_t group = i_k ? i_q / i_k : 0;
    if (int32_t rc = check_extent(fn, "i_t * i_q / i_k", i_t * group, kMostRows)) return rc;
    if (!(fabsf((float)s) < INFINITY)) return bad(fn, "s is not finite in Float32");
    if (!qstart || !kstart) return bad(fn, "null pointer");
    const int most = 1 << 30;
    seqs = Seqs{qstart, kstart, (int)i_n, i_t, i_tk, (int)group, window < 0 || window > most ? most : (int)window, (int)sinks, nullptr};
    return 0;
}

}  // namespace attn
}  // namespace stade
