// Products of rows with the weights of the expert that each row was sent to, and their adjoint.
// The rows lie in expert order: expert e has the rows start[e] .. start[e+1] (any number, none too).
//
//   expert_mul     y[:, t]  (+)= w[:, :, e]  x[:, t]        (column-major: w is i_out x i_in x i_e)
//   expert_mul_b   xb[:, t] (+)= w[:, :, e]' yb[:, t],   wb[:, :, e] (+)= sum over e's rows of yb[:, t] x[:, t]'
//
// Row by row in memory: x[t][i], y[t][o], w[e][i][o]; so y = x w, xb = yb w^T, wb = x^T yb.
// Rows that no expert has get zeros (with `add`, nothing).
//
// Products run on the matrix cores (v_mfma 32x32x16 for bf16 and f16, 32x32x2 for fp32), summed in
// fp32 and rounded once.  The tape's values are exact in 16 bits, so wb from the tape needs no further rounding.
//
// Bound by the matrix cores for many rows, by reading w for few.  On an MI355X in bf16:
//   one round of 256 x 256 tiles (4096 x 4096): 41, 65, 116 and 218 us for k = 1024, 2048, 4096 and 8192 (1190 TFLOP/s at
//     4096): 1.6 us a step of 64 k and 14 us whatever k is (launch, prologue and epilogue).
//   16384 rows, 16 experts with as many each, 2048 x 4096: y 252 us (1090 TFLOP/s), xb 248 (1110), wb in fp32 326 (844; its
//     537 MB alone take 107 us), wb from the tape 347 (the bytes become 16-bit values between the products).  With uneven
//     shares (a standard deviation of 30 %) xb 289 us, wb from the tape 360.  Added to what is there: y 313 us, xb 278, wb in fp32
//     469, in bf16 410 (293 set): 16-bit results that add go out straight from the registers.
//   24 rows, 8 experts, 2048 x 4096: y 23.5 us, xb 21.8 (5.7 and 6.2 TB/s of w, which the last-level cache holds in part).
#include "tape8.hpp"

#include <algorithm>
#include <type_traits>

namespace stade {
namespace {

using namespace rows;

constexpr int kMostExperts = 4096;

// A piece of work on rows: `rows` of them from `row`, with expert `e`'s weights (-1: of no expert)
struct Rows {
    int e;
    int64_t row;
    int rows;
};

// the same value in every lane, in scalar registers
__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    return (int64_t)((uint64_t)(uint32_t)uniform((int)(v >> 32)) << 32 | (uint32_t)uniform((int)v));
}
__device__ __forceinline__ Rows uniform(const Rows& r) { return Rows{uniform(r.e), uniform(r.row), uniform(r.rows)}; }

// The experts' offsets 64 at a time, one a lane: lane l has boundary i = base + l, in order and in range
// (the largest of the offsets up to i, each between 0 and t: offsets that are neither raise the device
// error flag, and no row has two experts).  Segment i, the rows between boundaries i - 1 and i,
// belongs to expert i - 1.
struct Chunk {
    int64_t from, end;       // segment i
    int64_t before, mine;    // pieces of the segments before i (from segment 1 on), and of i
};
template <int BM>
__device__ __forceinline__ Chunk scan(const int64_t* start, int ne, int64_t t, int base, int64_t reach, int64_t pieces, int32_t* flag) {
    const int lane = threadIdx.x & 63, i = base + lane;
    const int64_t raw = i <= ne ? start[i] : 0;
    Chunk c;
    c.end = i <= ne ? min(max(raw, (int64_t)0), t) : 0;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(c.end, o, 64);
        if (lane >= o) c.end = max(c.end, up);
    }
    c.end = max(c.end, reach);
    if (i <= ne && c.end != raw && flag) *flag = kErrIndex;
    c.from = __shfl_up(c.end, 1, 64);
    if (lane == 0) c.from = reach;
    c.mine = i >= 1 && i <= ne ? (c.end - c.from + BM - 1) / BM : 0;
    int64_t sum = c.mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
    }
    c.before = pieces + sum - c.mine;
    return c;
}

// All pieces of at most BM rows: the experts', in order, then those of the rows before the first
// expert and after the last.  Every wave finds them by itself.
template <int BM>
struct Pieces {
    const int64_t* start;
    int ne;
    int64_t t;
    Chunk first;
    int64_t experts, head, reach;   // pieces of the experts; rows before the first; the last one's end

    __device__ __forceinline__ Pieces(const int64_t* start_, int ne_, int64_t t_, int32_t* flag) : start(start_), ne(ne_), t(t_) {
        first = scan<BM>(start, ne, t, 0, 0, 0, flag);
        head = uniform((int64_t)__shfl(first.end, 0, 64));
        Chunk c = first;
        for (int base = 64; base <= ne; base += 64)
            c = scan<BM>(start, ne, t, base, __shfl(c.end, 63, 64), __shfl(c.before + c.mine, 63, 64), flag);
        experts = uniform((int64_t)__shfl(c.before + c.mine, 63, 64));
        reach = uniform((int64_t)__shfl(c.end, 63, 64));
    }
    __device__ __forceinline__ int64_t count() const { return experts + (head + BM - 1) / BM + (t - reach + BM - 1) / BM; }
    __device__ __forceinline__ Rows at(int64_t piece) const {
        if (piece >= experts) {
            piece -= experts;
            const int64_t heads = (head + BM - 1) / BM;
            const int64_t row = piece < heads ? piece * BM : reach + (piece - heads) * BM, end = piece < heads ? head : t;
            return Rows{-1, row, (int)min((int64_t)BM, end - row)};
        }
        Chunk c = first;
        for (int base = 0;;) {
            const uint64_t hit = __ballot(c.mine > 0 && piece >= c.before && piece < c.before + c.mine);
            if (hit) {
                const int l = __builtin_ctzll(hit);
                const int64_t row = __shfl(c.from, l, 64) + (piece - __shfl(c.before, l, 64)) * BM;
                return uniform(Rows{base + l - 1, row, (int)min((int64_t)BM, __shfl(c.end, l, 64) - row)});
            }
            base += 64;   // (a piece below `experts` is found before the offsets end)
            if (base > ne) return Rows{-1, 0, 0};
            c = scan<BM>(start, ne, t, base, __shfl(c.end, 63, 64), __shfl(c.before + c.mine, 63, 64), nullptr);
        }
    }
};

// expert e's rows
__device__ __forceinline__ Rows expert_rows(const int64_t* start, int ne, int64_t t, int e, int32_t* flag) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = 0, raw = 0;
    for (int base = 0; base <= e + 1; base += 64) {
        const int i = base + lane;
        raw = i <= e + 1 ? start[i] : 0;
        if (i <= e + 1 && (raw < 0 || raw > t) && flag) *flag = kErrIndex;
        int64_t a = i <= e ? min(max(raw, (int64_t)0), t) : 0, b = i <= e + 1 ? min(max(raw, (int64_t)0), t) : 0;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            a = max(a, (int64_t)__shfl_xor(a, o, 64));
            b = max(b, (int64_t)__shfl_xor(b, o, 64));
        }
        lo = max(lo, a);
        hi = max(hi, b);
    }
    if (lane == ((e + 1) & 63) && raw < lo && flag) *flag = kErrIndex;
    return Rows{e, lo, (int)(hi - lo)};
}

// ------------------------------------------------------------------------------------------
// One product: tiles of BM x BN of the result on the matrix cores
// ------------------------------------------------------------------------------------------
struct Mul {
    const void* a; int64_t lda;            // rows (x, or yb for xb)
    const void* b; int64_t ldb;            // w, or yb for wb
    void* c; int64_t ldc;
    const uint8_t* q; const uint8_t* qs;   // the rows' tape in place of a (wb)
    const int64_t* start;
    int ne;
    int64_t t;
    int m, n, k;       // of one expert's product (m of xb and y, k of wb: its rows)
    int tiles_n;       // column tiles
    int64_t pieces;    // row pieces at most (y, xb), or experts times row tiles (wb)
    int add;
    int cus;           // of the device
    int split;         // slices of k (1: none); a slice's result goes to the c'th of so many whole results, fp32
    int32_t* flag;
};

enum Form { Y = 0, XB = 1, WB = 2 };

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef float v4f __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short v4s __attribute__((ext_vector_type(4)));

// Operand tiles in LDS, in 16-byte chunks of CE values.  A step takes BK values of k.
//   k-contiguous operand (x and yb rows; w for xb): ROWS rows of 128 bytes; row r holds its chunk c at
//     place c ^ (r / 2 & 7), so that sixteen lanes that read one chunk of sixteen rows meet all the banks.
//   row-contiguous operand (w for y; x and yb for wb): BK rows of ROWS values.  The 16-bit types are
//     read through the transposing LDS read (16 lanes: four k of 16 rows, 32 bytes of each); the 32-byte
//     pieces of row k lie at place p ^ turn_of(k), so that no two of the eight pieces that half a wave reads,
//     be it lanes 0..31 or every other 16, lie on the same banks.
template <class T> constexpr int kBK = 128 / (int)sizeof(T);
template <class T> constexpr int kCE = 16 / (int)sizeof(T);

template <int ROWS>
__device__ __forceinline__ int turn_of(int k) {
    return ((k & 3) << 1 | (k >> 3 & 1)) & (ROWS / 16 - 1);
}

// byte offset of chunk `c` of row `r` (KC), or of row k (not KC), in its tile
template <class T, bool KC, int ROWS>
__device__ __forceinline__ int chunk_at(int r, int c) {
    if constexpr (KC) return r * 128 + ((c ^ (r >> 1 & 7)) << 4);
    else if constexpr (sizeof(T) == 2) return r * ROWS * 2 + ((((c >> 1) ^ turn_of<ROWS>(r)) << 5) | ((c & 1) << 4));
    else return r * ROWS * 4 + (c << 4);
}

// A thread's chunks of a tile: chunk number NT i + tid, in the order of the places, so that a wave's
// lanes fill consecutive places.  (row, first value) of the operand's own indexes: KC: row of ROWS and
// k; else k and row.
template <class T, bool KC, int ROWS, int NT>
__device__ __forceinline__ void my_chunk(int i, int& outer, int& inner) {
    const int at = i * NT + threadIdx.x;
    if constexpr (KC) {
        outer = at >> 3;
        inner = ((at & 7) ^ (outer >> 1 & 7)) * kCE<T>;
    } else {
        constexpr int PER = ROWS / kCE<T>;
        outer = at / PER;
        int c = at % PER;
        if constexpr (sizeof(T) == 2) c = ((c >> 1) ^ turn_of<ROWS>(outer)) << 1 | (c & 1);
        inner = c * kCE<T>;
    }
}

// 16 bytes of the operand through registers, at any alignment: the first `left` values, and zeros.  PAST: what
// lies behind them may come along instead of the zeros, as far as the matrix goes (`end`).
template <bool PAST, class T>
__device__ __forceinline__ v4u load_chunk(const T* p, int left, const T* end) {
    typedef T vec __attribute__((ext_vector_type(kCE<T>)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    vec v = {};
    if (left >= kCE<T> || (PAST && left > 0 && p + kCE<T> <= end)) {
        v = *reinterpret_cast<const loose*>(p);
    } else if (left > 0) {   // (rare, and every load is waited for: lanes without values stay out)
#pragma unroll
        for (int i = 0; i < kCE<T>; ++i) v[i] = i < left ? p[i] : (T)0.f;
    }
    return __builtin_bit_cast(v4u, v);
}

// 16 bytes a lane from the buffer `r` at `off` to LDS, the wave's lanes from `at` on.  In assembly because
// of the waits: for the builtin the compiler waits for all loads before the next LDS read of any
// kind, as it cannot tell the buffers apart, and nothing is left in flight during the products.  It has
// no output register (m0 is reserved: the compiler keeps nothing in it); wait_loads below counts it.
__device__ __forceinline__ void load_to_lds(v4u r, uint32_t off, uint32_t at) {
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tbuffer_load_dwordx4 %0, %1, 0 offen lds" ::"v"(off), "s"(r), "s"(at) : "memory");
}

// An operand's staging.  The chunks of the step at k0 go from memory to registers (load), and
// later to LDS (store); or straight to LDS (DIRECT: 16-byte aligned rows, whole chunks).
// `rows`: of this tile; `kmax`: the product's k.
template <class T, bool KC, int ROWS, int NT>
struct Stage {
    static constexpr int PER = ROWS * 128 / 16 / NT;
    static_assert(ROWS * 8 % NT == 0, "whole chunks a thread");
    const T* p;
    int64_t ld;
    int rows, kmax;
    const T* end;    // of the whole matrix

    using Held = v4u;
    __device__ __forceinline__ void load(Held& v, int i, int k0) const {
        int o, n;
        my_chunk<T, KC, ROWS, NT>(i, o, n);
        const int left = KC ? (o < rows ? kmax - k0 - n : 0) : (k0 + o < kmax ? rows - n : 0);
        // (rows past the tile's make results that are not stored; k past the product's must be zeros)
        v = load_chunk<!KC>(KC ? p + (int64_t)o * ld + k0 + n : p + (int64_t)(k0 + o) * ld + n, left, end);
    }
    __device__ __forceinline__ static void store(const Held& v, int i, char* lds) {
        *reinterpret_cast<v4u*>(lds + (i * NT + threadIdx.x) * 16) = v;
    }
    // straight to LDS: lanes past the rows or past k get an offset past the buffer, and zeros
    __device__ __forceinline__ void direct(const char* lds, int k0) const {
        const uint64_t base = (uint64_t)(KC ? p + k0 : p + (int64_t)k0 * ld);
        const v4u r = {(uint32_t)base, (uint32_t)(base >> 32) & 0xffffu, 0x7fffffffu, 0x00020000u};
        const uint32_t at = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const char*)lds + uniform((int)(threadIdx.x >> 6)) * 1024;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int o, n;
            my_chunk<T, KC, ROWS, NT>(i, o, n);
            const bool here = KC ? o < rows && k0 + n < kmax : k0 + o < kmax && n < rows;
            load_to_lds(r, here ? (uint32_t)o * (uint32_t)ld * sizeof(T) + n * sizeof(T) : 0x80000000u, at + i * NT * 16);
        }
    }
};

// the tape's staging (a row-contiguous operand): 8 bytes and a scale become 8 values, exactly
template <class T, int ROWS, int NT>
struct TapeStage {
    static constexpr int CE = kCE<T>, PER = ROWS * 128 / 16 / NT;
    const uint8_t* q; const uint8_t* qs;   // at the expert's first row
    int64_t ng;
    int col, rows, kmax;                   // the tile's first column of the tape's rows

    // (by buffer loads, one for the bytes and one for the scale at every step: chunks past the rows or
    // past k are zeros, and the loads in flight can be counted)
    static constexpr int LOADS = 2 * PER;
    typedef uint32_t Bytes __attribute__((ext_vector_type(CE / 4)));
    struct Held { Bytes q; uint8_t s; };
    __device__ __forceinline__ void load(Held& v, int i, int k0) const {
        const __amdgpu_buffer_rsrc_t rq = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(q + (int64_t)k0 * ng * tape8::kGroup), (short)0,
                                                                            0x7fffffff, 0x00020000);
        const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(qs + (int64_t)k0 * ng), (short)0, 0x7fffffff,
                                                                            0x00020000);
        int o, n;
        my_chunk<T, false, ROWS, NT>(i, o, n);
        const bool here = k0 + o < kmax && n < rows;   // (a chunk past the last value is zeros in the tape)
        const uint32_t at = (uint32_t)o * (uint32_t)ng;
        const uint32_t oq = here ? at * tape8::kGroup + col + n : 0x80000000u, os = here ? at + (col + n) / tape8::kGroup : 0x80000000u;
        if constexpr (CE == 8) v.q = __builtin_bit_cast(Bytes, __builtin_amdgcn_raw_buffer_load_b64(rq, oq, 0, 0));
        else v.q = (Bytes)(__builtin_amdgcn_raw_buffer_load_b32(rq, oq, 0, 0));
        v.s = __builtin_amdgcn_raw_buffer_load_b8(rs, os, 0, 0);
    }
    __device__ __forceinline__ static void store(const Held& v, int i, char* lds) {
        typedef T vec __attribute__((ext_vector_type(CE)));
        const float u = tape8::unit(v.s);
        vec x;
#pragma unroll
        for (int j = 0; j < CE; ++j) x[j] = (T)tape8::value(v.q[j >> 2] ^ 0x80808080u, j & 3, u);
        *reinterpret_cast<v4u*>(lds + (i * NT + threadIdx.x) * 16) = __builtin_bit_cast(v4u, x);
    }
};

// A lane's values of 32 rows from `row0` and the s-th quarter of a step: 16-bit types k = 16 s + 8 h + 0..7
// of row lane % 32, h = lane / 32; fp32 k = 8 s + 4 h + 0..3.
template <class T, bool KC, int ROWS>
__device__ __forceinline__ v4u fragment(const char* lds, int row0, int s) {
    const int lane = threadIdx.x & 63, h = lane >> 5;
    if constexpr (KC) {
        return *reinterpret_cast<const v4u*>(lds + chunk_at<T, true, ROWS>(row0 + (lane & 31), 2 * s + h));
    } else if constexpr (sizeof(T) == 2) {
        const int k = 16 * s + 8 * h + ((lane & 15) >> 2), seg = ((row0 >> 4) + ((lane >> 4) & 1)) ^ turn_of<ROWS>(k);
        const char* at = lds + k * ROWS * 2 + seg * 32 + (lane & 3) * 8;
        typedef __attribute__((address_space(3))) v4s* lp;
        const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at)), hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)(at + 4 * ROWS * 2));
        typedef short v8s __attribute__((ext_vector_type(8)));
        return __builtin_bit_cast(v4u, (v8s){lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]});
    } else {
        v4f v;
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(lds + (8 * s + 4 * h + j) * ROWS * 4 + (row0 + (lane & 31)) * 4);
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

// A tile's place in the order of the tiles: kBand row pieces by all the columns, band after band, so that
// the tiles which run at one time share rows and columns in L2.
constexpr int kBand = 4;
__device__ __forceinline__ void tile_place(int64_t id, int64_t pieces, int tiles_n, int64_t& piece, int& tn) {
    const int64_t band = id / (kBand * tiles_n), in = id - band * kBand * tiles_n, rows = min((int64_t)kBand, pieces - band * kBand);
    tn = (int)(in / rows);
    piece = band * kBand + in % rows;
}
// Blocks go round the 8 XCDs, each with an L2 of its own: an XCD gets a range of the tiles that lie
// together; of wb, whose experts differ in their work, a range of each expert's tiles.  items(): how many
// numbers there are (some without a tile); item_place(): a number's tile, or false.
template <int FORM>
__device__ __forceinline__ int64_t items(const Mul& p, int64_t pieces) {
    if constexpr (FORM == WB) return (pieces / p.ne * p.tiles_n + 7) / 8 * 8 * p.ne;
    else return (pieces * p.tiles_n + 7) / 8 * 8;
}
template <int FORM>
__device__ __forceinline__ bool item_place(const Mul& p, int64_t item, int64_t pieces, int64_t& piece, int& tn) {
    if constexpr (FORM == WB) {
        const int64_t mine = pieces / p.ne, per = (mine * p.tiles_n + 7) / 8, slot = item >> 3, e = slot / per;
        const int64_t id = ((item + e) & 7) * per + slot - e * per;   // (turned by e: few tiles an expert go round too)
        if (id >= mine * p.tiles_n) return false;
        tile_place(id, mine, p.tiles_n, piece, tn);
        piece += e * mine;
    } else {
        const int64_t total = pieces * p.tiles_n, per = (total + 7) / 8, id = (item & 7) * per + (item >> 3);
        if (id >= total || (item >> 3) >= per) return false;
        tile_place(id, pieces, p.tiles_n, piece, tn);
    }
    return true;
}

// wait until at most N of the wave's loads are under way
template <int N>
__device__ __forceinline__ void wait_loads() {
    static_assert(N < 64);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// One tile by a block.  ST buffers in LDS go round.  Straight loads of a step are issued ST - 1 steps before
// it; what comes through registers is loaded two steps before and put into LDS one step before, a part
// between each two quarters of the products.  One barrier a step: behind it the next step's tiles are
// whole, and the buffer of this one is free.
// The tile: rows m0 .. of the piece r (y, xb), or of expert r.e's weights (wb); columns n0 .. .
template <class T, class TC, int FORM, bool TAPE, bool DIRECT, int BM, int BN, int WM, int WN, int ST>
struct Tile {
    static constexpr int NT = 64 * WM * WN, MT = BM / WM / 32, NTL = BN / WN / 32, BK = kBK<T>, LDS = ST * (BM + BN) * 128;
    static_assert(ST == 2 || (DIRECT && !TAPE), "more buffers are for straight loads");
    static __device__ __forceinline__ void run(const Mul& p, Rows r, int m0, int n0, char* lds, int slice = 0) {
    const int rows = min(BM, (FORM == WB ? p.m : r.rows) - m0), cols = min(BN, p.n - n0);
    if (rows <= 0 || cols <= 0) return;
    constexpr bool AKC = FORM != WB, BKC = FORM == XB;
    using SA = std::conditional_t<TAPE, TapeStage<T, BM, NT>, Stage<T, AKC, BM, NT>>;
    using SB = Stage<T, BKC, BN, NT>;
    int k = FORM == WB ? r.rows : r.e < 0 ? 0 : p.k, k_first = 0;
    if (p.split > 1) {   // this slice's part of k
        const int each = ((k + p.split - 1) / p.split + BK - 1) / BK * BK;
        k_first = min(k, slice * each);
        k = min(k - k_first, each);
        if (FORM == WB) r.row += k_first;
    }
    const int steps = (k + BK - 1) / BK;
    const int64_t e = r.e < 0 ? 0 : r.e;
    const T* b = (const T*)p.b + (FORM == WB ? r.row * p.ldb + n0 : FORM == Y ? (e * p.k + k_first) * p.n + n0 : (e * p.n + n0) * p.k + k_first);
    const SB sb{b, p.ldb, cols, k, (const T*)p.b + (FORM == WB ? (p.t - 1) * p.ldb + p.n : (int64_t)p.ne * p.k * p.n)};
    SA sa;
    if constexpr (TAPE) {
        const int64_t ng = tape8::groups(p.m);
        sa = SA{p.q + r.row * ng * tape8::kGroup, p.qs + r.row * ng, ng, m0, rows, k};
    } else {
        sa = SA{(const T*)p.a + (FORM == WB ? r.row * p.lda + m0 : (r.row + m0) * p.lda + k_first), p.lda, rows, k,
                (const T*)p.a + (p.t - 1) * p.lda + (FORM == WB ? p.m : p.k)};
    }

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / WN * MT * 32, wn = wave % WN * NTL * 32;
    floatx16 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;

    const auto buffer = [&](int t) { return lds + t % ST * ((BM + BN) * 128); };
    constexpr bool AREG = TAPE || !DIRECT, BREG = !DIRECT;
    typename SA::Held ra[AREG ? SA::PER : 1];
    typename SB::Held rb[BREG ? SB::PER : 1];
    const auto straight = [&](int t) {
        char* at = buffer(t);
        if constexpr (!AREG) sa.direct(at, t * BK);
        if constexpr (!BREG) sb.direct(at + BM * 128, t * BK);
    };
    // part s of 4: what the registers hold goes to `at`, and step t's values take its place
    const auto part = [&](int s, char* at, int t, bool put, bool get) {
        if constexpr (AREG) {
#pragma unroll
            for (int i = SA::PER * s / 4; i < SA::PER * (s + 1) / 4; ++i) {
                if (put) SA::store(ra[i], i, at);
                if (get) sa.load(ra[i], i, t * BK);
            }
        }
        if constexpr (BREG) {
#pragma unroll
            for (int i = SB::PER * s / 4; i < SB::PER * (s + 1) / 4; ++i) {
                if (put) SB::store(rb[i], i, at + BM * 128);
                if (get) sb.load(rb[i], i, t * BK);
            }
        }
    };
    // the fragments of quarter s of step t, into one of two sets of registers
    v4u fa[2][MT], fb[2][NTL];
    const auto read = [&](int t, int s) {
        const char *A = buffer(t), *B = A + BM * 128;
#pragma unroll
        for (int i = 0; i < MT; ++i) fa[s & 1][i] = fragment<T, AKC, BM>(A, wm + 32 * i, s);
#pragma unroll
        for (int j = 0; j < NTL; ++j) fb[s & 1][j] = fragment<T, BKC, BN>(B, wn + 32 * j, s);
    };
    const auto products = [&](int s) {
        // (the weights come first: each lane gets four consecutive columns of one row)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
            for (int j = 0; j < NTL; ++j) acc[i][j] = multiply<T>(fb[s & 1][j], fa[s & 1][i], acc[i][j]);
    };
    if (steps > 0) {
        if constexpr (AREG || BREG) {
            // (past the last step the operands' guards give zeros)
#pragma unroll
            for (int s = 0; s < 4; ++s) part(s, lds, 0, false, true);
#pragma unroll
            for (int s = 0; s < 4; ++s) part(s, lds, 1, true, true);
        }
        for (int t = 0; t < ST - 1; ++t) straight(t);
        if constexpr (DIRECT) wait_loads<TAPE ? 0 : (ST - 2) * (SA::PER + SB::PER)>();
        __syncthreads();
        straight(ST - 1);
        read(0, 0);
    }
    for (int t = 0; t < steps; ++t) {
        char* next = buffer(t + 1);
#pragma unroll
        for (int s = 0; s < 3; ++s) {
            read(t, s + 1);
            __builtin_amdgcn_sched_barrier(0);
            products(s);
            if constexpr (AREG || BREG) part(s, next, t + 2, true, true);
        }
        if constexpr (AREG || BREG) part(3, next, t + 2, true, true);
        // the step's fragments are read and the next step's tiles are there (behind its straight loads
        // only the tape's, or those of later steps, are under way): the buffer of step t is free
        if constexpr (TAPE && DIRECT) wait_loads<TapeStage<T, BM, NT>::LOADS>();
        else if constexpr (DIRECT) wait_loads<(ST - 2) * (SA::PER + SB::PER)>();
        __syncthreads();
        // (the loads in two parts around the products: all at once before them cost 4 % of a large product)
        read(t + 1, 0);
        if constexpr (!AREG) sa.direct(buffer(t + ST), (t + ST) * BK);
        __builtin_amdgcn_sched_barrier(0);
        products(3);
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!BREG) sb.direct(buffer(t + ST) + BM * 128, (t + ST) * BK);
    }
    if constexpr (DIRECT) wait_loads<0>();   // (of steps past the last: nothing may land after the block's end)
    // A lane has row lane % 32 of each 32 and columns 8 g + 4 (lane / 32) + 0..3 of each 32: each wave
    // turns 32 rows at a time in LDS of its own, so that a row's columns go out together (straight
    // from the registers a store touches 32 rows with 16 or 32 bytes each, 7 us more for a 256 x 256 tile).
    // The 16-byte chunks of row r lie at place c ^ (r & 7).
    constexpr int CE = kCE<TC>, CHUNKS = NTL * 32 / CE;
    static_assert(WM * WN * 32 * CHUNKS * 16 <= LDS && CHUNKS >= 4, "the waves' parts fit");
    __syncthreads();
    char* own = lds + wave * (32 * CHUNKS * 16);
    TC* c = (TC*)p.c + (FORM == WB ? ((int64_t)r.e * p.m + m0) * p.n : (r.row + m0) * p.ldc) + n0;
    if (p.split > 1) c += slice * (FORM == WB ? (int64_t)p.ne * p.m : p.t) * p.n;
    const int64_t ldc = FORM == WB ? p.n : p.ldc;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = lane & 31;
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                typedef TC vec __attribute__((ext_vector_type(4)));
                vec v;
#pragma unroll
                for (int x = 0; x < 4; ++x) v[x] = (TC)0.f;
                if constexpr (sizeof(TC) == 4) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = acc[i][j][4 * g + x];
                    *reinterpret_cast<vec*>(own + (row * CHUNKS + ((8 * j + 2 * g + (lane >> 5)) ^ (row & 7 & (CHUNKS - 1)))) * 16) = v;
                } else if (!p.add) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = (TC)acc[i][j][4 * g + x];
                    *reinterpret_cast<vec*>(own + (row * CHUNKS + ((4 * j + g) ^ (row & 7 & (CHUNKS - 1)))) * 16 + 8 * (lane >> 5)) = v;
                }
            }
        if (sizeof(TC) == 4 || !p.add) {
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int q = 0; q < 32 * CHUNKS / 64; ++q) {
                const int at = q * 64 + lane, rr = at / CHUNKS, cc = at % CHUNKS, col = wn + cc * CE, mm = wm + 32 * i + rr;
                typedef TC vec __attribute__((ext_vector_type(CE)));
                const vec v = *reinterpret_cast<const vec*>(own + (rr * CHUNKS + (cc ^ (rr & 7 & (CHUNKS - 1)))) * 16);
                if (mm < rows && col < cols) {
                    float f[CE];
                    TC* to = c + mm * ldc + col;
                    if (p.add) {
                        load_row(f, to, cols - col);
#pragma unroll
                        for (int x = 0; x < CE; ++x) f[x] += (float)v[x];
                    } else {
#pragma unroll
                        for (int x = 0; x < CE; ++x) f[x] = (float)v[x];
                    }
                    store_row(to, f, cols - col);
                }
            }
            __builtin_amdgcn_wave_barrier();
        } else {
            // (16-bit results that add to what is there are rounded once: straight from the registers)
            const int mm = wm + 32 * i + row;
            if (mm < rows) {
#pragma unroll
                for (int j = 0; j < NTL; ++j)
#pragma unroll
                    for (int g = 0; g < 4; ++g) {
                        const int col = wn + 32 * j + 8 * g + 4 * (lane >> 5);
                        if (col >= cols) continue;
                        float f[4];
                        TC* to = c + mm * ldc + col;
                        load_row(f, to, cols - col);
#pragma unroll
                        for (int x = 0; x < 4; ++x) f[x] += acc[i][j][4 * g + x];
                        store_row(to, f, cols - col);
                    }
            }
        }
    }
    }
};

// buffers of a tile of 64 x 64
constexpr int small_buffers(bool tape, bool direct) { return direct && !tape ? 4 : 2; }

// the piece that holds tile `piece` of the pieces of BM rows, and its first row in it
template <int FORM, int BM>
__device__ __forceinline__ Rows piece_rows(const Mul& p, const Pieces<BM>* all, int64_t piece, int& m0) {
    if constexpr (FORM == WB) {
        const int tiles_m = (p.m + BM - 1) / BM;
        m0 = (int)(piece % tiles_m) * BM;
        return uniform(expert_rows(p.start, p.ne, p.t, (int)(piece / tiles_m), p.flag));
    } else {
        m0 = 0;
        return all->at(piece);
    }
}

// (where results are added to what is there, rows of no expert and experts without rows change nothing: 24 rows that go to
// 2 of 8 experts, 2048 x 4096, bf16: wb in fp32 36 us, 96 with the others read and written)
__device__ __forceinline__ bool nothing(const Mul& p, const Rows& r) { return p.add && (r.e < 0 || r.rows == 0); }

// one size of tile: block `block` of the launch
template <class One, int FORM, int BM, int BN>
__device__ __forceinline__ void product(const Mul& p, unsigned block, char* lds) {
    const Pieces<BM> all(p.start, FORM == WB ? 0 : p.ne, p.t, FORM == WB ? nullptr : p.flag);
    const int64_t pieces = FORM == WB ? p.pieces : all.count();
    int64_t piece;
    int tn, m0;
    const int64_t all_items = items<FORM>(p, pieces);
    const int slice = (int)(block / all_items);
    if (slice >= p.split || !item_place<FORM>(p, block % all_items, pieces, piece, tn)) return;
    const Rows r = piece_rows<FORM, BM>(p, &all, piece, m0);
    if (nothing(p, r)) return;
    One::run(p, r, m0, tn * BN, lds, slice);
}
template <class T, class TC, int FORM, bool TAPE, bool DIRECT, int BM, int BN, int WM, int WN, int ST>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(Mul p) {
    using One = Tile<T, TC, FORM, TAPE, DIRECT, BM, BN, WM, WN, ST>;
    __shared__ char lds[One::LDS];
    product<One, FORM, BM, BN>(p, blockIdx.x, lds);
}

// xb and wb in one launch, where both take tiles of 64 x 64: the first blocks, a multiple of 8, are xb's
template <class T, class TC, bool TAPE, bool DIRECT>
__global__ __launch_bounds__(256) void shadows_kernel(Mul px, Mul pw, unsigned first) {
    using X = Tile<T, T, XB, false, DIRECT, 64, 64, 2, 2, small_buffers(false, DIRECT)>;
    using W = Tile<T, TC, WB, TAPE, DIRECT, 64, 64, 2, 2, small_buffers(TAPE, DIRECT)>;
    __shared__ char lds[X::LDS > W::LDS ? X::LDS : W::LDS];
    if (blockIdx.x < first) product<X, XB, 64, 64>(px, blockIdx.x, lds);
    else product<W, WB, 64, 64>(pw, blockIdx.x - first, lds);
}

// Large tiles, 256 x 256, for as many whole rounds as the CUs make of them (one block a CU); the rest,
// where it would leave half of the CUs or more idle, in 128 x 128 quarters: a round of those takes
// less than half as long.
template <class T, class TC, int FORM, bool TAPE, bool DIRECT>
__global__ __launch_bounds__(512) void mixed_kernel(Mul p) {
    using Large = Tile<T, TC, FORM, TAPE, DIRECT, 256, 256, 2, 4, 2>;
    using Quarter = Tile<T, TC, FORM, TAPE, DIRECT, 128, 128, 2, 4, DIRECT && !TAPE ? 4 : 2>;
    __shared__ char lds[Large::LDS > Quarter::LDS ? Large::LDS : Quarter::LDS];
    const Pieces<256> all(p.start, FORM == WB ? 0 : p.ne, p.t, FORM == WB ? nullptr : p.flag);
    const int64_t pieces = FORM == WB ? p.pieces : all.count(), total = items<FORM>(p, pieces);
    const int64_t rest = total % p.cus, large = rest <= p.cus / 2 ? total - rest : total;
    int64_t piece, item = blockIdx.x;
    int tn, m0, quarter = -1;
    if (item >= large) {   // (a tile's quarters lie 8 blocks apart: on one XCD)
        const int64_t b = item - large;
        quarter = (int)(b >> 3 & 3);
        item = large + ((b >> 5) << 3 | (b & 7));
        if (item >= total) return;
    }
    if (!item_place<FORM>(p, item, pieces, piece, tn)) return;
    const Rows r = piece_rows<FORM, 256>(p, &all, piece, m0);
    if (nothing(p, r)) return;
    if (quarter < 0) Large::run(p, r, m0, tn * 256, lds);
    else Quarter::run(p, r, m0 + (quarter >> 1) * 128, tn * 256 + (quarter & 1) * 128, lds);
}

// the slices' results added in order: 8 columns of a row a thread
template <class TC>
__global__ __launch_bounds__(256) void join_kernel(const float* part, int slices, TC* c, int64_t ldc, int64_t rows, int n, int add) {
    const int vecs = (n + 7) / 8;
    const int64_t all = rows * vecs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += (int64_t)gridDim.x * 256) {
        const int64_t row = i / vecs;
        const int col = (int)(i - row * vecs) * 8;
        float sum[8], v[8];
        load_row(sum, part + row * n + col, n - col);
        for (int s = 1; s < slices; ++s) {
            load_row(v, part + ((int64_t)s * rows + row) * n + col, n - col);
#pragma unroll
            for (int x = 0; x < 8; ++x) sum[x] += v[x];
        }
        TC* to = c + row * ldc + col;
        if (add) {
            load_row(v, to, n - col);
#pragma unroll
            for (int x = 0; x < 8; ++x) sum[x] += v[x];
        }
        store_row(to, sum, n - col);
    }
}

// the tiles of p, and of its launch; or an error
template <int FORM, int BM, int BN, int NT>
int32_t count_tiles(Mul& p, int64_t& tiles, const char* name) {
    p.tiles_n = (p.n + BN - 1) / BN;
    p.pieces = FORM == WB ? (int64_t)p.ne * ((p.m + BM - 1) / BM) : (p.t + BM - 1) / BM + p.ne + 2;
    tiles = FORM == WB ? ((p.m + BM - 1) / BM * p.tiles_n + 7) / 8 * 8 * p.ne : (p.pieces * p.tiles_n + 7) / 8 * 8;
    // (a launch has less than 2^32 threads)
    if ((tiles + 4 * (int64_t)p.cus) * p.split >= (1ll << 32) / NT) return set_error(STADE_HIP_ERANGE, "%s: too many tiles for a launch", name);
    return 0;
}

template <class T, class TC, int FORM, bool TAPE, bool DIRECT, int BM, int BN, int WM, int WN, int ST = 2>
int32_t launch(Mul p, hipStream_t stream, const char* name) {
    if (BM == 256) p.split = 1;
    int64_t tiles;
    if (int32_t rc = count_tiles<FORM, BM, BN, 64 * WM * WN>(p, tiles, name)) return rc;
    if constexpr (BM == 256) {
        const unsigned blocks = (unsigned)(tiles + 3 * ((p.cus / 2 + 7) / 8 * 8));
        STADE_TIMED(name, stream, mixed_kernel<T, TC, FORM, TAPE, DIRECT><<<blocks, 512, 0, stream>>>(p));
    } else {
        STADE_TIMED(name, stream, product_kernel<T, TC, FORM, TAPE, DIRECT, BM, BN, WM, WN, ST><<<(unsigned)(tiles * p.split), 64 * WM * WN, 0, stream>>>(p));
    }
    STADE_LAUNCHED(name);
    return STADE_HIP_OK;
}

// whether all chunks of a matrix are whole and aligned, and a tile's offsets fit 31 bits
inline bool whole(const void* p, int64_t ld, int64_t d, int64_t tile, size_t size) {
    return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0 && d * size % 16 == 0 && tile * ld * (int64_t)size < (1ll << 31);
}

// How a product is done: by tiles of 64 x 64 (in `slices` of k), of 64 x 128 with three steps in flight, of 128 x 128, or of
// 256 x 256; `direct`: by straight loads
enum Size { SMALL, FLAT, MIDDLE, LARGE };
struct Plan {
    bool direct;
    Size size;
    int slices;
};
template <class T, int FORM, bool TAPE>
Plan plan(const Mul& p) {
    const bool direct = (TAPE || whole(p.a, p.lda, FORM == WB ? p.m : p.k, 256, sizeof(T))) &&
                        whole(p.b, p.ldb, FORM == XB ? p.k : p.n, 256, sizeof(T));
    // the tiles of 256 x 256 that the rows will make, half a tile more an expert
    const int64_t est = (FORM == WB ? (int64_t)p.ne * ((p.m + 255) / 256) : p.t / 256 + (p.ne + 1) / 2) * ((p.n + 255) / 256);
    // Fewer tiles of 64 x 64 than CUs and a long k: k in slices, for two blocks a CU, where that saves 12 steps or more
    // (a step takes a microsecond; the launch that adds the slices up takes five).  64 rows, 4 experts, 1672 x 2484, bf16: y
    // 43.4 -> 31.3 us, xb 45.7 -> 25.8; 3584 rows, 2 experts, 128 x 295: wb 37 -> 20; in fp32 137 rows, 4 experts, 1856 x 256: y
    // 71 -> 18.  Saving 8 steps: 1000 rows, 7 experts, 500 x 700, fp32: 18.7 -> 23.7.
    const int64_t small = std::max<int64_t>(1, (FORM == WB ? (int64_t)p.ne * ((p.m + 63) / 64) : p.t / 64 + std::min<int64_t>(p.ne, p.t)) * ((p.n + 63) / 64));
    // (no experts, no products: nothing to slice)
    const int64_t steps = p.ne == 0 ? 0 : (FORM == WB ? p.t / p.ne : p.k) / kBK<T>, slices = std::min<int64_t>(std::min<int64_t>(2 * p.cus / small, steps / 4), 32);
    if (small < p.cus && slices >= 2 && steps - steps / slices >= 12) return Plan{direct, SMALL, (int)slices};
    // Few rows an expert (y and xb: at most 64): bound by reading w, so small tiles, many blocks and three or four
    // steps in flight.  24 rows, 8 experts, 2048 x 4096, bf16: y 26.6 us (128 x 128 tiles 28.7, quarters 27.4), xb 24.8
    // (45, 37).
    const bool few = FORM != WB && p.t <= 64 * (int64_t)p.ne;
    if (direct && few) return Plan{direct, FORM == Y ? FLAT : SMALL, 1};
    // fp32 is bound by its matrix instructions: the tile that fills the CUs.  1000 rows, 7 experts, 500 x 700: y 15 us with
    // 64 x 64 tiles, 39 with 128 x 128 (xb 18 and 51, wb 17 and 18); 16384 rows, 16 experts, 2048 x 2048 (`est` 576):
    // y 1169 and 1016, xb 1121 and 997, wb 1192 and 1037.  Between these the rule takes the small tiles where the large
    // ones win: 8192 rows, 8 experts, 2048 x 1024 (`est` 144, of wb 256): y 296 and 258, xb 294 and 257, wb 302 and 262.
    if (sizeof(T) == 4) return Plan{direct, est < 2 * p.cus ? SMALL : MIDDLE, 1};
    // Less than a round of large tiles, more than one of quarters: 128 x 128 tiles of four waves, two
    // blocks a CU.  4096 rows, 8 experts, 1024 x 1024: 22.8 us, with quarters 29.0; 1024 rows, 4 experts,
    // 2048 x 2048, one round of quarters: 25.4 us, with these 28.4.
    if (direct) return Plan{direct, est < p.cus && 4 * est > p.cus ? MIDDLE : LARGE, 1};
    // Through registers: 1000 rows, 7 experts, 500 x 700 18 us, with large tiles and quarters 20.7; 24 rows, 8 experts,
    // 2044 x 4100 55 us (113); 8000 rows 377 us, with large tiles 245.
    return Plan{direct, few || 4 * est <= p.cus ? SMALL : LARGE, 1};
}

// the rows of a product's result, and the scratch that its slices take
template <int FORM>
int64_t result_rows(const Mul& p) {
    return FORM == WB ? (int64_t)p.ne * p.m : p.t;
}
template <int FORM>
size_t slice_bytes(const Mul& p, const Plan& how) {
    return how.slices > 1 ? (size_t)how.slices * result_rows<FORM>(p) * p.n * sizeof(float) : 0;
}

template <class T, class TC, int FORM, bool TAPE>
int32_t run(const Mul& p, hipStream_t stream, const char* name) {
    const Plan how = plan<T, FORM, TAPE>(p);
    if (how.slices > 1) {
        const int64_t rows = result_rows<FORM>(p);
        Mul q = p;
        q.split = how.slices;
        q.add = 0;
        q.ldc = p.n;
        if (!(q.c = scratch(slice_bytes<FORM>(p, how)))) return scratch_error();
        const int32_t rc = how.direct ? launch<T, float, FORM, TAPE, true, 64, 64, 2, 2, small_buffers(TAPE, true)>(q, stream, name)
                                      : launch<T, float, FORM, TAPE, false, 64, 64, 2, 2>(q, stream, name);
        if (rc) return rc;
        const unsigned grid = (unsigned)std::min<int64_t>((rows * ((p.n + 7) / 8) + 255) / 256, 1 << 14);
        STADE_TIMED("expert_mul_join", stream,
                    join_kernel<TC><<<grid, 256, 0, stream>>>((const float*)q.c, q.split, (TC*)p.c, FORM == WB ? p.n : p.ldc, rows, p.n, p.add));
        STADE_LAUNCHED("expert_mul join_kernel");
        return STADE_HIP_OK;
    }
    if constexpr (FORM == Y)
        if (how.size == FLAT) return launch<T, TC, FORM, TAPE, true, 64, 128, 1, 4, 3>(p, stream, name);
    if constexpr (sizeof(T) == 4 || FORM != WB)   // (wb of 16-bit types takes no small tiles by straight loads, but in slices)
        if (how.size == SMALL && how.direct) return launch<T, TC, FORM, TAPE, true, 64, 64, 2, 2, small_buffers(TAPE, true)>(p, stream, name);
    if (how.size == SMALL) return launch<T, TC, FORM, TAPE, false, 64, 64, 2, 2>(p, stream, name);
    if constexpr (sizeof(T) == 4) {
        if (how.direct) return launch<T, TC, FORM, TAPE, true, 128, 128, 2, 2>(p, stream, name);
        return launch<T, TC, FORM, TAPE, false, 128, 128, 2, 2>(p, stream, name);
    } else {
        if (how.size == MIDDLE) return launch<T, TC, FORM, TAPE, true, 128, 128, 2, 2>(p, stream, name);
        if (how.direct) return launch<T, TC, FORM, TAPE, true, 256, 256, 2, 4>(p, stream, name);
        return launch<T, TC, FORM, TAPE, false, 256, 256, 2, 4>(p, stream, name);
    }
}

// xb and wb.  One launch where both take small tiles: 1000 rows, 7 experts, 500 x 700, f16: 15.4 us, two launches
// 23.6; 4000 rows, 6 experts, 215 x 331, bf16: 16.9 and 24.5; fp32, 504 x 704: 28.5 and 38.8.
template <class T, class TC, bool TAPE>
int32_t run_both(Mul px, Mul pw, hipStream_t stream) {
    const Plan x = plan<T, XB, false>(px), w = plan<T, WB, TAPE>(pw);
    if (x.size == SMALL && w.size == SMALL && x.slices == 1 && w.slices == 1 && x.direct == w.direct) {
        int64_t first, more;
        if (int32_t rc = count_tiles<XB, 64, 64, 512>(px, first, "expert_mul_b")) return rc;
        if (int32_t rc = count_tiles<WB, 64, 64, 512>(pw, more, "expert_mul_b")) return rc;
        const auto go = [&](auto direct) -> int32_t {
            STADE_TIMED("expert_mul_b", stream,
                        shadows_kernel<T, TC, TAPE, decltype(direct)::value><<<(unsigned)(first + more), 256, 0, stream>>>(px, pw, (unsigned)first));
            STADE_LAUNCHED("expert_mul shadows_kernel");
            return STADE_HIP_OK;
        };
        if constexpr (sizeof(T) == 4)   // (as in run)
            if (x.direct) return go(std::true_type{});
        return go(std::false_type{});
    }
    // (a call that is refused its scratch enqueues nothing: the larger one's first)
    const size_t bytes = std::max(slice_bytes<XB>(px, x), slice_bytes<WB>(pw, w));
    if (bytes > 0 && !scratch(bytes)) return scratch_error();
    if (int32_t rc = run<T, T, XB, false>(px, stream, "expert_mul_xb")) return rc;
    return run<T, TC, WB, TAPE>(pw, stream, "expert_mul_wb");
}

int32_t check(const char* fn, int64_t tx, const int64_t* start, int64_t i_in, int64_t i_out, int64_t i_t, int64_t i_e) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_extent(fn, "i_in", i_in, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_out", i_out, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (int32_t rc = check_extent(fn, "i_e", i_e, kMostExperts)) return rc;
    return start ? 0 : bad(fn, "start is null");
}

int cu_count() {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
    return cus > 0 ? cus : 256;
}

int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

// Small products take scratch where large ones take none (`plan`): every eager call makes sure of what any product in
// slices needs, so that a smaller one may be captured after it.  There are at most 2 cus tiles of 64 x 64 in fp32: `slices`
// is 2 cus / small at most, and the result lies in `small` tiles (8 MiB for 256 CUs).
int32_t reserve(const WsCall& call, int cus) {
    const size_t bytes = (size_t)2 * cus * 64 * 64 * sizeof(float);
    if (call.capturing() || call.ws->scratch_bytes >= bytes) return 0;
    return scratch(bytes) ? 0 : scratch_error();
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_expert_mul(int64_t tx, void* y, int64_t ldy, const void* x, int64_t ldx, const void* w, const int64_t* start, int64_t i_in,
                             int64_t i_out, int64_t i_t, int64_t i_e, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_expert_mul";
    if (int32_t rc = check(fn, tx, start, i_in, i_out, i_t, i_e)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_out)) return rc;
    if (int32_t rc = check_ld(fn, "ldx", ldx, i_in)) return rc;
    if (i_t == 0 || i_out == 0) return STADE_HIP_OK;
    if (!y || (i_in > 0 && (!x || (i_e > 0 && !w)))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    Mul p{};
    p.a = x; p.lda = ldx; p.b = w; p.ldb = i_out; p.c = y; p.ldc = ldy;
    p.start = start; p.ne = (int)i_e; p.t = i_t; p.n = (int)i_out; p.k = (int)i_in; p.add = add != 0; p.flag = error_flag(call.ws);
    p.cus = cu_count();
    p.split = 1;
    if (int32_t rc = reserve(call, p.cus)) return rc;
    return with_type(tx, [&](auto t) -> int32_t { return run<decltype(t), decltype(t), Y, false>(p, stream, "expert_mul"); });
}

int32_t stade_hip_expert_mul_b(int64_t tx, int64_t twb, const void* yb, int64_t ldyb, const void* x, int64_t ldx, const int8_t* q,
                               const uint8_t* qs, void* xb, int64_t ldxb, const void* w, void* wb, const int64_t* start, int64_t i_in,
                               int64_t i_out, int64_t i_t, int64_t i_e, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_expert_mul_b";
    if (int32_t rc = check(fn, tx, start, i_in, i_out, i_t, i_e)) return rc;
    if (wb && twb != STADE_HIP_F32 && twb != tx) return bad(fn, "wb is neither Float32 nor of x's type");
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_out)) return rc;
    if (x)
        if (int32_t rc = check_ld(fn, "ldx", ldx, i_in)) return rc;
    if (xb)
        if (int32_t rc = check_ld(fn, "ldxb", ldxb, i_in)) return rc;
    if (i_in == 0 || (i_t == 0 && (!wb || add || i_out == 0 || i_e == 0))) return STADE_HIP_OK;
    if (i_t > 0 && i_out > 0 && (!yb || (xb && i_e > 0 && !w))) return bad(fn, "null pointer");
    if (wb && i_t > 0 && i_out > 0 && !x == !q) return bad(fn, "one of x and its tape (q, qs) is needed, and not both");
    if (!q != !qs) return bad(fn, "q and qs go together");
    if ((uintptr_t)q % 8) return bad(fn, "q is not aligned to 8 bytes");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    Mul p{};
    p.start = start; p.ne = (int)i_e; p.t = i_t; p.add = add != 0; p.flag = error_flag(call.ws);
    p.cus = cu_count();
    p.split = 1;
    if (int32_t rc = reserve(call, p.cus)) return rc;
    Mul px = p, pw = p;
    px.a = yb; px.lda = ldyb; px.b = w; px.ldb = i_out; px.c = xb; px.ldc = ldxb; px.n = (int)i_in; px.k = (int)i_out;
    pw.a = x; pw.lda = ldx; pw.q = (const uint8_t*)q; pw.qs = qs; pw.b = yb; pw.ldb = ldyb; pw.c = wb; pw.m = (int)i_in; pw.n = (int)i_out;
    const bool do_x = xb && i_t > 0, do_w = wb && i_out > 0 && i_e > 0;
    return with_type(tx, [&](auto t) -> int32_t {
        using T = decltype(t);
        if (!do_w) return do_x ? run<T, T, XB, false>(px, stream, "expert_mul_xb") : STADE_HIP_OK;
        const auto go = [&](auto tw, auto tape) -> int32_t {
            using TW = decltype(tw);
            constexpr bool TAPE = decltype(tape)::value;
            return do_x ? run_both<T, TW, TAPE>(px, pw, stream) : run<T, TW, WB, TAPE>(pw, stream, "expert_mul_wb");
        };
        if (twb == STADE_HIP_F32) return q ? go(float{}, std::true_type{}) : go(float{}, std::false_type{});
        return q ? go(t, std::true_type{}) : go(t, std::false_type{});
    });
}

}  // extern "C"
