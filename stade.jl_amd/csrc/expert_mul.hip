// Products of rows with the weights of the expert that each row was sent to, and their adjoint.
// The rows lie in expert order: expert e has the rows start[e] .. start[e+1] (any number, none too).
//
//   expert_mul     y[:, t]  (+)= w[:, :, e]  x[:, t]        (column-major: w is i_out x i_in x i_e)
//   expert_mul_b   xb[:, t] (+)= w[:, :, e]' yb[:, t],   wb[:, :, e] (+)= sum over e's rows of yb[:, t] x[:, t]'
//
// Row by row in memory: x[t][i], y[t][o], w[e][i][o]; so y = x w, xb = yb w^T, wb = x^T yb.
// Rows that no expert has get zeros (with `add`, nothing).
#include "tape8.hpp"

#include <algorithm>

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

// start[i] in order and in range: the largest of the offsets up to i, each between 0 and t.  (Offsets
// that are neither raise the device error flag; no row then has two experts.)
//
// The job-th piece of at most BM rows, all experts' pieces counted in order, then those of the
// rows before the first expert and after the last: every wave finds it by itself, 64 experts at a
// time.  No rows: e = -2.
template <int BM>
__device__ __forceinline__ Rows find_rows(const int64_t* start, int ne, int64_t t, int64_t job, int32_t* flag) {
    const int lane = threadIdx.x & 63;
    int64_t reach = 0, first = 0, pieces = 0;
    Rows r{-2, 0, 0};
    // boundary i of 0..ne: expert i - 1's end; segment i lies between boundaries i - 1 and i.
    // Segment 0 is the rows before the first expert; it is counted after the experts.
    for (int base = 0; base <= ne; base += 64) {
        const int i = base + lane;
        const int64_t raw = i <= ne ? start[i] : t;
        int64_t end = min(max(raw, (int64_t)0), t);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t up = __shfl_up(end, o, 64);
            if (lane >= o) end = max(end, up);
        }
        end = max(end, reach);
        if (i <= ne && end != raw && flag) *flag = kErrIndex;
        int64_t from = __shfl_up(end, 1, 64);
        if (lane == 0) from = reach;
        if (base == 0) first = __shfl(end, 0, 64);
        const int64_t mine = i >= 1 && i <= ne ? (end - from + BM - 1) / BM : 0;
        int64_t sum = mine;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int64_t up = __shfl_up(sum, o, 64);
            if (lane >= o) sum += up;
        }
        const int64_t before = pieces + sum - mine;
        const uint64_t hit = __ballot(mine > 0 && job >= before && job < before + mine);
        if (hit) {
            const int l = __builtin_ctzll(hit);
            const int64_t row = __shfl(from, l, 64) + (job - __shfl(before, l, 64)) * BM;
            r.e = base + l - 1;
            r.row = row;
            r.rows = (int)min((int64_t)BM, __shfl(end, l, 64) - row);
            return r;
        }
        pieces += __shfl(sum, 63, 64);
        reach = __shfl(end, 63, 64);
        if (base + 64 > ne) reach = __shfl(end, ne - base, 64);
    }
    job -= pieces;
    const int64_t head = (first + BM - 1) / BM;
    const int64_t row = job < head ? job * BM : reach + (job - head) * BM, end = job < head ? first : t;
    if (row < end) {
        r.e = -1;
        r.row = row;
        r.rows = (int)min((int64_t)BM, end - row);
    }
    return r;
}

// expert e's rows
__device__ __forceinline__ Rows expert_rows(const int64_t* start, int ne, int64_t t, int e, int32_t* flag) {
    const int lane = threadIdx.x & 63;
    int64_t lo = 0, hi = 0;
    for (int base = 0; base <= e + 1; base += 64) {
        const int i = base + lane;
        const int64_t raw = i <= e + 1 ? start[i] : 0;
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
    int64_t pieces;    // row pieces (y, xb), or experts times row tiles (wb)
    int add;
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
//     place c ^ (r & 7), so that eight lanes that read one chunk of eight rows meet all the banks.
//   row-contiguous operand (w for y; x and yb for wb): BK rows of ROWS values.  The 16-bit types are
//     read through the transposing LDS read (16 lanes: four k of 16 rows); the 64-byte pieces of
//     row k lie at place p ^ (k & 3), so that the four rows it reads lie on different banks.
template <class T> constexpr int kBK = 128 / (int)sizeof(T);
template <class T> constexpr int kCE = 16 / (int)sizeof(T);

// byte offset of chunk `c` of row `r` (KC), or of row k (not KC), in its tile
template <class T, bool KC, int ROWS>
__device__ __forceinline__ int chunk_at(int r, int c) {
    if constexpr (KC) return r * 128 + ((c ^ (r & 7)) << 4);
    else if constexpr (sizeof(T) == 2) return r * ROWS * 2 + ((((c >> 2) ^ (r & 3)) << 6) | ((c & 3) << 4));
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
        inner = ((at & 7) ^ (outer & 7)) * kCE<T>;
    } else {
        constexpr int PER = ROWS / kCE<T>;
        outer = at / PER;
        int c = at % PER;
        if constexpr (sizeof(T) == 2) c = ((c >> 2) ^ (outer & 3)) << 2 | (c & 3);
        inner = c * kCE<T>;
    }
}

// 16 bytes of the operand through registers: any alignment, zeros past `left` values
template <class T>
__device__ __forceinline__ v4u load_chunk(const T* p, int left) {
    typedef T vec __attribute__((ext_vector_type(kCE<T>)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
    vec v;
    if (left >= kCE<T>) {
        v = *reinterpret_cast<const loose*>(p);
    } else {
#pragma unroll
        for (int i = 0; i < kCE<T>; ++i) v[i] = i < left ? p[i] : (T)0.f;
    }
    return __builtin_bit_cast(v4u, v);
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

    __device__ __forceinline__ void load(v4u (&v)[PER], int k0) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int o, n;
            my_chunk<T, KC, ROWS, NT>(i, o, n);
            const int left = KC ? (o < rows ? kmax - k0 - n : 0) : (k0 + o < kmax ? rows - n : 0);
            v[i] = load_chunk(KC ? p + (int64_t)o * ld + k0 + n : p + (int64_t)(k0 + o) * ld + n, left);
        }
    }
    __device__ __forceinline__ static void store(const v4u (&v)[PER], char* lds) {
#pragma unroll
        for (int i = 0; i < PER; ++i) *reinterpret_cast<v4u*>(lds + (i * NT + threadIdx.x) * 16) = v[i];
    }
    // straight to LDS by buffer loads: lanes past the rows or past k get an offset past the buffer,
    // and zeros
    __device__ __forceinline__ void direct(char* lds, int k0) const {
        const T* base = KC ? p + k0 : p + (int64_t)k0 * ld;
        const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), (short)0, 0x7fffffff, 0x00020000);
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int o, n;
            my_chunk<T, KC, ROWS, NT>(i, o, n);
            const bool here = KC ? o < rows && k0 + n < kmax : k0 + o < kmax && n < rows;
            const uint32_t off = here ? (uint32_t)o * (uint32_t)ld * sizeof(T) + n * sizeof(T) : 0x80000000u;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(lds + (i * NT + wave * 64) * 16), 16, off, 0,
                                                     0, 0);
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

    struct Held { uint2 q[PER]; uint32_t s[PER]; };
    __device__ __forceinline__ void load(Held& v, int k0) const {
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            int o, n;
            my_chunk<T, false, ROWS, NT>(i, o, n);
            v.q[i] = make_uint2(0, 0);
            v.s[i] = 0;
            if (k0 + o < kmax && n < rows) {   // (a chunk past the last value is zeros in the tape)
                const int64_t row = k0 + o;
                const uint8_t* at = q + row * ng * tape8::kGroup + col + n;
                if constexpr (CE == 8) v.q[i] = *reinterpret_cast<const uint2*>(at);
                else v.q[i].x = *reinterpret_cast<const uint32_t*>(at);
                v.s[i] = qs[row * ng + (col + n) / tape8::kGroup];
            }
        }
    }
    __device__ __forceinline__ static void store(const Held& v, char* lds) {
        typedef T vec __attribute__((ext_vector_type(CE)));
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            // q + 128 as an unsigned byte, times the unit, less 128 units: exact
            const float u = tape8::unit(v.s[i]), low = -128.f * u;
            const uint32_t w[2] = {v.q[i].x ^ 0x80808080u, v.q[i].y ^ 0x80808080u};
            vec x;
#pragma unroll
            for (int j = 0; j < CE; ++j) x[j] = (T)fmaf((float)((w[j >> 2] >> (8 * (j & 3))) & 0xffu), u, low);
            *reinterpret_cast<v4u*>(lds + (i * NT + threadIdx.x) * 16) = __builtin_bit_cast(v4u, x);
        }
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
        const int k = 16 * s + 8 * h + ((lane & 15) >> 2), seg = (row0 >> 5) ^ (k & 3);
        const char* at = lds + k * ROWS * 2 + seg * 64 + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
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

// The tile's place.  Blocks go round the 8 XCDs, each with an L2 of its own: an XCD gets a range of
// tiles that lie together (kBand row pieces by all the columns), so that those which run at one
// time share rows and columns in its L2.
constexpr int kBand = 4;
__device__ __forceinline__ bool my_tile(const Mul& p, int64_t& piece, int& tn) {
    const int64_t total = p.pieces * p.tiles_n, per = (total + 7) / 8, id = (int64_t)(blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((blockIdx.x >> 3) >= per || id >= total) return false;
    const int64_t band = id / (kBand * p.tiles_n), in = id - band * kBand * p.tiles_n, rows = min((int64_t)kBand, p.pieces - band * kBand);
    tn = (int)(in / rows);
    piece = band * kBand + in % rows;
    return true;
}

template <class T, class TC, int FORM, bool TAPE, bool DIRECT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(64 * WM * WN) void product_kernel(Mul p) {
    constexpr int NT = 64 * WM * WN, MT = BM / WM / 32, NTL = BN / WN / 32, BK = kBK<T>;
    constexpr bool AKC = FORM != WB, BKC = FORM == XB;
    __shared__ char lds[2][(BM + BN) * 128];
    int64_t piece;
    int tn;
    if (!my_tile(p, piece, tn)) return;
    Rows r;
    int m0 = 0;
    if constexpr (FORM == WB) {
        const int tiles_m = (p.m + BM - 1) / BM;
        r = uniform(expert_rows(p.start, p.ne, p.t, (int)(piece / tiles_m), p.flag));
        m0 = (int)(piece % tiles_m) * BM;
    } else {
        r = uniform(find_rows<BM>(p.start, p.ne, p.t, piece, p.flag));
    }
    if (r.e == -2 || (r.e < 0 && p.add)) return;
    const int n0 = tn * BN, rows = FORM == WB ? min(BM, p.m - m0) : r.rows, cols = min(BN, p.n - n0);
    const int k = FORM == WB ? r.rows : r.e < 0 ? 0 : p.k;
    const int64_t e = r.e < 0 ? 0 : r.e;
    const T* b = (const T*)p.b + (FORM == WB ? r.row * p.ldb + n0 : FORM == Y ? e * p.k * p.n + n0 : (e * p.n + n0) * p.k);
    const Stage<T, BKC, BN, NT> sb{b, p.ldb, cols, k};
    const Stage<T, AKC, BM, NT> sa{(const T*)p.a + r.row * p.lda + m0, p.lda, rows, k};
    const int64_t ng = tape8::groups(p.m);
    const TapeStage<T, BM, NT> st{p.q + r.row * ng * tape8::kGroup, p.qs + r.row * ng, ng, m0, rows, k};

    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, wm = wave / WN * MT * 32, wn = wave % WN * NTL * 32;
    floatx16 acc[MT][NTL];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int x = 0; x < 16; ++x) acc[i][j][x] = 0.f;

    // (the weights come second: the operand order of the instruction gives each lane four
    // consecutive columns of one row)
    const auto compute = [&](const char* A, const char* B) {
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            v4u fa[MT], fb[NTL];
#pragma unroll
            for (int i = 0; i < MT; ++i) fa[i] = fragment<T, AKC, BM>(A, wm + 32 * i, s);
#pragma unroll
            for (int j = 0; j < NTL; ++j) fb[j] = fragment<T, BKC, BN>(B, wn + 32 * j, s);
#pragma unroll
            for (int i = 0; i < MT; ++i)
#pragma unroll
                for (int j = 0; j < NTL; ++j) acc[i][j] = multiply<T>(fb[j], fa[i], acc[i][j]);
        }
    };
    // While a step is multiplied from one pair of buffers, the next one comes into the other.
    v4u ra[Stage<T, AKC, BM, NT>::PER], rb[Stage<T, BKC, BN, NT>::PER];
    typename TapeStage<T, BM, NT>::Held rt;
    const auto fetch = [&](char* A, char* B, int k0) {
        if constexpr (TAPE) st.load(rt, k0);
        else if constexpr (DIRECT) sa.direct(A, k0);
        else sa.load(ra, k0);
        if constexpr (DIRECT) sb.direct(B, k0);
        else sb.load(rb, k0);
    };
    const auto settle = [&](char* A, char* B) {
        if constexpr (TAPE) st.store(rt, A);
        else if constexpr (!DIRECT) sa.store(ra, A);
        if constexpr (!DIRECT) sb.store(rb, B);
        if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    if (k > 0) {
        fetch(lds[0], lds[0] + BM * 128, 0);
        settle(lds[0], lds[0] + BM * 128);
        int turn = 0;
        for (int k0 = BK; k0 < k; k0 += BK) {
            char* next = lds[turn ^ 1];
            fetch(next, next + BM * 128, k0);
            compute(lds[turn], lds[turn] + BM * 128);
            settle(next, next + BM * 128);
            turn ^= 1;
        }
        compute(lds[turn], lds[turn] + BM * 128);
    }
    // lane: row lane % 32 of each 32, columns 8 g + 4 (lane / 32) + 0..3
    TC* c = (TC*)p.c + (FORM == WB ? ((int64_t)r.e * p.m + m0) * p.n : r.row * p.ldc) + n0;
    const int64_t ldc = FORM == WB ? p.n : p.ldc;
#pragma unroll
    for (int i = 0; i < MT; ++i) {
        const int row = wm + 32 * i + (lane & 31);
        if (row >= rows) continue;
#pragma unroll
        for (int j = 0; j < NTL; ++j)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const int col = wn + 32 * j + 8 * g + 4 * (lane >> 5);
                if (col >= cols) continue;
                float v[4];
                TC* at = c + row * ldc + col;
                if (p.add) {
                    load_row(v, at, cols - col);
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] += acc[i][j][4 * g + x];
                } else {
#pragma unroll
                    for (int x = 0; x < 4; ++x) v[x] = acc[i][j][4 * g + x];
                }
                store_row(at, v, cols - col);
            }
    }
}

template <class T, class TC, int FORM, bool TAPE, bool DIRECT, int BM, int BN, int WM, int WN>
int32_t launch(Mul p, hipStream_t stream, const char* name) {
    p.tiles_n = (p.n + BN - 1) / BN;
    p.pieces = FORM == WB ? (int64_t)p.ne * ((p.m + BM - 1) / BM) : (p.t + BM - 1) / BM + p.ne + 2;
    const int64_t blocks = (p.pieces * p.tiles_n + 7) / 8 * 8;
    if (blocks > (1 << 23)) return set_error(STADE_HIP_ERANGE, "%s: more than 2^23 tiles", name);
    STADE_TIMED(name, stream, product_kernel<T, TC, FORM, TAPE, DIRECT, BM, BN, WM, WN><<<(unsigned)blocks, 64 * WM * WN, 0, stream>>>(p));
    STADE_LAUNCHED(name);
    return STADE_HIP_OK;
}

// whether all chunks of a matrix are whole and aligned, and a tile's offsets fit 31 bits
inline bool whole(const void* p, int64_t ld, int64_t d, int64_t tile, size_t size) {
    return (uintptr_t)p % 16 == 0 && ld * size % 16 == 0 && d * size % 16 == 0 && tile * ld * (int64_t)size < (1ll << 31);
}

template <class T, class TC, int FORM, bool TAPE>
int32_t run(const Mul& p, hipStream_t stream, const char* name) {
    if constexpr (sizeof(T) == 4) {
        return launch<T, TC, FORM, TAPE, false, 128, 128, 2, 2>(p, stream, name);
    } else {
        const bool direct = (TAPE || whole(p.a, p.lda, FORM == WB ? p.m : p.k, 256, sizeof(T))) &&
                            whole(p.b, p.ldb, FORM == XB ? p.k : p.n, 256, sizeof(T));
        const int64_t big = ((FORM == WB ? (int64_t)p.m * p.ne : p.t + 128 * (int64_t)p.ne) + 255) / 256 * ((p.n + 255) / 256);
        if (big >= 192) {
            if (direct) return launch<T, TC, FORM, TAPE, true, 256, 256, 2, 4>(p, stream, name);
            return launch<T, TC, FORM, TAPE, false, 256, 256, 2, 4>(p, stream, name);
        }
        if (direct) return launch<T, TC, FORM, TAPE, true, 128, 128, 2, 2>(p, stream, name);
        return launch<T, TC, FORM, TAPE, false, 128, 128, 2, 2>(p, stream, name);
    }
}

int32_t check(const char* fn, int64_t tx, const int64_t* start, int64_t i_in, int64_t i_out, int64_t i_t, int64_t i_e) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_extent(fn, "i_in", i_in, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_out", i_out, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (int32_t rc = check_extent(fn, "i_e", i_e, kMostExperts)) return rc;
    return start ? 0 : bad(fn, "start is null");
}

int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

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
    return with_type(tx, [&](auto t) -> int32_t {
        using T = decltype(t);
        if (xb && i_t > 0) {
            p.a = yb; p.lda = ldyb; p.b = w; p.ldb = i_out; p.c = xb; p.ldc = ldxb; p.n = (int)i_in; p.k = (int)i_out;
            if (int32_t rc = run<T, T, XB, false>(p, stream, "expert_mul_xb")) return rc;
        }
        if (wb && i_out > 0 && i_e > 0) {
            p.a = x; p.lda = ldx; p.q = (const uint8_t*)q; p.qs = qs; p.b = yb; p.ldb = ldyb; p.c = wb; p.m = (int)i_in; p.n = (int)i_out;
            const auto go = [&](auto tape) -> int32_t {
                if (twb == STADE_HIP_F32) return run<T, float, WB, decltype(tape)::value>(p, stream, "expert_mul_wb");
                return run<T, T, WB, decltype(tape)::value>(p, stream, "expert_mul_wb");
            };
            return q ? go(std::true_type{}) : go(std::false_type{});
        }
        return STADE_HIP_OK;
    });
}

}  // extern "C"
