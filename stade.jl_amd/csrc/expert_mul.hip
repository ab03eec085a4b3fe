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
// the simple form: 64 x 64 of the result a block, 4 x 4 a thread, fp32 FMAs, any type and size
// ------------------------------------------------------------------------------------------
struct Mul {
    const void* a; int64_t lda;    // rows
    const void* b; int64_t ldb;    // w, or yb for wb
    void* c; int64_t ldc;
    const uint8_t* q; const uint8_t* qs;   // the rows' tape in place of a (wb)
    const int64_t* start;
    int ne;
    int64_t t;
    int m, n, k;     // of one expert's product (m or k: its rows)
    int add;
    int32_t* flag;
};

constexpr int NT = 256, TM = 64, TN = 64, TK = 16;
enum Form { Y = 0, XB = 1, WB = 2 };

template <class T, class TC, int FORM, bool TAPE>
__global__ __launch_bounds__(NT) void simple_kernel(Mul p) {
    __shared__ float as[TK][TM + 4], bs[TK][TN + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    Rows r;
    int64_t m0;
    if constexpr (FORM == WB) {
        const int mt = (p.m + TM - 1) / TM;
        r = expert_rows(p.start, p.ne, p.t, blockIdx.y / mt, p.flag);
        m0 = (int64_t)(blockIdx.y % mt) * TM;
    } else {
        r = find_rows<TM>(p.start, p.ne, p.t, blockIdx.y, p.flag);
        m0 = 0;
    }
    if (r.e == -2) return;
    const int n0 = blockIdx.x * TN, m = FORM == WB ? p.m : r.rows, k = FORM == WB ? r.rows : r.e < 0 ? 0 : p.k;
    if (r.e < 0 && p.add) return;
    const T* a = (const T*)p.a + (FORM == WB ? r.row * p.lda : r.row * p.lda);
    const T* b = (const T*)p.b + (FORM == WB ? r.row * p.ldb : (int64_t)max(r.e, 0) * (FORM == Y ? (int64_t)p.k * p.n : (int64_t)p.k * p.n));
    TC* c = (TC*)p.c + (FORM == WB ? (int64_t)r.e * p.m * p.n : r.row * p.ldc);
    float acc[4][4] = {};
    for (int k0 = 0; k0 < k; k0 += TK) {
        for (int i = threadIdx.x; i < TK * TM; i += NT) {
            const int kk = FORM == WB ? i / TM : i % TK, mm = FORM == WB ? i % TM : i / TK;
            float v = 0.f;
            if (k0 + kk < k && m0 + mm < m) {
                if constexpr (FORM == WB) {
                    if constexpr (TAPE) {
                        const int64_t ng = tape8::groups(p.m), row = r.row + k0 + kk;
                        const int64_t col = m0 + mm;
                        v = (float)(int)(int8_t)p.q[row * ng * 32 + col] * tape8::unit(p.qs[row * ng + col / 32]);
                    } else {
                        v = (float)a[(int64_t)(k0 + kk) * p.lda + m0 + mm];
                    }
                } else {
                    v = (float)a[(int64_t)mm * p.lda + k0 + kk];
                }
            }
            as[kk][mm] = v;
        }
        for (int i = threadIdx.x; i < TK * TN; i += NT) {
            const int kk = FORM == XB ? i % TK : i / TN, nn = FORM == XB ? i / TK : i % TN;
            float v = 0.f;
            if (k0 + kk < k && n0 + nn < p.n)
                v = (float)(FORM == XB ? b[(int64_t)(n0 + nn) * p.ldb + k0 + kk] : b[(int64_t)(k0 + kk) * p.ldb + n0 + nn]);
            bs[kk][nn] = v;
        }
        __syncthreads();
#pragma unroll
        for (int kk = 0; kk < TK; ++kk) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(as[kk][ty * 4 + i], bs[kk][tx * 4 + j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t mm = m0 + ty * 4 + i;
            const int nn = n0 + tx * 4 + j;
            if (mm < m && nn < p.n) {
                TC* at = c + mm * (FORM == WB ? (int64_t)p.n : p.ldc) + nn;
                *at = (TC)(p.add ? (float)*at + acc[i][j] : acc[i][j]);
            }
        }
}

template <class T, class TC, int FORM, bool TAPE>
int32_t run(const Mul& p, hipStream_t stream, const char* name) {
    const int64_t pieces = FORM == WB ? (int64_t)p.ne * ((p.m + TM - 1) / TM) : (p.t + TM - 1) / TM + p.ne + 2;
    // (grid y is limited to 65535: the rest in further launches would need an offset)
    if (pieces > 65535) return set_error(STADE_HIP_ERANGE, "%s: more than 65535 row tiles", name);
    const dim3 grid((unsigned)((p.n + TN - 1) / TN), (unsigned)pieces);
    STADE_TIMED(name, stream, simple_kernel<T, TC, FORM, TAPE><<<grid, NT, 0, stream>>>(p));
    STADE_LAUNCHED(name);
    return STADE_HIP_OK;
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
