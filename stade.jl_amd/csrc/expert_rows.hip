// Tokens sent to several experts each, and back.  A token t has i_k slots, each with an expert's id (0: none); the slots'
// rows lie in the order of the experts, as expert_mul takes them, and place[k, t] says where slot (k, t)'s row is (from 1; 0:
// nowhere).
//
//   expert_order   the slots' stable order by expert, its inverse `place`, and where each expert's rows start
//   expert_take    xs[:, place[k, t]] = x[:, t]                    adjoint: xb[:, t] (+)= sum over k of xsb[:, place[k, t]]
//   expert_join    y[:, t] (+)= sum over k of p[k, t] ys[:, place[k, t]]
//                  adjoint: ysb[:, place[k, t]] (+)= p[k, t] yb[:, t],   pb[k, t] (+)= yb[:, t] . ys[:, place[k, t]]
//
// All go by `place`, token by token: x and yb are read once for all of a token's slots (by the order of the
// experts they would be read i_k times), and sums over slots go in the order of k, with no atomics.
// Bound by HBM: a wave takes 512 columns of one token (the adjoint of the join: a token's whole rows, for the
// dot products), four slots in flight.  Sums are fp32.  8192 tokens of 2048 values, two slots each, bf16: take 20 us (5.0 TB/s), its
// adjoint 30, join 25, its adjoint 35 (4.8 TB/s), the order of 64 experts 11 in two launches.
#include "rows.hpp"

#include <algorithm>

namespace stade {
namespace {

using namespace rows;

constexpr int NT = 256, kCols = 512, kAhead = 4;   // columns a wave takes; slots in flight
constexpr int64_t kMostSlots = 64, kMostExperts = 4096;

int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

// ------------------------------------------------------------------------------------------
// the order, by counting (up to kFewExperts): every block has a stretch of the slots
// ------------------------------------------------------------------------------------------
constexpr int kOrderNT = 512, kOrderWaves = kOrderNT / 64, kStretch = 256 * kOrderWaves;   // slots of a block: four of a lane, wave after wave
constexpr int kFewExperts = 1024, kBinsAThread = 3;
constexpr int64_t kMostCounts = 1 << 16;     // of all blocks, as each block reads them all

struct Order {
    const int64_t* ids;
    int64_t* order; int64_t* place; int64_t* start;
    int e, n, blocks;
    int32_t* counts;     // by block: e + 1 (the last: of no expert)
    int32_t* flag;
};
__device__ __forceinline__ int bin_of(const Order& p, int64_t slot) {
    const int64_t id = p.ids[slot];
    if (id >= 1 && id <= p.e) return (int)(id - 1);
    if (id != 0) *p.flag = kErrIndex;
    return p.e;
}
// a wave's four stretches of 64 slots in their bins, counted
__device__ __forceinline__ void count(const Order& p, int64_t first, int (&bin)[4], int* mine) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int64_t slot = first + 64 * i + lane;
        bin[i] = slot < p.n ? bin_of(p, slot) : -1;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (bin[i] >= 0) atomicAdd(&mine[bin[i]], 1);     // (whole numbers: in any order the same)
}

__global__ __launch_bounds__(kOrderNT) void count_kernel(Order p) {
    __shared__ int bins[kFewExperts + 1];
    for (int i = threadIdx.x; i <= p.e; i += kOrderNT) bins[i] = 0;
    __syncthreads();
    int bin[4];
    count(p, (int64_t)blockIdx.x * kStretch + (threadIdx.x >> 6) * 256, bin, bins);
    __syncthreads();
    for (int i = threadIdx.x; i <= p.e; i += kOrderNT) p.counts[(int64_t)blockIdx.x * (p.e + 1) + i] = bins[i];
}

// A slot's place: those of earlier experts, of its expert in earlier blocks, in earlier waves of the block, and before it in
// its wave (64 slots at a time: the lanes whose bins' bits all agree).
__global__ __launch_bounds__(kOrderNT) void order_kernel(Order p) {
    __shared__ int bins[kOrderWaves][kFewExperts + 1];
    __shared__ int sums[kOrderWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, b0 = threadIdx.x * kBinsAThread;
    for (int i = threadIdx.x; i < kOrderWaves * (kFewExperts + 1); i += kOrderNT) bins[0][i] = 0;
    __syncthreads();
    int bin[4];
    count(p, (int64_t)blockIdx.x * kStretch + wave * 256, bin, bins[wave]);
    __syncthreads();
    // of this thread's bins: all slots, and those in earlier blocks
    int all[kBinsAThread], before[kBinsAThread], total = 0;
#pragma unroll
    for (int i = 0; i < kBinsAThread; ++i) {
        all[i] = before[i] = 0;
        const int b = b0 + i;
        if (b > p.e) continue;
        if (p.blocks > 1) {
#pragma unroll 8
            for (int n = 0; n < p.blocks; ++n) {
                const int c = p.counts[(int64_t)n * (p.e + 1) + b];
                all[i] += c;
                before[i] += n < (int)blockIdx.x ? c : 0;
            }
        } else {
            for (int w = 0; w < kOrderWaves; ++w) all[i] += bins[w][b];
        }
        total += all[i];
    }
    int sum = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
    }
    if (lane == 63) sums[wave] = sum;
    __syncthreads();
    int at = sum - total;
    for (int w = 0; w < wave; ++w) at += sums[w];
#pragma unroll
    for (int i = 0; i < kBinsAThread; ++i) {
        const int b = b0 + i;
        if (b > p.e) continue;
        if (blockIdx.x == 0) p.start[b] = at;          // (start[e]: where those of no expert begin)
        int here = at + before[i];
        for (int w = 0; w < kOrderWaves; ++w) {
            const int c = bins[w][b];
            bins[w][b] = here;
            here += c;
        }
        at += all[i];
    }
    __syncthreads();
    int* mine = bins[wave];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        uint64_t same = __ballot(bin[i] >= 0);
        for (int bit = 0; (p.e >> bit) != 0; ++bit) {
            const uint64_t set = __ballot(bin[i] >= 0 && (bin[i] >> bit & 1));
            same &= bin[i] >> bit & 1 ? set : ~set;
        }
        const int64_t slot = (int64_t)blockIdx.x * kStretch + wave * 256 + 64 * i + lane;
        const int rank = __popcll(same & ((1ull << lane) - 1));
        int first = 0;
        if (bin[i] >= 0) {
            first = mine[bin[i]];
            p.order[first + rank] = slot + 1;
            p.place[slot] = bin[i] < p.e ? first + rank + 1 : 0;
        }
        // (all of the wave's reads come before the writes: it is one wave, and its LDS work goes in order)
        __builtin_amdgcn_wave_barrier();
        if (bin[i] >= 0 && rank == 0) mine[bin[i]] = first + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
}

// the inverse of the order: slots behind the last expert's rows have no place
__global__ __launch_bounds__(NT) void place_kernel(const int64_t* order, const int64_t* start, int64_t e, int64_t n, int64_t* place) {
    const int64_t here = start[e];
    for (int64_t j = (int64_t)blockIdx.x * NT + threadIdx.x; j < n; j += (int64_t)gridDim.x * NT) place[order[j] - 1] = j < here ? j + 1 : 0;
}

struct Moves {
    const void* a; int64_t lda;     // by token
    const void* s; int64_t lds;     // by place
    void* out; int64_t ldo;
    const float* p; float* pb;
    const int64_t* place;
    int d, k;
    int64_t t;
    int32_t* flag;
};

// a slot's row (from 0), or -1
__device__ __forceinline__ int64_t row_of(const Moves& m, int64_t slot) {
    const int64_t at = m.place[slot];
    if (at >= 1 && at <= m.t * m.k) return at - 1;
    if (at != 0) *m.flag = kErrIndex;
    return -1;
}

// A row's last vector is moved back to end with the row: what it shares with the one before is written
// twice, the same.
template <class T>
__global__ __launch_bounds__(NT) void take_kernel(Moves m) {
    typedef typename Pack<T, 8>::loose loose;
    const int lane = threadIdx.x & 63, strips = (m.d + kCols - 1) / kCols;
    const int64_t jobs = m.t * strips, step = (int64_t)gridDim.x * (NT / 64);
    for (int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); j < jobs; j += step) {
        const int64_t t = j / strips;
        int col = (int)(j - t * strips) * kCols + lane * 8;
        if (col >= m.d) continue;
        if (m.d >= 8) {
            col = min(col, m.d - 8);
            const typename Pack<T, 8>::vec v = *(const loose*)((const T*)m.a + t * m.lda + col);
            for (int k = 0; k < m.k; ++k) {
                const int64_t row = row_of(m, t * m.k + k);
                if (row >= 0) *(loose*)((T*)m.out + row * m.ldo + col) = v;
            }
        } else {
            for (int k = 0; k < m.k; ++k) {
                const int64_t row = row_of(m, t * m.k + k);
                if (row >= 0)
                    for (int i = 0; i < m.d; ++i) ((T*)m.out)[row * m.ldo + i] = ((const T*)m.a)[t * m.lda + i];
            }
        }
    }
}

// out[:, t] (+)= sum over k of p[k, t] s[:, place[k, t]]
template <class T, bool ADD>
__global__ __launch_bounds__(NT) void join_kernel(Moves m) {
    const int lane = threadIdx.x & 63, strips = (m.d + kCols - 1) / kCols;
    const int64_t jobs = m.t * strips, step = (int64_t)gridDim.x * (NT / 64);
    for (int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); j < jobs; j += step) {
        const int64_t t = j / strips;
        int col = (int)(j - t * strips) * kCols + lane * 8;
        if (col >= m.d) continue;
        if (!ADD && m.d >= 8) col = min(col, m.d - 8);
        float sum[8];
        T* out = (T*)m.out + t * m.ldo + col;
#pragma unroll
        for (int i = 0; i < 8; ++i) sum[i] = 0.f;
        if (ADD) load_row(sum, out, m.d - col);
        for (int k0 = 0; k0 < m.k; k0 += kAhead) {
            float v[kAhead][8], w[kAhead];
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                const int64_t row = k0 + k < m.k ? row_of(m, t * m.k + k0 + k) : -1;
                w[k] = row >= 0 && m.p ? m.p[t * m.k + k0 + k] : 1.f;
                load_row(v[k], (const T*)m.s + row * m.lds + col, row >= 0 ? m.d - col : 0);   // (no row: zeros)
            }
#pragma unroll
            for (int k = 0; k < kAhead; ++k)
#pragma unroll
                for (int i = 0; i < 8; ++i) sum[i] = fmaf(w[k], v[k][i], sum[i]);
        }
        store_row(out, sum, m.d - col);
    }
}

// out[:, place[k, t]] (+)= p[k, t] a[:, t] and pb[k, t] (+)= a[:, t] . s[:, place[k, t]], four slots a wave
template <class T, bool ADD>
__global__ __launch_bounds__(NT) void join_back_kernel(Moves m) {
    const int lane = threadIdx.x & 63, parts = (m.k + kAhead - 1) / kAhead;
    const int64_t jobs = m.t * parts, step = (int64_t)gridDim.x * (NT / 64);
    for (int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); j < jobs; j += step) {
        const int64_t t = j / parts;
        const int k0 = (int)(j - t * parts) * kAhead;
        int64_t row[kAhead];
        float w[kAhead], dot[kAhead];
#pragma unroll
        for (int k = 0; k < kAhead; ++k) {
            row[k] = k0 + k < m.k ? row_of(m, t * m.k + k0 + k) : -1;
            w[k] = row[k] >= 0 && m.p ? m.p[t * m.k + k0 + k] : 1.f;
            dot[k] = 0.f;
        }
        for (int col = lane * 8; col < m.d; col += kCols) {
            float a[8], v[kAhead][8];
            load_row(a, (const T*)m.a + t * m.lda + col, m.d - col);
            if (m.pb) {
#pragma unroll
                for (int k = 0; k < kAhead; ++k) load_row(v[k], (const T*)m.s + row[k] * m.lds + col, row[k] >= 0 ? m.d - col : 0);
#pragma unroll
                for (int k = 0; k < kAhead; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) dot[k] = fmaf(a[i], v[k][i], dot[k]);
            }
            if (m.out) {
#pragma unroll
                for (int k = 0; k < kAhead; ++k) {
                    if (row[k] < 0) continue;
                    T* out = (T*)m.out + row[k] * m.ldo + col;
                    float o[8];
                    if (ADD) load_row(o, out, m.d - col);
#pragma unroll
                    for (int i = 0; i < 8; ++i) o[i] = ADD ? fmaf(w[k], a[i], o[i]) : w[k] * a[i];
                    store_row(out, o, m.d - col);
                }
            }
        }
        if (m.pb) {
#pragma unroll
            for (int k = 0; k < kAhead; ++k) {
                dot[k] = wave_sum(dot[k]);
                if (row[k] < 0) dot[k] = 0.f;     // (also where `a` is not finite)
                float* pb = m.pb + t * m.k + k0 + k;
                if (lane == 0 && k0 + k < m.k) *pb = ADD ? *pb + dot[k] : dot[k];
            }
        }
    }
}

unsigned grid_of(int64_t jobs) { return (unsigned)std::min<int64_t>((jobs + NT / 64 - 1) / (NT / 64), 1 << 16); }

int32_t check(const char* fn, int64_t tx, int64_t i_d, int64_t i_k, int64_t i_t) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_k", i_k, kMostSlots)) return rc;
    return check_extent(fn, "i_t", i_t, kMostRows);
}

int32_t join(const char* fn, const char* what, int64_t tx, Moves m, int64_t i_d, int64_t add, hipStream_t stream) {
    if (i_d == 0 || m.t == 0 || (m.k == 0 && add)) return STADE_HIP_OK;
    if (!m.out || (m.k > 0 && (!m.s || !m.place))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    m.flag = error_flag(call.ws);
    const unsigned grid = grid_of(m.t * ((i_d + kCols - 1) / kCols));
    return with_type(tx, [&](auto t) -> int32_t {
        using T = decltype(t);
        STADE_TIMED(what, stream, {
            if (add) join_kernel<T, true><<<grid, NT, 0, stream>>>(m);
            else join_kernel<T, false><<<grid, NT, 0, stream>>>(m);
        });
        STADE_LAUNCHED("expert_rows join_kernel");
        return STADE_HIP_OK;
    });
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_expert_order(const int64_t* ids, int64_t* order, int64_t* place, int64_t* start, int64_t i_k, int64_t i_e, int64_t i_t,
                               hipStream_t stream) {
    const char* fn = "stade_hip_expert_order";
    if (int32_t rc = check_extent(fn, "i_k", i_k, kMostSlots)) return rc;
    if (int32_t rc = check_extent(fn, "i_e", i_e, kMostExperts)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    const int64_t n = i_k * i_t;
    if (int32_t rc = check_extent(fn, "i_k * i_t", n, kMostRows)) return rc;
    if (!start || (n > 0 && (!ids || !order || !place))) return bad(fn, "null pointer");
    const int64_t blocks = (n + kStretch - 1) / kStretch;
    if (n > 0) {
        WsCall call(stream);
        if (!call.ok()) return call.error();
        // (taken by every call, so that each smaller one is captured after an eager one)
        int32_t* counts = (int32_t*)scratch(kMostCounts * sizeof(int32_t));
        if (!counts) return scratch_error();
        // Few experts: by counting, a launch or two (16384 slots of 64 experts: 11 us, by sorting 28).
        if (i_e <= kFewExperts && blocks * (i_e + 1) <= kMostCounts) {
            const Order p{ids, order, place, start, (int)i_e, (int)n, (int)blocks, counts, error_flag(call.ws)};
            if (blocks > 1) {
                STADE_TIMED("expert_count", stream, count_kernel<<<(unsigned)blocks, kOrderNT, 0, stream>>>(p));
                STADE_LAUNCHED("expert_rows count_kernel");
            }
            STADE_TIMED("expert_order", stream, order_kernel<<<(unsigned)blocks, kOrderNT, 0, stream>>>(p));
            STADE_LAUNCHED("expert_rows order_kernel");
            return STADE_HIP_OK;
        }
    }
    if (int32_t rc = stade_hip_token_order(ids, order, start, i_e, n, stream)) return rc;
    if (n == 0) return STADE_HIP_OK;
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    STADE_TIMED("expert_place", stream,
                place_kernel<<<(unsigned)std::min<int64_t>((n + NT - 1) / NT, 1 << 16), NT, 0, stream>>>(order, start, i_e, n, place));
    STADE_LAUNCHED("expert_rows place_kernel");
    return STADE_HIP_OK;
}

int32_t stade_hip_expert_take(int64_t tx, void* xs, int64_t ldxs, const void* x, int64_t ldx, const int64_t* place, int64_t i_d, int64_t i_k,
                              int64_t i_t, hipStream_t stream) {
    const char* fn = "stade_hip_expert_take";
    if (int32_t rc = check(fn, tx, i_d, i_k, i_t)) return rc;
    if (int32_t rc = check_ld(fn, "ldxs", ldxs, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldx", ldx, i_d)) return rc;
    if (i_d == 0 || i_k == 0 || i_t == 0) return STADE_HIP_OK;
    if (!xs || !x || !place) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    const Moves m{x, ldx, nullptr, 0, xs, ldxs, nullptr, nullptr, place, (int)i_d, (int)i_k, i_t, error_flag(call.ws)};
    const unsigned grid = grid_of(i_t * ((i_d + kCols - 1) / kCols));
    return with_type(tx, [&](auto t) -> int32_t {
        STADE_TIMED("expert_take", stream, take_kernel<decltype(t)><<<grid, NT, 0, stream>>>(m));
        STADE_LAUNCHED("expert_rows take_kernel");
        return STADE_HIP_OK;
    });
}

int32_t stade_hip_expert_take_b(int64_t tx, const void* xsb, int64_t ldxsb, void* xb, int64_t ldxb, const int64_t* place, int64_t i_d,
                                int64_t i_k, int64_t i_t, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_expert_take_b";
    if (int32_t rc = check(fn, tx, i_d, i_k, i_t)) return rc;
    if (int32_t rc = check_ld(fn, "ldxsb", ldxsb, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldxb", ldxb, i_d)) return rc;
    return join(fn, "expert_take_b", tx, Moves{nullptr, 0, xsb, ldxsb, xb, ldxb, nullptr, nullptr, place, (int)i_d, (int)i_k, i_t}, i_d, add, stream);
}

int32_t stade_hip_expert_join(int64_t tx, void* y, int64_t ldy, const void* ys, int64_t ldys, const float* p, const int64_t* place, int64_t i_d,
                              int64_t i_k, int64_t i_t, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_expert_join";
    if (int32_t rc = check(fn, tx, i_d, i_k, i_t)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldys", ldys, i_d)) return rc;
    return join(fn, "expert_join", tx, Moves{nullptr, 0, ys, ldys, y, ldy, p, nullptr, place, (int)i_d, (int)i_k, i_t}, i_d, add, stream);
}

int32_t stade_hip_expert_join_b(int64_t tx, const void* yb, int64_t ldyb, const void* ys, int64_t ldys, void* ysb, int64_t ldysb, const float* p,
                                float* pb, const int64_t* place, int64_t i_d, int64_t i_k, int64_t i_t, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_expert_join_b";
    if (int32_t rc = check(fn, tx, i_d, i_k, i_t)) return rc;
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_d)) return rc;
    if (pb)
        if (int32_t rc = check_ld(fn, "ldys", ldys, i_d)) return rc;
    if (ysb)
        if (int32_t rc = check_ld(fn, "ldysb", ldysb, i_d)) return rc;
    if (i_k == 0 || i_t == 0 || (!ysb && !pb)) return STADE_HIP_OK;
    if (i_d == 0 && (!pb || add)) return STADE_HIP_OK;
    if (!place || (i_d > 0 && (!yb || (pb && !ys)))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    const Moves m{yb, ldyb, ys, ldys, ysb, ldysb, p, pb, place, (int)i_d, (int)i_k, i_t, error_flag(call.ws)};
    const unsigned grid = grid_of(i_t * ((i_k + kAhead - 1) / kAhead));
    return with_type(tx, [&](auto t) -> int32_t {
        using T = decltype(t);
        STADE_TIMED("expert_join_b", stream, {
            if (add) join_back_kernel<T, true><<<grid, NT, 0, stream>>>(m);
            else join_back_kernel<T, false><<<grid, NT, 0, stream>>>(m);
        });
        STADE_LAUNCHED("expert_rows join_back_kernel");
        return STADE_HIP_OK;
    });
}

}  // extern "C"
