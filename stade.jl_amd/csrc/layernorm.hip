// layernorm and its adjoint, row by row: with mu = mean(x), rs = 1 / sqrt(var(x) + eps) and
// xh = (x - mu) rs,
//   y  = xh g + b
//   a  = yb g,   xb (+)= rs (a - mean(a) - xh mean(a xh))
//   gb (+)= sum over the rows of yb xh,   bb (+)= sum over the rows of yb
// mu and rs go from the forward to the reverse sweep in fp32; the input goes as itself or as its
// 8-bit tape (tape8.hpp), which the forward sweep writes from the registers that hold the row.
//
// Bound by HBM: each row is read once and stays in registers (WPR waves a row, NV vectors of VE
// values a thread), so the variance is summed from the differences to the mean with no second read.
// The reverse sweep's blocks walk over the rows with gb and bb of their columns in registers;
// each block leaves one row of partial sums, which a second launch adds in a fixed order: no
// atomics, the same bits at every call.  Sums are fp32 throughout.
// Rows longer than the registers hold are read again for each of the sums.
//
// Measured on an MI355X (16384 x 4096 bf16, calls one after the other: arrays of 134 MB stay in the last-level cache in
// part; copy 4.7 TB/s): forward 45 us (6.0 TB/s), with the tape 69 (4.9); reverse 79 us (5.1 TB/s), from the tape 71 (4.7;
// the bytes turn into values by one conversion, one subtraction and one product each).  In the reverse sweep the next
// row, its statistics and the weights are in registers before the row's sums are waited for: without them 152 us.
// Longer rows are slower: 4096 x 12288 bf16 forward 50 us (4.0 TB/s), reverse 77 (3.9), from the tape 67 (3.8), fp32 147
// (4.1; in fp32 and from the tape the registers do not hold two rows' values and the sums, and some go through scratch
// memory, as from 16385 columns on in the forward sweep with the tape); 4096 x 24576 reverse 430 us (1.4 TB/s: read
// twice, and each block adds to its partial sums in memory).
#include "tape8.hpp"

#include <algorithm>
#include <type_traits>

namespace stade {
namespace {

using namespace rows;

struct Fwd {
    void* y; int64_t ldy;
    const void* x; int64_t ldx;
    const void* g; const void* b;
    float* mu; float* rs;
    uint8_t* q; uint8_t* qs;
    int d; int64_t n; float eps;
};
struct Bwd {
    const void* yb; int64_t ldyb;
    const void* x; int64_t ldx;
    const uint8_t* q; const uint8_t* qs;
    void* xb; int64_t ldxb;
    const void* g; const float* mu; const float* rs;
    float* part;      // partial sums: (gb, bb) of a block, 2 * d values; null without gb and bb,
    float* gb; float* bb;   // or, for a launch of one block, the weights' shadows themselves (each may be null)
    int d; int64_t n; int add;
};

// the sums of NS values over the WPR waves of a row, in every thread.  `lds`: 2 * 16 * NS floats,
// used in turns (`turn`), so that one barrier a call will do.
template <int WPR, int NS>
__device__ __forceinline__ void row_sum(float (&v)[NS], float* lds, int& turn) {
#pragma unroll
    for (int k = 0; k < NS; ++k) v[k] = wave_sum(v[k]);
    if constexpr (WPR > 1) {
        const int wave = threadIdx.x >> 6;
        float* at = lds + turn * 16 * NS;
        turn ^= 1;
        if ((threadIdx.x & 63) == 0) {
#pragma unroll
            for (int k = 0; k < NS; ++k) at[wave * NS + k] = v[k];
        }
        __syncthreads();
        const int first = wave / WPR * WPR;
#pragma unroll
        for (int k = 0; k < NS; ++k) {
            float s = at[first * NS + k];
#pragma unroll
            for (int w = 1; w < WPR; ++w) s += at[(first + w) * NS + k];
            v[k] = s;
        }
    }
}

template <int WPR> constexpr int block_of() { return WPR > 4 ? 64 * WPR : 256; }

template <class T, class G, int VE, int NV, int WPR, bool TAPE, bool W>
__global__ __launch_bounds__(block_of<WPR>()) void forward_kernel(Fwd p) {
    constexpr int NT = block_of<WPR>(), RPB = NT / (64 * WPR), STEP = 64 * WPR * VE;
    __shared__ float lds[2 * 16];
    int turn = 0;
    const int sub = threadIdx.x / (64 * WPR), tr = threadIdx.x % (64 * WPR), d = p.d;
    const int64_t trips = (p.n + RPB - 1) / RPB;
    for (int64_t trip = blockIdx.x; trip < trips; trip += gridDim.x) {
        const int64_t row = trip * RPB + sub;
        const bool here = row < p.n;   // (the others run along for the barriers)
        const T* x = (const T*)p.x + row * p.ldx;
        float v[NV][VE], s[1] = {0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) load_row<W>(v[k], x + k * STEP + tr * VE, here ? d - (k * STEP + tr * VE) : 0);
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) s[0] += v[k][i];
        row_sum<WPR, 1>(s, lds, turn);
        const float mu = s[0] / (float)d;
        s[0] = 0.f;
#pragma unroll
        for (int k = 0; k < NV; ++k)
#pragma unroll
            for (int i = 0; i < VE; ++i) {
                const float c = k * STEP + tr * VE + (W ? 0 : i) < d ? v[k][i] - mu : 0.f;
                s[0] = fmaf(c, c, s[0]);
            }
        row_sum<WPR, 1>(s, lds, turn);
        const float rs = 1.0f / sqrtf(s[0] / (float)d + p.eps);
        if (!here) continue;
        if (tr == 0) {
            if (p.mu) p.mu[row] = mu;
            if (p.rs) p.rs[row] = rs;
        }
        if constexpr (TAPE) {
            const int64_t ng = tape8::groups(d);
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int col = k * STEP + tr * VE;
                tape8::store_part<T>(p.q + row * ng * tape8::kGroup, p.qs + row * ng, v[k], col, ng);
            }
        }
        T* y = (T*)p.y + row * p.ldy;
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int col = k * STEP + tr * VE;
            if (col < d) {
                float g[VE], b[VE];
                if (p.g) load_row<W>(g, (const G*)p.g + col, d - col);
                if (p.b) load_row<W>(b, (const G*)p.b + col, d - col);
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float h = (v[k][i] - mu) * rs;
                    v[k][i] = fmaf(h, p.g ? g[i] : 1.f, p.b ? b[i] : 0.f);
                }
                store_row<W>(y + col, v[k], d - col);
            }
        }
    }
}

// the row's values that the reverse sweep works on
template <class T, int VE, bool TAPE>
__device__ __forceinline__ void load_input(float (&v)[VE], const Bwd& p, int64_t row, int col) {
    if constexpr (TAPE) {
        const int64_t ng = tape8::groups(p.d);
        if (col < p.d)
            tape8::values(v, p.q + row * ng * tape8::kGroup + col, tape8::unit(p.qs[row * ng + col / tape8::kGroup]));
    } else {
        load_row(v, (const T*)p.x + row * p.ldx + col, p.d - col);
    }
}

// a thread's values of a row as they come from memory, so that the next row's can be on their way
// while this one's are worked on
template <class T, int VE, bool TAPE, bool W>
struct Raw {
    typedef T vec __attribute__((ext_vector_type(VE)));
    std::conditional_t<TAPE, tape8::Word<VE>, vec> x;
    vec yb;
    uint8_t s;

    __device__ __forceinline__ void load(const Bwd& p, int64_t row, int col) {
        const int left = row < p.n ? p.d - col : 0;
        if constexpr (TAPE) {
            const int64_t ng = tape8::groups(p.d);
            if (left > 0) {   // (the tape's rows are whole groups)
                x = *reinterpret_cast<const tape8::Word<VE>*>(p.q + row * ng * tape8::kGroup + col);
                s = p.qs[row * ng + col / tape8::kGroup];
            }
        } else {
            get(x, (const T*)p.x + row * p.ldx + col, left);
        }
        get(yb, (const T*)p.yb + row * p.ldyb + col, left);
    }
    static __device__ __forceinline__ void get(vec& v, const T* at, int left) {
        if (W ? left > 0 : left >= VE) {
            v = *reinterpret_cast<const typename Pack<T, VE>::loose*>(at);
        } else if constexpr (!W) {
#pragma unroll
            for (int i = 0; i < VE; ++i) v[i] = i < left ? at[i] : (T)0.f;
        }
    }
    __device__ __forceinline__ void values(float (&h)[VE], float (&a)[VE]) const {
        if constexpr (TAPE) {
            tape8::values(h, x, tape8::unit(s));
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) h[i] = (float)x[i];
        }
#pragma unroll
        for (int i = 0; i < VE; ++i) a[i] = (float)yb[i];
    }
};

template <class T, class G, int VE, int NV, int WPR, int NT, bool TAPE, bool W>
__global__ __launch_bounds__(NT) void backward_kernel(Bwd p) {
    constexpr int RPB = NT / (64 * WPR), STEP = 64 * WPR * VE;
    __shared__ float lds[2 * 16 * 2];
    __shared__ float sums[RPB > 1 ? 2 * NV * STEP : 1];
    int turn = 0;
    const int sub = threadIdx.x / (64 * WPR), tr = threadIdx.x % (64 * WPR), d = p.d;
    float ag[NV][VE], ab[NV][VE], g[NV][VE];
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        if (p.g) load_row<W>(g[k], (const G*)p.g + k * STEP + tr * VE, d - (k * STEP + tr * VE));
#pragma unroll
        for (int i = 0; i < VE; ++i) {
            ag[k][i] = ab[k][i] = 0.f;
            if (!p.g) g[k][i] = 1.f;
        }
    }
    const int64_t trips = (p.n + RPB - 1) / RPB;
    Raw<T, VE, TAPE, W> raw[NV];
    int64_t row = (int64_t)blockIdx.x * RPB + sub;
    float mu = row < p.n ? p.mu[row] : 0.f, rs = row < p.n ? p.rs[row] : 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) raw[k].load(p, row, k * STEP + tr * VE);
    for (int64_t trip = blockIdx.x; trip < trips; trip += gridDim.x) {
        const bool here = row < p.n;   // (the others run along for the barriers)
        const int64_t next = row + (int64_t)gridDim.x * RPB;
        const float m = mu, r = rs;
        float h[NV][VE], a[NV][VE], s[2] = {0.f, 0.f};
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            raw[k].values(h[k], a[k]);
            raw[k].load(p, next, k * STEP + tr * VE);
        }
        if (next < p.n) {
            mu = p.mu[next];
            rs = p.rs[next];
        }
#pragma unroll
        for (int k = 0; k < NV; ++k) {
            const int col = k * STEP + tr * VE;
            if (here && col < d) {
#pragma unroll
                for (int i = 0; i < VE; ++i) {
                    const float xh = W || col + i < d ? (h[k][i] - m) * r : 0.f, yb = a[k][i];
                    ag[k][i] = fmaf(yb, xh, ag[k][i]);
                    ab[k][i] += yb;
                    h[k][i] = xh;
                    a[k][i] = yb * g[k][i];
                    s[0] += a[k][i];
                    s[1] = fmaf(a[k][i], xh, s[1]);
                }
            }
        }
        row_sum<WPR, 2>(s, lds, turn);
        if (here && p.xb) {
            const float m0 = s[0] / (float)d, m1 = s[1] / (float)d;
            T* xb = (T*)p.xb + row * p.ldxb;
#pragma unroll
            for (int k = 0; k < NV; ++k) {
                const int col = k * STEP + tr * VE;
                if (col < d) {
                    float o[VE];
                    if (p.add) load_row<W>(o, xb + col, d - col);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const float v = r * fmaf(-h[k][i], m1, a[k][i] - m0);
                        a[k][i] = p.add ? o[i] + v : v;
                    }
                    store_row<W>(xb + col, a[k], d - col);
                }
            }
        }
        row = next;
    }
    if (!p.part && !p.gb && !p.bb) return;
    // the block's rows of partial sums joined, one after the other
    if constexpr (RPB > 1) {
        for (int r = 1; r < RPB; ++r) {
            __syncthreads();
            if (sub == r) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        sums[k * STEP + tr * VE + i] = ag[k][i];
                        sums[NV * STEP + k * STEP + tr * VE + i] = ab[k][i];
                    }
            }
            __syncthreads();
            if (sub == 0) {
#pragma unroll
                for (int k = 0; k < NV; ++k)
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        ag[k][i] += sums[k * STEP + tr * VE + i];
                        ab[k][i] += sums[NV * STEP + k * STEP + tr * VE + i];
                    }
            }
        }
        if (sub != 0) return;
    }
    float* part = p.part + (int64_t)blockIdx.x * 2 * d;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
        const int col = k * STEP + tr * VE;
        if (col < d) {
            if (p.part) {
                store_row(part + col, ag[k], d - col);
                store_row(part + d + col, ab[k], d - col);
            } else {
                float o[VE];
                if (p.gb) {
                    load_row(o, p.gb + col, p.add ? d - col : 0);
#pragma unroll
                    for (int i = 0; i < VE; ++i) o[i] += ag[k][i];
                    store_row(p.gb + col, o, d - col);
                }
                if (p.bb) {
                    load_row(o, p.bb + col, p.add ? d - col : 0);
#pragma unroll
                    for (int i = 0; i < VE; ++i) o[i] += ab[k][i];
                    store_row(p.bb + col, o, d - col);
                }
            }
        }
    }
}

// Rows too long for the registers: one block a row, the row read again for each of its sums.
constexpr int kLongNT = 1024;
template <class T, class G, bool TAPE>
__global__ __launch_bounds__(kLongNT) void forward_long_kernel(Fwd p) {
    __shared__ float lds[2 * 16];
    int turn = 0;
    const int d = p.d;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const T* x = (const T*)p.x + row * p.ldx;
        float v[8], s[1] = {0.f};
        for (int col = threadIdx.x * 8; col < d; col += kLongNT * 8) {
            load_row(v, x + col, d - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) s[0] += v[i];
        }
        row_sum<16, 1>(s, lds, turn);
        const float mu = s[0] / (float)d;
        s[0] = 0.f;
        for (int col = threadIdx.x * 8; col < d; col += kLongNT * 8) {
            load_row(v, x + col, d - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float c = col + i < d ? v[i] - mu : 0.f;
                s[0] = fmaf(c, c, s[0]);
            }
        }
        row_sum<16, 1>(s, lds, turn);
        const float rs = 1.0f / sqrtf(s[0] / (float)d + p.eps);
        if (threadIdx.x == 0) {
            if (p.mu) p.mu[row] = mu;
            if (p.rs) p.rs[row] = rs;
        }
        const int64_t ng = tape8::groups(d);
        for (int col = threadIdx.x * 8; col < ng * tape8::kGroup; col += kLongNT * 8) {
            load_row(v, x + col, d - col);
            if constexpr (TAPE) {
                tape8::store_part<T>(p.q + row * ng * tape8::kGroup, p.qs + row * ng, v, col, ng);
            }
            if (col < d) {
                float g[8], b[8];
                if (p.g) load_row(g, (const G*)p.g + col, d - col);
                if (p.b) load_row(b, (const G*)p.b + col, d - col);
#pragma unroll
                for (int i = 0; i < 8; ++i) v[i] = fmaf((v[i] - mu) * rs, p.g ? g[i] : 1.f, p.b ? b[i] : 0.f);
                store_row((T*)p.y + row * p.ldy + col, v, d - col);
            }
        }
    }
}

template <class T, class G, bool TAPE>
__global__ __launch_bounds__(kLongNT) void backward_long_kernel(Bwd p) {
    __shared__ float lds[2 * 16 * 2];
    int turn = 0;
    const int d = p.d;
    float* part = p.part ? p.part + (int64_t)blockIdx.x * 2 * d : nullptr;
    bool first = true;
    for (int64_t row = blockIdx.x; row < p.n; row += gridDim.x) {
        const float mu = p.mu[row], rs = p.rs[row];
        const T* yb = (const T*)p.yb + row * p.ldyb;
        float h[8], a[8], g[8], s[2] = {0.f, 0.f};
        for (int col = threadIdx.x * 8; col < d; col += kLongNT * 8) {
            load_input<T, 8, TAPE>(h, p, row, col);
            load_row(a, yb + col, d - col);
            if (p.g) load_row(g, (const G*)p.g + col, d - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float xh = col + i < d ? (h[i] - mu) * rs : 0.f, w = p.g ? a[i] * g[i] : a[i];
                s[0] += w;
                s[1] += w * xh;
                h[i] = a[i] * xh;
            }
            if (part) {   // (each thread its own columns of the block's partial sums)
                float o[8];
                if (!first) {
                    load_row(o, part + col, d - col);
#pragma unroll
                    for (int i = 0; i < 8; ++i) h[i] += o[i];
                    load_row(o, part + d + col, d - col);
#pragma unroll
                    for (int i = 0; i < 8; ++i) a[i] += o[i];
                }
                store_row(part + col, h, d - col);
                store_row(part + d + col, a, d - col);
            }
        }
        first = false;
        row_sum<16, 2>(s, lds, turn);
        if (!p.xb) continue;
        const float m0 = s[0] / (float)d, m1 = s[1] / (float)d;
        T* xb = (T*)p.xb + row * p.ldxb;
        for (int col = threadIdx.x * 8; col < d; col += kLongNT * 8) {
            load_input<T, 8, TAPE>(h, p, row, col);
            load_row(a, yb + col, d - col);
            if (p.g) load_row(g, (const G*)p.g + col, d - col);
            float o[8];
            if (p.add) load_row(o, xb + col, d - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float r = rs * ((p.g ? a[i] * g[i] : a[i]) - m0 - (h[i] - mu) * rs * m1);
                a[i] = p.add ? o[i] + r : r;
            }
            store_row(xb + col, a, d - col);
        }
    }
}

// gb and bb from the blocks' partial sums: 32 columns a block, 32 threads a column, each over its
// share of the partial rows in order, then the 32 in order.
constexpr int kSumNT = 1024;
__global__ __launch_bounds__(kSumNT) void weight_sum_kernel(const float* part, int nparts, int d, float* gb, float* bb, int add) {
    __shared__ float lds[32][33];
    const int c = threadIdx.x & 31, r = threadIdx.x >> 5, col = blockIdx.x * 32 + c;
    float* out = blockIdx.y ? bb : gb;
    const float* p = part + (blockIdx.y ? d : 0) + col;
    float s = 0.f;
    if (col < d) {
        const int each = (nparts + 31) / 32, end = min(nparts, (r + 1) * each);
#pragma unroll 16
        for (int b = r * each; b < end; ++b) s += p[(int64_t)b * 2 * d];
    }
    lds[r][c] = s;
    __syncthreads();
    if (r == 0 && col < d && out) {
#pragma unroll
        for (int k = 1; k < 32; ++k) s += lds[k][c];
        out[col] = add ? out[col] + s : s;
    }
}

constexpr int kOneBlock = 4;        // trips of one block in the reverse sweep that spare a second launch
constexpr int kMostHeldBack = 16384;   // the longest row that the reverse sweep holds in registers
constexpr int kSumParts = 512;      // blocks of the reverse sweep at most: two a CU

template <class T, class G, int VE, int NV, int WPR, bool TAPE>
void start(const Fwd& p, hipStream_t stream) {
    constexpr int NT = block_of<WPR>(), RPB = NT / (64 * WPR);
    const unsigned grid = (unsigned)std::min<int64_t>((p.n + RPB - 1) / RPB, 1 << 16);
    if (p.d % VE == 0) forward_kernel<T, G, VE, NV, WPR, TAPE, true><<<grid, NT, 0, stream>>>(p);
    else forward_kernel<T, G, VE, NV, WPR, TAPE, false><<<grid, NT, 0, stream>>>(p);
}
template <class T, class G, int VE, int NV, int WPR, int NT, bool TAPE>
void start(const Bwd& p, unsigned grid, hipStream_t stream) {
    if (p.d % VE == 0) backward_kernel<T, G, VE, NV, WPR, NT, TAPE, true><<<grid, NT, 0, stream>>>(p);
    else backward_kernel<T, G, VE, NV, WPR, NT, TAPE, false><<<grid, NT, 0, stream>>>(p);
}

// The form by the row's length.  Forward: a wave a row up to 1024, then the waves that hold it in at most 4 vectors a
// thread.  Other splits come close (bf16, and with the tape): 16384 x 2048 four waves of one vector 26.4 us (29.5), one
// wave of four 24.5 (28.1); 16384 x 4096 two waves of four 43.3 (66.9), four of two 42.4 (65.0); 4096 x 12288 sixteen waves of
// two 50.4 (62.4), eight of four 36.2 (63.0).
template <class T, class G, bool TAPE>
void launch(const Fwd& p, hipStream_t s) {
    const int d = p.d;
    if (d <= 128) start<T, G, 2, 1, 1, TAPE>(p, s);
    else if (d <= 512) start<T, G, 8, 1, 1, TAPE>(p, s);
    else if (d <= 1024) start<T, G, 8, 2, 1, TAPE>(p, s);
    else if (d <= 2048) start<T, G, 8, 1, 4, TAPE>(p, s);
    else if (d <= 4096) start<T, G, 8, 4, 2, TAPE>(p, s);
    else if (d <= 8192) start<T, G, 8, 4, 4, TAPE>(p, s);
    else if (d <= 16384) start<T, G, 8, 2, 16, TAPE>(p, s);
    else if (d <= 32768) start<T, G, 8, 4, 16, TAPE>(p, s);
    else forward_long_kernel<T, G, TAPE><<<(unsigned)std::min<int64_t>(p.n, 1 << 16), kLongNT, 0, s>>>(p);
}
// Reverse: one vector a thread up to 8192, so that two rows' values, their sums and the weights leave
// room for 16 waves a CU.
constexpr int back_rows(int64_t d) { return d <= 512 ? 8 : d <= 1024 ? 4 : d <= 2048 ? 2 : 1; }   // rows a block works on at a time
template <class T, class G, bool TAPE>
void launch(const Bwd& p, unsigned grid, hipStream_t s) {
    const int d = p.d;
    if (d <= 128) start<T, G, 2, 1, 1, 512, TAPE>(p, grid, s);
    else if (d <= 512) start<T, G, 8, 1, 1, 512, TAPE>(p, grid, s);
    else if (d <= 1024) start<T, G, 8, 1, 2, 512, TAPE>(p, grid, s);
    else if (d <= 2048) start<T, G, 8, 1, 4, 512, TAPE>(p, grid, s);
    else if (d <= 4096) start<T, G, 8, 1, 8, 512, TAPE>(p, grid, s);
    else if (d <= 8192) start<T, G, 8, 1, 16, 1024, TAPE>(p, grid, s);
    else if (d <= kMostHeldBack) start<T, G, 8, 4, 8, 512, TAPE>(p, grid, s);
    else backward_long_kernel<T, G, TAPE><<<grid, kLongNT, 0, s>>>(p);
}

// f(T{}, G{}): the rows' type, and the weights': fp32 or the rows' own
template <class F>
int32_t with_types(int64_t tx, int64_t tg, F&& f) {
    return with_type(tx, [&](auto t) -> int32_t {
        if (tg == STADE_HIP_F32) return f(t, float{});
        return f(t, t);
    });
}

int32_t check(const char* fn, int64_t tx, int64_t tg, int64_t i_d, int64_t i_n) {
    if (int32_t rc = check_type(fn, "x", tx)) return rc;
    if (int32_t rc = check_type(fn, "g", tg)) return rc;
    if (tg != STADE_HIP_F32 && tg != tx) return bad(fn, "g is neither Float32 nor of x's type");
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostCols)) return rc;
    return check_extent(fn, "i_n", i_n, kMostRows);
}

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_layernorm(int64_t tx, int64_t tg, void* y, int64_t ldy, const void* x, int64_t ldx, const void* g, const void* b,
                            float* mu, float* rs, int8_t* q, uint8_t* qs, int64_t i_d, int64_t i_n, double eps, hipStream_t stream) {
    const char* fn = "stade_hip_layernorm";
    if (int32_t rc = check(fn, tx, tg, i_d, i_n)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldx", ldx, i_d)) return rc;
    if (!(eps >= 0.0)) return bad(fn, "eps is negative or NaN");
    if (i_d == 0 || i_n == 0) return STADE_HIP_OK;
    if (!y || !x) return bad(fn, "null pointer");
    if (!q != !qs) return bad(fn, "q and qs go together");
    if ((uintptr_t)q % 8) return bad(fn, "q is not aligned to 8 bytes");
    WsCall call(stream, false);
    if (!call.ok()) return call.error();
    const Fwd p{y, ldy, x, ldx, g, b, mu, rs, (uint8_t*)q, qs, (int)i_d, i_n, (float)eps};
    return with_types(tx, tg, [&](auto t, auto w) -> int32_t {
        STADE_TIMED("layernorm", stream, {
            if (q) launch<decltype(t), decltype(w), true>(p, stream);
            else launch<decltype(t), decltype(w), false>(p, stream);
        });
        STADE_LAUNCHED("layernorm forward_kernel");
        return STADE_HIP_OK;
    });
}

int32_t stade_hip_layernorm_b(int64_t tx, int64_t tg, const void* yb, int64_t ldyb, const void* x, int64_t ldx, const int8_t* q,
                              const uint8_t* qs, void* xb, int64_t ldxb, const void* g, float* gb, float* bb, const float* mu,
                              const float* rs, int64_t i_d, int64_t i_n, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_layernorm_b";
    if (int32_t rc = check(fn, tx, tg, i_d, i_n)) return rc;
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_d)) return rc;
    if (x)
        if (int32_t rc = check_ld(fn, "ldx", ldx, i_d)) return rc;
    if (xb)
        if (int32_t rc = check_ld(fn, "ldxb", ldxb, i_d)) return rc;
    if (i_d == 0) return STADE_HIP_OK;
    const bool some = i_n > 0;
    if (some && (!yb || !mu || !rs)) return bad(fn, "null pointer");
    if (some && !x == !q) return bad(fn, "one of x and its tape (q, qs) is needed, and not both");
    if (!q != !qs) return bad(fn, "q and qs go together");
    if ((uintptr_t)q % 8) return bad(fn, "q is not aligned to 8 bytes");
    const bool sums = gb || bb;
    if (!some && (!sums || add)) return STADE_HIP_OK;
    // a block's rows: enough blocks for two a CU, and no more (each leaves a row of partial sums)
    const unsigned rpb = back_rows(i_d);
    const int64_t trips = (i_n + rpb - 1) / rpb;
    const bool one = some && trips <= kOneBlock && i_d <= kMostHeldBack, parts = sums && some && !one;
    WsCall call(stream, parts);   // (the workspace for the partial sums only: without them nothing has to be allocated before a capture)
    if (!call.ok()) return call.error();
    Bwd p{yb, ldyb, x, ldx, (const uint8_t*)q, qs, xb, ldxb, g, mu, rs, nullptr, nullptr, nullptr, (int)i_d, i_n, add != 0};
    // Few rows: one block, which leaves gb and bb whole (each of its trips takes about a microsecond, the second
    // launch and the scratch five).
    if (one) {
        p.gb = gb;
        p.bb = bb;
        return with_types(tx, tg, [&](auto t, auto w) -> int32_t {
            STADE_TIMED("layernorm_b", stream, {
                if (q) launch<decltype(t), decltype(w), true>(p, 1, stream);
                else launch<decltype(t), decltype(w), false>(p, 1, stream);
            });
            STADE_LAUNCHED("layernorm backward_kernel");
            return STADE_HIP_OK;
        });
    }
    // (long rows: not over 256 MiB of partial sums, but 16 blocks at least)
    const int64_t most = std::min<int64_t>(kSumParts, std::max<int64_t>(16, ((int64_t)1 << 28) / (8 * i_d)));
    const unsigned grid = (unsigned)std::min<int64_t>(trips, most);
    float* part = nullptr;
    // (as much as any fewer rows and columns take, so that a call captured after a larger eager one finds its scratch:
    // `most` rounds down, and 2^16 columns take all of the 256 MiB where some longer rows take less)
    const size_t room = std::max<size_t>((size_t)1 << 28, (size_t)16 * 8 * i_d);
    const size_t bytes = std::min((size_t)std::min<int64_t>(trips, kSumParts) * 8 * (size_t)i_d, room);
    if (parts && !(part = (float*)scratch(bytes))) return scratch_error();
    p.part = part;
    return with_types(tx, tg, [&](auto t, auto w) -> int32_t {
        if (some) {
            STADE_TIMED("layernorm_b", stream, {
                if (q) launch<decltype(t), decltype(w), true>(p, grid, stream);
                else launch<decltype(t), decltype(w), false>(p, grid, stream);
            });
            STADE_LAUNCHED("layernorm backward_kernel");
        }
        if (sums) {
            STADE_TIMED("layernorm_sum", stream,
                        weight_sum_kernel<<<dim3((unsigned)((i_d + 31) / 32), 2), kSumNT, 0, stream>>>(part, some ? (int)grid : 0, (int)i_d,
                                                                                                      gb, bb, add != 0));
            STADE_LAUNCHED("layernorm weight_sum_kernel");
        }
        return STADE_HIP_OK;
    });
}

}  // extern "C"
