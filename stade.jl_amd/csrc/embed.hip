// Rows taken by token, and the reverse sweep that adds them back by sorted tokens.
//
//   embed        y[:, t] = s w[:, tok[t]]
//   embed_b      wb[:, v] (+)= s sum over t with tok[t] = v of yb[:, t]
//   token_order  the tokens' places in stable order of their ids, and where each id starts
//
// Ids count from 1.  0 is "no token": a zero row, and no part in wb.  Any other id outside
// 1..i_v is taken as 0 and raises the device error flag.
//
// embed is a copy, bound by HBM (a wave takes 512 columns of one row).
//
// embed_b adds no two rows by atomics: the ids are sorted first, and the sums go over the sorted
// places in order, so the same call gives the same bits.  Launches:
//   1. rank_kernel (up to 8192 tokens): every block finds the sorted places of some of them by counting,
//      or sort_block_kernel (up to 16384): block 0 sorts the ids in LDS; the same blocks, or the others,
//      write the zero rows of ids that no token has, where wb is to be set.
//   2. run_sum_kernel: the sorted places in chunks; a wave adds 512 columns of a
//      chunk's rows in fp32.  A run of one id that lies inside a chunk goes to wb at once; what a
//      chunk holds of a run that spans chunks goes to a row of partial sums (at most two a chunk).
//   3. run_join_kernel: for each run that spans chunks, its partial sums in order.
// Up to 256 tokens take one launch, few_kernel.  More tokens than one block sorts go through a radix sort over blocks, 8 bits a pass.
// Bound by HBM: yb read once, wb written once.  Measured on an MI355X: 16384 tokens of 2048 (bf16) into 65536 rows
// (fp32) 139 us, 86 of them for the zero rows (5.4 TB/s) with the sort hidden behind them, 71 added to what is there (no zero
// rows); 3001 tokens of 515 into 10007 rows (fp32) 20 us, three dependent launches.  Above 16384 tokens nothing hides the
// zero rows: 65536 tokens of 1024 into 65536 rows 190 us, added 135, of which the order by id takes 65.
#include "rows.hpp"

#include <algorithm>

namespace stade {
namespace {

using namespace rows;

constexpr int NT = 256, kCols = 512;    // columns a wave takes: 64 lanes of 8

// the id's key: id - 1, or v for no token (sorted last)
__device__ __forceinline__ uint32_t key_of(int64_t id, int64_t v, int32_t* flag) {
    if (id >= 1 && id <= v) return (uint32_t)(id - 1);
    if (id != 0 && flag) *flag = kErrIndex;
    return (uint32_t)v;
}

// ------------------------------------------------------------------------------------------
// embed
// ------------------------------------------------------------------------------------------
// A row's last vector is moved back to end with the row (the values it shares with the one before are
// written twice, the same): no tests value by value for rows of 8 or more.
template <class TY, class TW>
__global__ __launch_bounds__(NT) void embed_kernel(TY* y, int64_t ldy, const TW* w, int64_t ldw, const int64_t* tok, float s, int d, int64_t v,
                                                   int64_t t, int32_t* flag) {
    const int lane = threadIdx.x & 63, strips = (d + kCols - 1) / kCols;
    const int64_t jobs = t * strips, step = (int64_t)gridDim.x * (NT / 64);
    for (int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); j < jobs; j += step) {
        const int64_t row = j / strips;
        int col = (int)(j - row * strips) * kCols + lane * 8;
        const uint32_t key = key_of(tok[row], v, flag);
        if (col >= d) continue;
        if (d >= 8) col = min(col, d - 8);
        float x[8];
        if (key < v) {
            load_row(x, w + (int64_t)key * ldw + col, d - col);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= s;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = 0.f;
        }
        store_row(y + row * ldy + col, x, d - col);
    }
}

// ------------------------------------------------------------------------------------------
// the order by id, in one block
// ------------------------------------------------------------------------------------------
constexpr int kSortNT = 1024, kSortWaves = kSortNT / 64, kDigit = 9, kBins = 1 << kDigit;
constexpr int kSortMost = 16 * kSortNT;   // an item is 32 bits of LDS: the id's key above the place

inline int bits_of(uint64_t most) {
    int b = 1;
    while (b < 63 && (most >> b)) ++b;
    return b;
}

// Exclusive sums of the counters, digit by digit and wave by wave within it: cnt[w][b] becomes the first
// place of wave w's items of digit b.  Thread b takes digit b.
__device__ __forceinline__ void scan_bins(uint32_t (*cnt)[kBins], int bins, uint32_t* lds) {
    const int b = threadIdx.x, lane = b & 63, wave = b >> 6;
    uint32_t c[kSortWaves], total = 0;
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c[w] = b < bins ? cnt[w][b] : 0;   // (all in flight together)
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) total += c[w];
    uint32_t sum = total;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const uint32_t up = __shfl_up(sum, o, 64);
        if (lane >= o) sum += up;
    }
    if (lane == 63 && wave < kBins / 64) lds[wave] = sum;
    __syncthreads();
    if (b < bins) {
        uint32_t at = sum - total;
#pragma unroll
        for (int w = 0; w < kBins / 64; ++w) at += w < wave ? lds[w] : 0;
#pragma unroll
        for (int w = 0; w < kSortWaves; ++w) {
            cnt[w][b] = at;
            at += c[w];
        }
    }
    __syncthreads();
}

// One pass of a stable counting sort by `bits` (at most kDigit) bits from `shift` of the K items a
// thread holds: wave w holds the items w * 64 K .. in order, 64 a row.  A row's items of one
// digit find each other by ballots over the digit's bits.
template <int K>
__device__ __forceinline__ void sort_pass(uint32_t (&v)[K], int shift, int bits, uint32_t* items, uint32_t (*cnt)[kBins]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < kSortWaves << bits; i += kSortNT) cnt[i >> bits][i & (bins - 1)] = 0;
    __syncthreads();
    volatile uint32_t* mine = cnt[wave];
    uint32_t rank[K];
    const uint32_t mask = (1u << bits) - 1;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const uint32_t digit = (v[k] >> shift) & mask;
        uint64_t same = ~0ull;
        for (int b = 0; b < bits; ++b) {
            const uint64_t on = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? on : ~on;
        }
        const uint32_t before = mine[digit], below = __popcll(same & ((1ull << lane) - 1));
        rank[k] = before + below;
        __builtin_amdgcn_wave_barrier();
        if (below == 0) mine[digit] = before + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    scan_bins(cnt, bins, items);   // (the items are in registers: their place holds the waves' sums)
#pragma unroll
    for (int k = 0; k < K; ++k) items[cnt[wave][(v[k] >> shift) & mask] + rank[k]] = v[k];
    __syncthreads();
}

struct Sort {
    const int64_t* tok;
    uint32_t* key;        // out (or null): the sorted keys,
    uint32_t* place;      // and the places they had
    int64_t* order;       // out (or null): the places counted from 1
    int64_t* start;       // out (or null): the first sorted place of each of 1..i_v, and i_v's end, from 0
    int64_t v;
    int n;
    int key_bits, place_bits;
    int32_t* flag;
    // zero rows of the ids that no token has (blocks from 1 on)
    char* wb;
    int64_t row_bytes;    // stride
    int64_t width;        // bytes to be set
};

template <int K>
__device__ void sort_items(const Sort& p, uint32_t* items, uint32_t (*cnt)[kBins]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t v[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = (wave * K + k) * 64 + lane;
        v[k] = i < p.n ? key_of(p.tok[i], p.v, p.flag) << p.place_bits | (uint32_t)i : ~0u;   // (the rest sorts last)
    }
    const int passes = (p.key_bits + kDigit - 1) / kDigit, each = (p.key_bits + passes - 1) / passes;
    for (int q = 0; q < passes; ++q) {
        sort_pass<K>(v, p.place_bits + q * each, min(each, p.key_bits - q * each), items, cnt);
#pragma unroll
        for (int k = 0; k < K; ++k) v[k] = items[(wave * K + k) * 64 + lane];
        __syncthreads();
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int i = (wave * K + k) * 64 + lane;
        const uint32_t place = v[k] & ((1u << p.place_bits) - 1);
        items[i] = v[k];
        if (i < p.n) {
            if (p.key) p.key[i] = v[k] >> p.place_bits;
            if (p.place) p.place[i] = place;
            if (p.order) p.order[i] = (int64_t)place + 1;
        }
    }
    if (p.start) {
        __syncthreads();
        for (int64_t id = threadIdx.x; id <= p.v; id += kSortNT) {   // the first item of a key >= id
            int lo = 0, hi = p.n;
            while (lo < hi) {
                const int mid = (lo + hi) >> 1;
                if ((int64_t)(items[mid] >> p.place_bits) < id) lo = mid + 1;
                else hi = mid;
            }
            p.start[id] = lo;
        }
    }
}

// a row's bytes set to zero by one wave
__device__ __forceinline__ void zero_row(char* row, int64_t width) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef v4u loose4 __attribute__((aligned(2)));
    const v4u z = {0, 0, 0, 0};
    const int lane = threadIdx.x & 63;
    const int64_t whole = width / 16 * 16;
    int64_t o = lane * 16;
    for (; o + 3 * 1024 < whole; o += 4 * 1024) {
#pragma unroll
        for (int k = 0; k < 4; ++k) *reinterpret_cast<loose4*>(row + o + k * 1024) = z;
    }
    for (; o < whole; o += 1024) *reinterpret_cast<loose4*>(row + o) = z;
    for (o = whole + lane * 2; o < width; o += 64 * 2) *reinterpret_cast<uint16_t*>(row + o) = 0;
}

constexpr int kZeroRows = 1024;   // ids a block looks for at a time

// Part `part` of `parts` of the ids: marks those that a token has (reading all the tokens' keys: they are
// few, and in LDS or L2) and clears the others' rows.
template <class Key>
__device__ __forceinline__ void zero_rows(const Sort& p, int part, int parts, uint32_t* marks, Key&& key) {
    const int64_t share = (p.v + parts - 1) / parts, first = (int64_t)part * share;
    const int64_t last = min(p.v, first + share);
    for (int64_t from = first; from < last; from += kZeroRows) {
        const int rows = (int)min((int64_t)kZeroRows, last - from);
        for (int i = threadIdx.x; i < kZeroRows; i += kSortNT) marks[i] = 0;
        __syncthreads();
        for (int i = threadIdx.x; i < p.n; i += kSortNT) {
            const int64_t at = key(i) - from;
            if (at >= 0 && at < rows) marks[at] = 1;
        }
        __syncthreads();
        for (int r = threadIdx.x >> 6; r < rows; r += kSortWaves)
            if (!marks[r]) zero_row(p.wb + (from + r) * p.row_bytes, p.width);
        __syncthreads();
    }
}

// The order of few tokens by counting: an item's place is the number of items before it, those of a
// smaller key and those of its own key that came first.  Every block holds all the keys in LDS; a
// wave takes an item at a time.  n^2 comparisons over all the CUs: the launch takes 3.9, 5.6, 10.3 and 16.3 us for 1000, 3001,
// 5000 and 8192 items; the sort in one block 18.7, 26.7, 15.6 and 15.9 (of 300, 10007, 60 and 60 ids: it takes more passes
// for more ids).  The same blocks then clear rows.
constexpr int kRankMost = 8192;
__global__ __launch_bounds__(kSortNT) void rank_kernel(Sort p) {
    __shared__ uint32_t keys[kRankMost], marks[kZeroRows];
    const int lane = threadIdx.x & 63, padded = (p.n + 255) / 256 * 256;
    int64_t tok[kRankMost / kSortNT];
#pragma unroll
    for (int k = 0; k < kRankMost / kSortNT; ++k) {   // (all in flight together)
        const int i = k * kSortNT + threadIdx.x;
        tok[k] = i < p.n ? p.tok[i] : 0;
    }
#pragma unroll
    for (int k = 0; k < kRankMost / kSortNT; ++k) {
        const int i = k * kSortNT + threadIdx.x;
        if (i < padded) keys[i] = i < p.n ? key_of(tok[k], p.v, blockIdx.x == 0 ? p.flag : nullptr) : ~0u;
    }
    __syncthreads();
    const auto below = [&](uint32_t key, int place) {   // items before (key, place)
        int count = 0;
        for (int j = lane * 4; j < padded; j += 256) {
            const uint4 k = *reinterpret_cast<const uint4*>(keys + j);
            count += k.x < key + (j < place);
            count += k.y < key + (j + 1 < place);
            count += k.z < key + (j + 2 < place);
            count += k.w < key + (j + 3 < place);
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) count += __shfl_xor(count, o, 64);
        return count;
    };
    const int waves = (int)gridDim.x * kSortWaves, ids = p.start ? (int)p.v + 1 : 0;
    for (int w = (int)blockIdx.x * kSortWaves + (threadIdx.x >> 6); w < p.n + ids; w += waves) {
        if (w < p.n) {
            const uint32_t key = keys[w];
            const int at = below(key, w);
            if (lane == 0) {
                if (p.key) p.key[at] = key;
                if (p.place) p.place[at] = (uint32_t)w;
                if (p.order) p.order[at] = (int64_t)w + 1;
            }
        } else {
            const int at = below((uint32_t)(w - p.n), 0);
            if (lane == 0) p.start[w - p.n] = at;
        }
    }
    if (p.wb) {
        zero_rows(p, blockIdx.x, gridDim.x, marks, [&](int i) { return (int64_t)keys[i]; });
    }
}

template <int K>
__global__ __launch_bounds__(kSortNT) void sort_block_kernel(Sort p) {
    __shared__ uint32_t items[K * kSortNT];
    __shared__ uint32_t cnt[kSortWaves][kBins];
    if (blockIdx.x > 0) {
        zero_rows(p, blockIdx.x - 1, gridDim.x - 1, &cnt[0][0], [&](int i) { return p.tok[i] - 1; });
        return;
    }
    sort_items<K>(p, items, cnt);
}

// ------------------------------------------------------------------------------------------
// the order by id over many blocks: a radix sort of (key, place), 8 bits a pass
// ------------------------------------------------------------------------------------------
constexpr int kTile = 2048, kRadix = 256, kPer = kTile / NT;

// (pass 0 reads the tokens, the others the pairs of the pass before)
__device__ __forceinline__ uint64_t item_at(const int64_t* tok, const uint64_t* in, int64_t i, int64_t v, int32_t* flag) {
    return in ? in[i] : (uint64_t)key_of(tok[i], v, flag) << 32 | (uint64_t)i;
}

__global__ __launch_bounds__(NT) void radix_count_kernel(const int64_t* tok, const uint64_t* in, int64_t n, int64_t v, int shift, uint32_t* count,
                                                         int32_t* flag) {
    __shared__ uint32_t bins[kRadix];
    bins[threadIdx.x] = 0;
    __syncthreads();
    const int64_t first = (int64_t)blockIdx.x * kTile;
    for (int k = 0; k < kPer; ++k) {
        const int64_t i = first + k * NT + threadIdx.x;
        if (i < n) atomicAdd(&bins[(item_at(tok, in, i, v, flag) >> shift) & (kRadix - 1)], 1u);
    }
    __syncthreads();
    count[(int64_t)threadIdx.x * gridDim.x + blockIdx.x] = bins[threadIdx.x];
}

// exclusive sums of all the counters, digit by digit and block by block within it (one block)
__global__ __launch_bounds__(kSortNT) void radix_scan_kernel(uint32_t* count, int64_t m) {
    __shared__ uint32_t lds[kSortWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    uint32_t base = 0;
    for (int64_t at = 0; at < m; at += kSortNT) {
        const int64_t i = at + threadIdx.x;
        const uint32_t c = i < m ? count[i] : 0;
        uint32_t sum = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t up = __shfl_up(sum, o, 64);
            if (lane >= o) sum += up;
        }
        if (lane == 63) lds[wave] = sum;
        __syncthreads();
        uint32_t first = base, all = 0;
        for (int w = 0; w < kSortWaves; ++w) {
            if (w < wave) first += lds[w];
            all += lds[w];
        }
        if (i < m) count[i] = first + sum - c;
        base += all;
        __syncthreads();
    }
}

__global__ __launch_bounds__(NT) void radix_place_kernel(const int64_t* tok, const uint64_t* in, uint64_t* out, int64_t n, int64_t v, int shift,
                                                         const uint32_t* count) {
    __shared__ uint32_t cnt[NT / 64][kRadix];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    for (int i = threadIdx.x; i < NT / 64 * kRadix; i += NT) (&cnt[0][0])[i] = 0;
    __syncthreads();
    volatile uint32_t* mine = cnt[wave];
    const int64_t first = (int64_t)blockIdx.x * kTile + wave * 64 * kPer;
    uint64_t item[kPer];
    uint32_t rank[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
        const int64_t i = first + k * 64 + lane;
        const bool here = i < n;
        item[k] = here ? item_at(tok, in, i, v, nullptr) : 0;
        const uint32_t digit = (uint32_t)(item[k] >> shift) & (kRadix - 1);
        uint64_t same = __ballot(here);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
            const uint64_t on = __ballot((digit >> b) & 1);
            same &= (digit >> b) & 1 ? on : ~on;
        }
        const uint32_t before = mine[digit], below = __popcll(same & ((1ull << lane) - 1));
        rank[k] = before + below;
        __builtin_amdgcn_wave_barrier();
        if (here && below == 0) mine[digit] = before + __popcll(same);
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    uint32_t at = count[(int64_t)threadIdx.x * gridDim.x + blockIdx.x];
    for (int w = 0; w < NT / 64; ++w) {
        const uint32_t c = cnt[w][threadIdx.x];
        cnt[w][threadIdx.x] = at;
        at += c;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kPer; ++k)
        if (first + k * 64 + lane < n) out[cnt[wave][(uint32_t)(item[k] >> shift) & (kRadix - 1)] + rank[k]] = item[k];
}

__global__ __launch_bounds__(NT) void radix_out_kernel(const uint64_t* in, int64_t n, uint32_t* key, uint32_t* place, int64_t* order) {
    const int64_t i = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (i >= n) return;
    const uint64_t it = in[i];
    if (key) key[i] = (uint32_t)(it >> 32);
    if (place) place[i] = (uint32_t)it;
    if (order) order[i] = (int64_t)(uint32_t)it + 1;
}

// the first sorted place of each id (counted from 1), and the last id's end
__global__ __launch_bounds__(NT) void start_kernel(const uint32_t* key, int64_t n, int64_t v, int64_t* start) {
    const int64_t id = (int64_t)blockIdx.x * NT + threadIdx.x;
    if (id > v) return;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)key[mid] < id) lo = mid + 1;
        else hi = mid;
    }
    start[id] = lo;
}

// zero rows of the ids that no sorted key has (a block looks for NT ids at a time)
__global__ __launch_bounds__(NT) void zero_missing_kernel(const uint32_t* key, int64_t n, int64_t v, char* wb, int64_t row_bytes, int64_t width) {
    __shared__ uint32_t marks[NT];
    const int64_t from = (int64_t)blockIdx.x * NT, id = from + threadIdx.x;
    int64_t lo = 0, hi = n;
    while (lo < hi) {
        const int64_t mid = (lo + hi) >> 1;
        if ((int64_t)key[mid] < id) lo = mid + 1;
        else hi = mid;
    }
    marks[threadIdx.x] = lo < n && (int64_t)key[lo] == id;
    __syncthreads();
    const int rows = (int)min((int64_t)NT, v - from);
    for (int r = threadIdx.x >> 6; r < rows; r += NT / 64)
        if (!marks[r]) zero_row(wb + (from + r) * row_bytes, width);
}

// ------------------------------------------------------------------------------------------
// sums over runs of one id
// ------------------------------------------------------------------------------------------
// Sorted places a wave adds: 16, or 8 where those make few waves.  (32: 16384 rows of 2048 take 50 us, 3001 of 515 19.)
constexpr int kChunk = 16, kShortChunk = 8;

struct Runs {
    const void* yb; int64_t ldyb;
    void* wb; int64_t ldwb;
    const uint32_t* key; const uint32_t* place;
    float* part;         // two rows of d a chunk: of the run it begins with, and of the one it ends with
    float s;
    int d, add, chunk;
    int64_t n, v;
};

template <class TW, bool W>
__device__ __forceinline__ void put(const Runs& p, uint32_t key, int col, const float (&acc)[8]) {
    TW* out = (TW*)p.wb + (int64_t)key * p.ldwb + col;
    float o[8];
    if (p.add) load_row<W>(o, out, p.d - col);
#pragma unroll
    for (int i = 0; i < 8; ++i) o[i] = p.add ? fmaf(p.s, acc[i], o[i]) : p.s * acc[i];
    if (W && p.add && col % 8 != 0) {   // (moved back: what it shares with the vector before is that lane's to write)
#pragma unroll
        for (int i = 1; i < 8; ++i)
            if (i >= 8 - p.d % 8) out[i] = (TW)o[i];
    } else {
        store_row<W>(out, o, p.d - col);
    }
}

// W: no tests value by value.  A row's last vector is moved back to end with the row; what it shares with the
// one before is written twice, the same, or with `add` by the one before alone: a lane may read what it shares after the
// other has written it.
template <class TY, class TW, bool W>
__global__ __launch_bounds__(NT) void run_sum_kernel(Runs p) {
    const int strips = (p.d + kCols - 1) / kCols;
    const int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6), chunk = j / strips;
    const int64_t first = chunk * p.chunk;
    if (first >= p.n) return;
    const int lane = threadIdx.x & 63;
    int col = (int)(j - chunk * strips) * kCols + lane * 8;
    if (W && col < p.d) col = min(col, p.d - 8);
    const int len = (int)min((int64_t)p.chunk, p.n - first);
    // lane i: the chunk's i-th key and place; and the keys on both sides
    const uint32_t mykey = lane < len ? p.key[first + lane] : 0, myplace = lane < len ? p.place[first + lane] : 0;
    const uint32_t none = (uint32_t)p.v;
    const uint32_t prev = first > 0 ? p.key[first - 1] : ~0u, next = first + len < p.n ? p.key[first + len] : ~0u;
    float acc[8];
    bool begins = (uint32_t)__builtin_amdgcn_readlane((int)mykey, 0) != prev;   // the run began in this chunk
    constexpr int AHEAD = sizeof(TY) == 2 ? 16 : 8;   // rows on their way
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = 0.f;
    for (int at = 0; at < len; at += AHEAD) {
        float x[AHEAD][8];
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int i = min(at + q, len - 1);
            const int64_t row = (int64_t)(uint32_t)__builtin_amdgcn_readlane((int)myplace, i);
            load_row<W>(x[q], (const TY*)p.yb + row * p.ldyb + col, p.d - col);
        }
#pragma unroll
        for (int q = 0; q < AHEAD; ++q) {
            const int i = at + q;
            if (i >= len) break;
            const uint32_t key = (uint32_t)__builtin_amdgcn_readlane((int)mykey, i);
            if (key == none) return;   // (no token sorts last)
            const uint32_t after = i + 1 < len ? (uint32_t)__builtin_amdgcn_readlane((int)mykey, i + 1) : next;
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[c] += x[q][c];
            if (i + 1 < len && after == key) continue;
            // the run's end in this chunk
            if (col < p.d) {
                if (begins && after != key) put<TW, W>(p, key, col, acc);
                else store_row<W>(p.part + (chunk * 2 + (begins ? 1 : 0)) * p.d + col, acc, p.d - col);
            }
            begins = true;
#pragma unroll
            for (int c = 0; c < 8; ++c) acc[c] = 0.f;
        }
    }
}

template <class TW, bool W>
__global__ __launch_bounds__(NT) void run_join_kernel(Runs p) {
    const int strips = (p.d + kCols - 1) / kCols;
    const int64_t j = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6), chunk = j / strips;
    const int64_t first = chunk * p.chunk, past = first + p.chunk;
    if (past >= p.n) return;
    // the run that ends this chunk begins in it and goes on in the next one
    const uint32_t key = p.key[past - 1];
    if (key == (uint32_t)p.v || p.key[past] != key) return;
    if (p.key[first] == key && first > 0 && p.key[first - 1] == key) return;
    int col = (int)(j - chunk * strips) * kCols + (threadIdx.x & 63) * 8;
    if (W && col < p.d) col = min(col, p.d - 8);
    // the first chunk that does not begin with the run's key, looked for in 64 chunks at a time
    const int64_t chunks = (p.n + p.chunk - 1) / p.chunk;
    int64_t lo = chunk + 1;
    for (;;) {
        const int64_t c = lo + (threadIdx.x & 63);
        const uint64_t out = __ballot(c >= chunks || p.key[c * p.chunk] != key);
        if (out) {
            lo += __builtin_ctzll(out);
            break;
        }
        lo += 64;
    }
    if (col >= p.d) return;
    float acc[8], x[8];
    load_row<W>(acc, p.part + (chunk * 2 + 1) * p.d + col, p.d - col);
#pragma unroll 8
    for (int64_t c = chunk + 1; c < lo; ++c) {
        load_row<W>(x, p.part + c * 2 * p.d + col, p.d - col);
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] += x[i];
    }
    put<TW, W>(p, key, col, acc);
}

// The whole adjoint of few tokens in one launch (three take 15 us whatever their work): every wave looks among
// all the keys for those equal to its token's; the first such token's wave adds the rows of all, in
// order.  The same blocks clear the rows of the ids that no token has.
constexpr int kFewTokens = 256;
template <class TY, class TW, bool W>
__global__ __launch_bounds__(kSortNT) void few_kernel(Runs p, Sort o) {
    __shared__ uint32_t keys[kFewTokens], marks[kZeroRows];
    const int lane = threadIdx.x & 63, strips = (p.d + kCols - 1) / kCols;
    if (threadIdx.x < kFewTokens)
        keys[threadIdx.x] = (int)threadIdx.x < o.n ? key_of(o.tok[threadIdx.x], o.v, blockIdx.x == 0 ? o.flag : nullptr) : ~0u;
    __syncthreads();
    constexpr int Q = kFewTokens / 64, AHEAD = 8;
    uint32_t mine[Q];
#pragma unroll
    for (int q = 0; q < Q; ++q) mine[q] = keys[q * 64 + lane];
    const int jobs = o.n * strips, step = (int)gridDim.x * kSortWaves;
    for (int j = (int)blockIdx.x * kSortWaves + (threadIdx.x >> 6); j < jobs; j += step) {
        const int place = j / strips;
        int col = (j - place * strips) * kCols + lane * 8;
        if (W && col < p.d) col = min(col, p.d - 8);
        const uint32_t key = keys[place];
        if (key == (uint32_t)o.v) continue;
        uint64_t same[Q];
        bool first = true;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            same[q] = __ballot(mine[q] == key);
            const int before = min(64, place - q * 64);   // places of this word that lie before this one
            if (before > 0 && (same[q] & (before >= 64 ? ~0ull : (1ull << before) - 1))) first = false;
        }
        if (!first) continue;
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
        for (int q = 0; q < Q; ++q) {
            uint64_t left = same[q];
            while (left) {
                float x[AHEAD][8];
#pragma unroll
                for (int a = 0; a < AHEAD; ++a) {
                    const int row = q * 64 + (left ? __builtin_ctzll(left) : 0);
                    load_row<W>(x[a], (const TY*)p.yb + (int64_t)row * p.ldyb + col, left ? p.d - col : 0);
                    left &= left - 1;
                }
#pragma unroll
                for (int a = 0; a < AHEAD; ++a)
#pragma unroll
                    for (int i = 0; i < 8; ++i) acc[i] += x[a][i];
            }
        }
        if (col < p.d) put<TW, W>(p, key, col, acc);
    }
    if (o.wb) zero_rows(o, blockIdx.x, gridDim.x, marks, [&](int i) { return (int64_t)keys[i]; });
}

// ------------------------------------------------------------------------------------------
// host
// ------------------------------------------------------------------------------------------

// sorted keys and places into key/place, and order/start where asked; `work`: radix_bytes(n)
// of scratch, for more tokens than one block sorts
size_t radix_blocks(int64_t n) { return (size_t)((n + kTile - 1) / kTile); }
size_t radix_bytes(int64_t n) { return 2 * (size_t)n * 8 + radix_blocks(n) * kRadix * 4 + 256; }

constexpr int64_t kFewIds = 1024;   // whose starts the sorting launch finds; more ids in a launch of their own

bool one_block(int64_t n, int64_t v) {
    return n <= kRankMost || (n <= kSortMost && bits_of((uint64_t)v) + bits_of((uint64_t)(n - 1)) <= 32);
}

int32_t sort(Sort s, bool zero, void* work, int cus, hipStream_t stream) {
    const int64_t n = s.n;
    s.key_bits = bits_of((uint64_t)s.v);
    if (one_block(n, s.v)) {
        int64_t* start = s.start;
        const bool apart = s.v > kFewIds;
        if (apart) s.start = nullptr;
        if (!zero) s.wb = nullptr;
        STADE_TIMED("token_sort", stream, {
            if (n <= kRankMost) {
                const int64_t waves = (n + (s.start ? s.v + 1 : 0) + kSortWaves - 1) / kSortWaves;
                rank_kernel<<<(unsigned)std::min<int64_t>(zero ? 2 * cus : waves, 2 * cus), kSortNT, 0, stream>>>(s);
            } else {
                // block 0 sorts; the others clear rows, one a CU
                s.place_bits = bits_of((uint64_t)(n - 1));
                sort_block_kernel<kSortMost / kSortNT><<<zero ? (unsigned)std::min<int64_t>(1 + s.v, cus) : 1, kSortNT, 0, stream>>>(s);
            }
        });
        STADE_LAUNCHED("embed rank_kernel or sort_block_kernel");
        if (apart && start) {
            STADE_TIMED("token_start", stream, start_kernel<<<(unsigned)((s.v + NT) / NT), NT, 0, stream>>>(s.key, n, s.v, start));
            STADE_LAUNCHED("embed start_kernel");
        }
        return STADE_HIP_OK;
    }
    const unsigned nb = (unsigned)radix_blocks(n);
    uint64_t* a = (uint64_t*)work;
    uint64_t* b = a + n;
    uint32_t* count = (uint32_t*)(b + n);
    const uint64_t* in = nullptr;
    for (int shift = 32; shift < 32 + s.key_bits; shift += 8) {
        STADE_TIMED("token_sort", stream, {
            radix_count_kernel<<<nb, NT, 0, stream>>>(s.tok, in, n, s.v, shift, count, s.flag);
            radix_scan_kernel<<<1, kSortNT, 0, stream>>>(count, (int64_t)nb * kRadix);
            radix_place_kernel<<<nb, NT, 0, stream>>>(s.tok, in, a, n, s.v, shift, count);
        });
        STADE_LAUNCHED("embed radix kernels");
        in = a;
        std::swap(a, b);
    }
    STADE_TIMED("token_sort", stream,
                radix_out_kernel<<<(unsigned)((n + NT - 1) / NT), NT, 0, stream>>>(in, n, s.key, s.place, s.order));
    STADE_LAUNCHED("embed radix_out_kernel");
    if (s.start) {
        STADE_TIMED("token_start", stream, start_kernel<<<(unsigned)((s.v + NT) / NT), NT, 0, stream>>>(s.key, n, s.v, s.start));
        STADE_LAUNCHED("embed start_kernel");
    }
    if (zero) {
        STADE_TIMED("embed_zero", stream,
                    zero_missing_kernel<<<(unsigned)((s.v + NT - 1) / NT), NT, 0, stream>>>(s.key, n, s.v, s.wb, s.row_bytes, s.width));
        STADE_LAUNCHED("embed zero_missing_kernel");
    }
    return STADE_HIP_OK;
}

int cu_count() {
    int dev = 0, cus = 0;
    if (hipGetDevice(&dev) != hipSuccess || hipDeviceGetAttribute(&cus, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 256;
    return cus > 0 ? cus : 256;
}

int32_t* error_flag(Workspace* ws) { return (int32_t*)(ws->dscalars + kErrFlagSlot); }

__global__ __launch_bounds__(NT) void zero_all_kernel(char* wb, int64_t rows, int64_t row_bytes, int64_t width) {
    for (int64_t r = (int64_t)blockIdx.x * (NT / 64) + (threadIdx.x >> 6); r < rows; r += (int64_t)gridDim.x * (NT / 64)) zero_row(wb + r * row_bytes, width);
}

// Bytes of partial sums, two rows a chunk: enough for any fewer tokens and columns too, so that a call captured after a
// larger eager one finds its scratch.  Short chunks are for less than 2048 strips (below), whose partial
// sums take less than 17 MiB: t / 16 * strips < 2048 and d <= 512 strips.
constexpr size_t kShortMost = (size_t)17 << 20;
size_t part_bytes(int64_t t, int64_t d) {
    const size_t whole = (size_t)((t + kChunk - 1) / kChunk) * 2 * (size_t)d * 4, brief = (size_t)((t + kShortChunk - 1) / kShortChunk) * 2 * (size_t)d * 4;
    return (std::max(whole, std::min(brief, kShortMost)) + 255) / 256 * 256;
}

constexpr int64_t kMostIds = (int64_t)1 << 30;

}  // namespace
}  // namespace stade

using namespace stade;

extern "C" {

int32_t stade_hip_token_order(const int64_t* tok, int64_t* order, int64_t* start, int64_t i_v, int64_t i_t, hipStream_t stream) {
    const char* fn = "stade_hip_token_order";
    if (int32_t rc = check_extent(fn, "i_v", i_v, kMostIds)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (!start || (i_t > 0 && (!tok || !order))) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    if (i_t == 0) {
        STADE_TIMED("token_start", stream, start_kernel<<<(unsigned)((i_v + NT) / NT), NT, 0, stream>>>(nullptr, 0, i_v, start));
        STADE_LAUNCHED("embed start_kernel");
        return STADE_HIP_OK;
    }
    const bool one = one_block(i_t, i_v);
    Sort s{};
    s.tok = tok;
    s.order = order;
    s.start = start;
    s.v = i_v;
    s.n = (int)i_t;
    s.flag = error_flag(call.ws);
    char* work = nullptr;
    if (!one || i_v > kFewIds) {
        const size_t keys = ((size_t)i_t * 4 + 255) / 256 * 256;
        if (!(work = (char*)scratch(keys + (one ? 0 : radix_bytes(i_t))))) return scratch_error();
        s.key = (uint32_t*)work;
        work += keys;
    }
    return sort(s, false, work, cu_count(), stream);
}

int32_t stade_hip_embed(int64_t ty, int64_t tw, void* y, int64_t ldy, const void* w, int64_t ldw, const int64_t* tok, double s, int64_t i_d,
                        int64_t i_v, int64_t i_t, hipStream_t stream) {
    const char* fn = "stade_hip_embed";
    if (int32_t rc = check_type(fn, "y", ty)) return rc;
    if (int32_t rc = check_type(fn, "w", tw)) return rc;
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_v", i_v, kMostIds)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (int32_t rc = check_ld(fn, "ldy", ldy, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldw", ldw, i_d)) return rc;
    if (i_d == 0 || i_t == 0) return STADE_HIP_OK;
    if (!y || !tok || (i_v > 0 && !w)) return bad(fn, "null pointer");
    WsCall call(stream);
    if (!call.ok()) return call.error();
    const int64_t jobs = i_t * ((i_d + kCols - 1) / kCols);
    const unsigned grid = (unsigned)std::min<int64_t>((jobs + NT / 64 - 1) / (NT / 64), 1 << 16);
    return with_type(ty, [&](auto a) -> int32_t {
        return with_type(tw, [&](auto b) -> int32_t {
            using TY = decltype(a);
            using TW = decltype(b);
            STADE_TIMED("embed", stream,
                        embed_kernel<TY, TW><<<grid, NT, 0, stream>>>((TY*)y, ldy, (const TW*)w, ldw, tok, (float)s, (int)i_d, i_v, i_t,
                                                                      error_flag(call.ws)));
            STADE_LAUNCHED("embed embed_kernel");
            return STADE_HIP_OK;
        });
    });
}

int32_t stade_hip_embed_b(int64_t ty, int64_t tw, const void* yb, int64_t ldyb, void* wb, int64_t ldwb, const int64_t* tok, double s,
                          int64_t i_d, int64_t i_v, int64_t i_t, int64_t add, hipStream_t stream) {
    const char* fn = "stade_hip_embed_b";
    if (int32_t rc = check_type(fn, "yb", ty)) return rc;
    if (int32_t rc = check_type(fn, "wb", tw)) return rc;
    if (int32_t rc = check_extent(fn, "i_d", i_d, kMostCols)) return rc;
    if (int32_t rc = check_extent(fn, "i_v", i_v, kMostIds)) return rc;
    if (int32_t rc = check_extent(fn, "i_t", i_t, kMostRows)) return rc;
    if (int32_t rc = check_ld(fn, "ldyb", ldyb, i_d)) return rc;
    if (int32_t rc = check_ld(fn, "ldwb", ldwb, i_d)) return rc;
    if (i_d == 0 || (i_v == 0 && i_t == 0)) return STADE_HIP_OK;
    if ((i_v > 0 && !wb) || (i_t > 0 && (!yb || !tok))) return bad(fn, "null pointer");
    const int64_t row_bytes = ldwb * type_size(tw), width = i_d * type_size(tw);
    if (i_t == 0 && add) return STADE_HIP_OK;
    WsCall call(stream, i_t > 0);
    if (!call.ok()) return call.error();
    if (i_t == 0) {
        STADE_TIMED("embed_zero", stream,
                    zero_all_kernel<<<(unsigned)std::min<int64_t>(i_v, 1 << 16), NT, 0, stream>>>((char*)wb, i_v, row_bytes, width));
        STADE_LAUNCHED("embed zero_all_kernel");
        return STADE_HIP_OK;
    }
    const int64_t strips = (i_d + kCols - 1) / kCols;
    const bool w = i_d >= 8;
    if (i_t <= kFewTokens) {
        Sort o{};
        o.tok = tok;
        o.v = i_v;
        o.n = (int)i_t;
        o.flag = error_flag(call.ws);
        o.wb = add || i_v == 0 ? nullptr : (char*)wb;
        o.row_bytes = row_bytes;
        o.width = width;
        Runs p{};
        p.yb = yb; p.ldyb = ldyb; p.wb = wb; p.ldwb = ldwb; p.s = (float)s; p.d = (int)i_d; p.add = add != 0;
        const int64_t cus = cu_count();
        const unsigned grid = (unsigned)(o.wb ? 2 * cus : std::min<int64_t>((i_t * strips + kSortWaves - 1) / kSortWaves, 4 * cus));
        return with_type(ty, [&](auto a) -> int32_t {
            return with_type(tw, [&](auto b) -> int32_t {
                using TY = decltype(a);
                using TW = decltype(b);
                STADE_TIMED("embed_few", stream, {
                    if (w) few_kernel<TY, TW, true><<<grid, kSortNT, 0, stream>>>(p, o);
                    else few_kernel<TY, TW, false><<<grid, kSortNT, 0, stream>>>(p, o);
                });
                STADE_LAUNCHED("embed few_kernel");
                return STADE_HIP_OK;
            });
        });
    }
    const int64_t chunk = i_t / kChunk * strips < 2048 ? kShortChunk : kChunk, chunks = (i_t + chunk - 1) / chunk;
    const size_t keys = ((size_t)i_t * 4 + 255) / 256 * 256, parts = part_bytes(i_t, i_d);
    const bool one = one_block(i_t, i_v);
    char* work = (char*)scratch(2 * keys + parts + (one ? 0 : radix_bytes(i_t)));
    if (!work) return scratch_error();
    Sort o{};
    o.tok = tok;
    o.key = (uint32_t*)work;
    o.place = (uint32_t*)(work + keys);
    o.v = i_v;
    o.n = (int)i_t;
    o.flag = error_flag(call.ws);
    o.wb = (char*)wb;
    o.row_bytes = row_bytes;
    o.width = width;
    if (int32_t rc = sort(o, !add && i_v > 0, work + 2 * keys + parts, cu_count(), stream)) return rc;
    const Runs p{yb, ldyb, wb, ldwb, o.key, o.place, (float*)(work + 2 * keys), (float)s, (int)i_d, add != 0, (int)chunk, i_t, i_v};
    const unsigned grid = (unsigned)((chunks * strips + NT / 64 - 1) / (NT / 64));
    return with_type(ty, [&](auto a) -> int32_t {
        return with_type(tw, [&](auto b) -> int32_t {
            using TY = decltype(a);
            using TW = decltype(b);
            STADE_TIMED("embed_runs", stream, {
                if (w) run_sum_kernel<TY, TW, true><<<grid, NT, 0, stream>>>(p);
                else run_sum_kernel<TY, TW, false><<<grid, NT, 0, stream>>>(p);
            });
            STADE_LAUNCHED("embed run_sum_kernel");
            if (chunks > 1) {
                STADE_TIMED("embed_join", stream, {
                    if (w) run_join_kernel<TW, true><<<grid, NT, 0, stream>>>(p);
                    else run_join_kernel<TW, false><<<grid, NT, 0, stream>>>(p);
                });
                STADE_LAUNCHED("embed run_join_kernel");
            }
            return STADE_HIP_OK;
        });
    });
}

}  // extern "C"
