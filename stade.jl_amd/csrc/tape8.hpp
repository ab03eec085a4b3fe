// The 8-bit tape of an activation: what a reverse sweep needs of a forward value, held in 8 bits.
//
// A row is cut into groups of 32.  A group has one scale 2^e, the least power of two with
// max|x| <= 127 * 2^e, held as the byte e + 127, and each value is the whole number
// q = rint(x / 2^e) (to nearest even) in an int8.  x / 2^e is exact, so q is a function of x alone,
// and q * 2^e has 7 bits: it is exact in fp32, bf16 and f16 (the type that x had), so a product may
// take it as a 16-bit operand without a further rounding.  |x - q 2^e| <= 2^(e-1) <= max|x| / 127.
//   - e is at least -126 (byte 1; also of a group of zeros): there |x - q 2^e| <= 2^-127, and values
//     of at most 2^-127 become 0;
//   - where 64 * 2^e would be the element type's infinity, e is one less, and |q| stops at 127: the
//     largest values are below 128 of that scale, so they too are within max|x| / 127;
//   - a group with an infinity or a NaN has byte 255 and reads back as NaN (0 * inf).
// Rows are held at a stride of 32 * ceil(d / 32) bytes, the places past d zero, so that every
// group's 32 bytes are aligned whatever d is.
#pragma once

#include "rows.hpp"

#include <type_traits>

namespace stade {
namespace tape8 {

constexpr int kGroup = 32;
inline __host__ __device__ int64_t groups(int64_t d) { return (d + kGroup - 1) / kGroup; }

// the biased exponent of the element type's largest values
template <class T> constexpr uint32_t top_exponent() { return 254; }
template <> constexpr uint32_t top_exponent<rows::f16>() { return 142; }

struct Scale {
    uint32_t byte;   // e + 127
    float inv;       // 2^-e
};

// `big`: the largest |x| of the group as bits (bit order is size order, with NaN above infinity)
template <class T>
__device__ __forceinline__ Scale scale_of(uint32_t big) {
    const uint32_t k = big >> 23;
    // max|x| = m 2^(k-127): m 2^6 <= 127 for m up to 127/64, else one binade more, if there is one
    const bool up = (big & 0x7fffffu) > 0x7e0000u && k != top_exponent<T>();
    Scale s;
    const int b = (int)k - 6 + (up ? 1 : 0);
    s.byte = k == 255u ? 255u : (uint32_t)(b < 1 ? 1 : b);
    s.inv = k == 255u ? 0.f : __uint_as_float((254u - s.byte) << 23);
    return s;
}

__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

template <int Ctrl>
__device__ __forceinline__ uint32_t dpp_max(uint32_t v) {
    const uint32_t o = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, Ctrl, 0xF, 0xF, false);
    return v > o ? v : o;
}
// the largest over the lanes that hold a group (N values a lane: 4 lanes of 8 or 16 of 2), in each
template <int N>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
    v = dpp_max<kDppQuadSwap2>(dpp_max<kDppQuadSwap1>(v));
    if constexpr (N == 2) v = dpp_max<kDppRowRor8>(dpp_max<kDppRowRor4>(v));
    return v;
}

// The whole numbers of N values as bytes, 4 a word.  Adding 1.5 * 2^23 rounds a small fp32 value to a
// whole number, to nearest even, and leaves it in the low bits; v_perm_b32 takes the low bytes together.
// (`keep`: nothing of a group that is not finite.)
template <int N>
__device__ __forceinline__ void put(uint8_t* q, const float (&x)[N], const Scale& s) {
    uint32_t w[N];
#pragma unroll
    for (int i = 0; i < N; ++i) w[i] = __float_as_uint(__builtin_amdgcn_fmed3f(x[i] * s.inv, -127.f, 127.f) + 12582912.f);
    const uint32_t keep = s.byte == 255u ? 0u : ~0u;
    const auto two = [](uint32_t a, uint32_t b) { return __builtin_amdgcn_perm(b, a, 0x0c0c0400u); };
    if constexpr (N == 8) {
        const auto four = [&](int i) { return __builtin_amdgcn_perm(two(w[i + 2], w[i + 3]), two(w[i], w[i + 1]), 0x05040100u) & keep; };
        *reinterpret_cast<uint2*>(q) = make_uint2(four(0), four(4));
    } else {
        *reinterpret_cast<uint16_t*>(q) = (uint16_t)(two(w[0], w[1]) & keep);
    }
}

// a lane's part of a group written, from the registers that hold it: x's values at `col` of a row with
// `ng` groups (all lanes of a group together)
template <class T, int N>
__device__ __forceinline__ void store_part(uint8_t* q, uint8_t* qs, const float (&x)[N], int col, int64_t ng) {
    uint32_t big = 0;
#pragma unroll
    for (int i = 0; i < N; ++i) big = max(big, abs_bits(x[i]));
    const Scale s = scale_of<T>(group_max<N>(big));
    if (col < ng * kGroup) {
        put(q + col, x, s);
        if (col % kGroup == 0) qs[col / kGroup] = (uint8_t)s.byte;
    }
}

// 2^e of a scale byte; infinite for 255, so that its q = 0 reads as NaN
__device__ __forceinline__ float unit(uint32_t byte) { return __uint_as_float(byte << 23); }

// N bytes as they lie in memory, and their values: q + 128 as an unsigned byte, less 128, times the unit
// (both exact; 128 units may be infinite, so the unit comes last)
template <int N> using Word = std::conditional_t<N == 8, uint2, uint16_t>;
__device__ __forceinline__ float value(uint32_t biased, int byte, float u) {
    return ((float)((biased >> (8 * byte)) & 0xffu) - 128.f) * u;
}
template <int N>
__device__ __forceinline__ void values(float (&x)[N], Word<N> q, float u) {
    if constexpr (N == 8) {
        const uint32_t w[2] = {q.x ^ 0x80808080u, q.y ^ 0x80808080u};
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = value(w[i >> 2], i & 3, u);
    } else {
        const uint32_t w = (uint32_t)q ^ 0x8080u;
        x[0] = value(w, 0, u);
        x[1] = value(w, 1, u);
    }
}
template <int N>
__device__ __forceinline__ void values(float (&x)[N], const uint8_t* q, float u) {
    values(x, *reinterpret_cast<const Word<N>*>(q), u);
}

}  // namespace tape8
}  // namespace stade
