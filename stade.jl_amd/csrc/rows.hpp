// Element types and row access shared by the language-model operators (embed, layernorm, tape8,
// expert_mul): rows of float, bf16 or f16 values, each row's values one after the other and rows a
// stride apart.  Values are widened to fp32 when loaded and rounded once, to nearest even, when
// stored.
#pragma once

#include "internal.hpp"
#include "../../include/stade_hip.h"

namespace stade {
namespace rows {

typedef __bf16 bf16;
typedef _Float16 f16;

template <class T> struct Code;
template <> struct Code<float> { static constexpr int64_t value = STADE_HIP_F32; };
template <> struct Code<bf16> { static constexpr int64_t value = STADE_HIP_BF16; };
template <> struct Code<f16> { static constexpr int64_t value = STADE_HIP_F16; };

inline bool known_type(int64_t t) { return t == STADE_HIP_F32 || t == STADE_HIP_BF16 || t == STADE_HIP_F16; }
inline int64_t type_size(int64_t t) { return t == STADE_HIP_F32 ? 4 : 2; }

// f(T{}) for the element type of a code
template <class F>
inline int32_t with_type(int64_t code, F&& f) {
    return code == STADE_HIP_F32 ? f(float{}) : code == STADE_HIP_BF16 ? f(bf16{}) : f(f16{});
}

// N consecutive values at any element alignment: the hardware's wide loads and stores need no more
// than that, so views and odd row lengths take the same path as aligned rows.
template <class T, int N>
struct Pack {
    typedef T vec __attribute__((ext_vector_type(N)));
    typedef vec loose __attribute__((aligned(sizeof(T))));
};

// p[0..N) into v; values at and past `left` read as zero.  WHOLE: `left` is a multiple of N (rows whose
// length is one), and there are no tests value by value.
template <bool WHOLE = false, int N, class T>
__device__ __forceinline__ void load_row(float (&v)[N], const T* p, int left) {
    if constexpr (WHOLE) {
        typename Pack<T, N>::vec x = {};
        if (left > 0) x = *reinterpret_cast<const typename Pack<T, N>::loose*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)x[i];
    } else if (left >= N) {
        const typename Pack<T, N>::loose x = *reinterpret_cast<const typename Pack<T, N>::loose*>(p);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = (float)x[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
        if (left > 0) {   // (lanes past the row stay out of the loads and their waits)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] = i < left ? (float)p[i] : 0.f;
        }
    }
}

template <bool WHOLE = false, int N, class T>
__device__ __forceinline__ void store_row(T* p, const float (&v)[N], int left) {
    if (WHOLE ? left > 0 : left >= N) {
        typename Pack<T, N>::vec x;
#pragma unroll
        for (int i = 0; i < N; ++i) x[i] = (T)v[i];
        *reinterpret_cast<typename Pack<T, N>::loose*>(p) = x;
    } else if constexpr (!WHOLE) {
        if (left > 0) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (i < left) p[i] = (T)v[i];
        }
    }
}

// the argument checks that the operators share
inline int32_t bad(const char* fn, const char* what) { return set_error(STADE_HIP_EINVAL, "%s: %s", fn, what); }
inline int32_t check_type(const char* fn, const char* name, int64_t t) {
    return known_type(t) ? 0 : set_error(STADE_HIP_EINVAL, "%s: %s: unknown element type %lld", fn, name, (long long)t);
}
inline int32_t check_extent(const char* fn, const char* name, int64_t v, int64_t most) {
    if (v < 0) return set_error(STADE_HIP_EINVAL, "%s: %s is negative", fn, name);
    if (v > most) return set_error(STADE_HIP_ERANGE, "%s: %s = %lld is above %lld", fn, name, (long long)v, (long long)most);
    return 0;
}
inline int32_t check_ld(const char* fn, const char* name, int64_t ld, int64_t d) {
    return ld >= d ? 0 : set_error(STADE_HIP_EINVAL, "%s: %s = %lld is less than the row's %lld", fn, name, (long long)ld, (long long)d);
}

constexpr int64_t kMostRows = (int64_t)1 << 30, kMostCols = (int64_t)1 << 24;

}  // namespace rows
}  // namespace stade
