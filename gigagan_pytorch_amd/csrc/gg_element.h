// gg_element.h — element types of the transformer operators: bf16, IEEE half and fp32 rows, read and written eight values at a time
// and computed in fp32.
#pragma once
#include "gg_device.h"

enum { GG_ELT_BF16 = 0, GG_ELT_F16 = 1, GG_ELT_F32 = 2 };

template <int T> struct GgElt { typedef unsigned short type; };
template <> struct GgElt<GG_ELT_F32> { typedef float type; };

template <int T>
GG_HOST_DEVICE float gg_elt_f(typename GgElt<T>::type x) {
    if constexpr (T == GG_ELT_BF16) return gg_bf2f(x);
    else if constexpr (T == GG_ELT_F16) return gg_h2f(x);
    else return x;
}
template <int T>
GG_HOST_DEVICE typename GgElt<T>::type gg_elt(float f) {
    if constexpr (T == GG_ELT_BF16) return gg_f2bf(f);
    else if constexpr (T == GG_ELT_F16) return gg_f2h(f);
    else return f;
}

// 16 bytes at any element address: a row whose width no vector divides starts anywhere. (The target reads and writes global memory at
// any byte; an aligned address costs the same through these types.)
typedef u32x4 __attribute__((aligned(2))) gg_u32x4_a2;

// eight consecutive elements as they lie in memory
template <int T> struct GgRaw8 { u32x4 w[T == GG_ELT_F32 ? 2 : 1]; };

template <int T>
GG_DEVICE GgRaw8<T> gg_raw8_load(const typename GgElt<T>::type* p, int n) {     // n valid elements (>= 8: all), the rest zero
    GgRaw8<T> r;
    if (n >= 8) {
        r.w[0] = *(const gg_u32x4_a2*)p;
        if constexpr (T == GG_ELT_F32) r.w[1] = *(const gg_u32x4_a2*)(p + 4);
        return r;
    }
    if constexpr (T == GG_ELT_F32) {
        for (int e = 0; e < 8; ++e) r.w[e >> 2][e & 3] = e < n ? __builtin_bit_cast(unsigned, p[e]) : 0u;
    } else {
        for (int e = 0; e < 4; ++e)
            r.w[0][e] = (2 * e < n ? (unsigned)p[2 * e] : 0u) | ((2 * e + 1 < n ? (unsigned)p[2 * e + 1] : 0u) << 16);
    }
    return r;
}
template <int T>
GG_DEVICE float gg_raw8_get(const GgRaw8<T>& r, int e) {
    if constexpr (T == GG_ELT_F32) {
        const unsigned u = r.w[e >> 2][e & 3];          // (a bit cast of the vector element itself reads element 0)
        return __builtin_bit_cast(float, u);
    }
    else return gg_elt_f<T>((unsigned short)(r.w[0][e >> 1] >> (16 * (e & 1))));
}
template <int T>
GG_DEVICE void gg_raw8_set(GgRaw8<T>& r, const float* v) {
    if constexpr (T == GG_ELT_F32) {
        for (int e = 0; e < 8; ++e) r.w[e >> 2][e & 3] = __builtin_bit_cast(unsigned, v[e]);
    } else {
        for (int e = 0; e < 4; ++e) r.w[0][e] = (unsigned)gg_elt<T>(v[2 * e]) | ((unsigned)gg_elt<T>(v[2 * e + 1]) << 16);
    }
}
template <int T>
GG_DEVICE void gg_raw8_store(typename GgElt<T>::type* p, const GgRaw8<T>& r, int n) {
    if (n >= 8) {
        *(gg_u32x4_a2*)p = r.w[0];
        if constexpr (T == GG_ELT_F32) *(gg_u32x4_a2*)(p + 4) = r.w[1];
        return;
    }
    for (int e = 0; e < 8; ++e)
        if (e < n) {
            if constexpr (T == GG_ELT_F32) p[e] = gg_raw8_get<T>(r, e);
            else p[e] = (unsigned short)(r.w[0][e >> 1] >> (16 * (e & 1)));
        }
}
