// Sines and cosines of rotary positions, rows in pieces of 1 to 8 elements, the rotation of a piece.
#pragma once

#include "pe_common.h"

namespace pe {

struct SinCos {
    float s, c;
};

// amp * (sin, cos) of pos * f quarter turns.
PE_DEV SinCos sincos_quarters(double pos, double f, float amp) {
    const double p = pos * f, e = fma(pos, f, -p), n = rint(p);
    const float x = (float)((p - n) + e) * 1.5707963267948966f;
    const int q = (int)(int64_t)(n - 4.0 * floor(n * 0.25));
    const float z = x * x;
    float s = fmaf(z, -2.5052108385441720e-8f, 2.7557319223985893e-6f);
    s = fmaf(z, s, -1.9841269841269841e-4f);
    s = fmaf(z, s, 8.3333333333333333e-3f);
    s = fmaf(z, s, -1.6666666666666667e-1f);
    s = fmaf(x * z, s, x);
    float c = fmaf(z, -2.7557319223985888e-7f, 2.4801587301587302e-5f);
    c = fmaf(z, c, -1.3888888888888889e-3f);
    c = fmaf(z, c, 4.1666666666666667e-2f);
    c = fmaf(z, c, -0.5f);
    c = fmaf(z, c, 1.0f);
    const float a = q & 1 ? c : s, b = q & 1 ? s : c;
    return {(q & 2 ? -a : a) * amp, ((q + 1) & 2 ? -b : b) * amp};
}

template <typename T, int V>
struct Vec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct Vec<T, 1> {
    typedef T type;
};

template <typename T, int V>
PE_DEV void load_vec(const T* p, float* v) {
    const auto x = *reinterpret_cast<const typename Vec<T, V>::type*>(p);
    if constexpr (V == 1) {
        v[0] = (float)x;
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)x[i];
    }
}
template <typename T, int V>
PE_DEV void store_vec(T* p, const float* v) {
    typename Vec<T, V>::type x;
    if constexpr (V == 1) {
        x = (T)v[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)v[i];
    }
    *reinterpret_cast<typename Vec<T, V>::type*>(p) = x;
}

PE_DEV int64_t position_of(const void* positions, int wide, int64_t t) {
    return wide ? static_cast<const int64_t*>(positions)[t] : (int64_t) static_cast<const int*>(positions)[t];
}

// One item is V pairs: the elements at[0 .. V) and at[far .. far + V), or, interleaved, the 2 V
// elements from at on.
template <int V, bool IL>
PE_DEV void rotate(float* a, float* b, const SinCos* w) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
        float& x = IL ? (2 * i < V ? a[2 * i] : b[2 * i - V]) : a[i];
        float& y = IL ? (2 * i + 1 < V ? a[2 * i + 1] : b[2 * i + 1 - V]) : b[i];
        const float u = x * w[i].c - y * w[i].s;
        y = x * w[i].s + y * w[i].c;
        x = u;
    }
}

}  // namespace pe
