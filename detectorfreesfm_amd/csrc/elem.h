// Element types and row vectors of the kernels that take fp32, bf16 and fp16 tensors alike (norm_train.hip, rotary.hip,
// cross_attention.hip).
#pragma once
#include "common.h"

namespace dfsfm {

using bf16 = __bf16;
using f16 = _Float16;

// V elements as one load or store.  The vectors are declared with the ELEMENT's alignment: rows of odd width or stride keep the wide
// access (gfx950 serves global accesses of any alignment), so no kernel needs a scalar form beside it.
template <typename T, int V>
struct Vec {
    typedef T raw __attribute__((ext_vector_type(V)));
    typedef raw type __attribute__((aligned(sizeof(T))));
};

template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, float (&r)[V]) {
    const typename Vec<T, V>::type v = *reinterpret_cast<const typename Vec<T, V>::type*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) r[e] = (float)v[e];
}

// the first n of V elements, zeros behind them
template <typename T, int V>
__device__ __forceinline__ void load_f32(const T* p, int64_t n, float (&r)[V]) {
    if (n >= V) {
        load_f32<T, V>(p, r);
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) r[e] = e < n ? (float)p[e] : 0.f;
    }
}

// round to nearest even, once
template <typename T, int V>
__device__ __forceinline__ void store_f32(T* p, int64_t n, const float (&r)[V]) {
    if (n >= V) {
        typename Vec<T, V>::type v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = (T)r[e];
        *reinterpret_cast<typename Vec<T, V>::type*>(p) = v;
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (e < n) p[e] = (T)r[e];
    }
}

}  // namespace dfsfm
