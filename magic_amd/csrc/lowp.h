// Element access of the operators that take float32 or bfloat16 operands: VEC consecutive elements as floats.
#pragma once
#include <hip/hip_runtime.h>

namespace magic {

typedef __bf16 bf16_t;

template <typename T, int VEC> struct vec_of {
    typedef T type __attribute__((ext_vector_type(VEC)));
};

// predicated load, zeros where !ok (the pointer is not touched then)
template <typename T, int VEC> __device__ __forceinline__ void load_vec(const T *p, bool ok, float (&v)[VEC]) {
    if constexpr (VEC == 1) {
        v[0] = ok ? (float)*p : 0.f;
    } else {
        typedef typename vec_of<T, VEC>::type vt;
        if (ok) {
            const vt x = *reinterpret_cast<const vt *>(p);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = (float)x[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[e] = 0.f;
        }
    }
}

template <typename T, int VEC> __device__ __forceinline__ void store_vec(T *p, bool ok, const float (&v)[VEC]) {
    if (!ok) return;
    if constexpr (VEC == 1) {
        *p = (T)v[0];
    } else {
        typedef typename vec_of<T, VEC>::type vt;
        vt x;
#pragma unroll
        for (int e = 0; e < VEC; ++e) x[e] = (T)v[e];
        *reinterpret_cast<vt *>(p) = x;
    }
}

}  // namespace magic
