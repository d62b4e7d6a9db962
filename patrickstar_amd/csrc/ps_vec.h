// Element types of the operators and their vector accesses: registers hold 32-bit floats, memory fp16, bf16 or fp32.
#ifndef PS_VEC_H
#define PS_VEC_H

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

namespace {

typedef _Float16 half_t;
typedef __bf16 bf16_t;

template <int N>
using Int = std::integral_constant<int, N>;

// Operands are device memory: said so, the compiler need not use flat accesses.
template <typename T>
__device__ __forceinline__ __attribute__((address_space(1))) T* global(T* p)
{
    return (__attribute__((address_space(1))) T*)(p);
}

template <typename T>
__device__ __forceinline__ float to_float(T x)
{
    return (float)x;
}

// Rounds to nearest, ties to even; what is beyond the type's range becomes infinite.
template <typename T>
__device__ __forceinline__ T from_float(float x)
{
    return (T)x;
}

template <typename T, int V>
struct VecOf {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct VecOf<T, 1> {
    typedef T type;
};

// V elements whose address is a multiple of their size.
template <typename T, int V>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[V])
{
    if constexpr (V == 1) {
        out[0] = to_float<T>(*global(p));
    } else {
        typedef typename VecOf<T, V>::type vec;
        const vec v = *global(reinterpret_cast<const vec*>(p));
#pragma unroll
        for (int e = 0; e < V; ++e) out[e] = to_float<T>(v[e]);
    }
}

template <typename T, int V>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[V])
{
    if constexpr (V == 1) {
        *global(p) = from_float<T>(in[0]);
    } else {
        typedef typename VecOf<T, V>::type vec;
        vec v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = from_float<T>(in[e]);
        *global(reinterpret_cast<vec*>(p)) = v;
    }
}

}  // namespace

#endif  // PS_VEC_H
