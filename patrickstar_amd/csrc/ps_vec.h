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
__device__ __forceinline__ typename VecOf<T, V>::type load_raw(const T* p)
{
    return *global(reinterpret_cast<const typename VecOf<T, V>::type*>(p));
}
// STREAM: with the non-temporal hint
template <typename T, int V, bool STREAM = false>
__device__ __forceinline__ void store_raw(T* p, typename VecOf<T, V>::type v)
{
    if constexpr (STREAM)
        __builtin_nontemporal_store(v, global(reinterpret_cast<typename VecOf<T, V>::type*>(p)));
    else
        *global(reinterpret_cast<typename VecOf<T, V>::type*>(p)) = v;
}

template <typename T, int V>
__device__ __forceinline__ float element(typename VecOf<T, V>::type v, int e)
{
    if constexpr (V == 1)
        return to_float<T>(v);
    else
        return to_float<T>(v[e]);
}
template <typename T, int V>
__device__ __forceinline__ T get(typename VecOf<T, V>::type v, int e)
{
    if constexpr (V == 1)
        return v;
    else
        return v[e];
}
template <typename T, int V>
__device__ __forceinline__ void put(typename VecOf<T, V>::type& v, int e, T x)
{
    if constexpr (V == 1)
        v = x;
    else
        v[e] = x;
}
template <typename T, int V>
__device__ __forceinline__ void set_element(typename VecOf<T, V>::type& v, int e, float x)
{
    put<T, V>(v, e, from_float<T>(x));
}

// A value of 32 or 64 bits of another lane of the same 16, as CTRL says, and of one lane for the whole wave.  (All lanes take part.)
template <typename N>
struct Words {
    int w[sizeof(N) / 4];
};
template <int CTRL, typename N>
__device__ __forceinline__ N moved(N v)
{
    Words<N> x = __builtin_bit_cast(Words<N>, v);
#pragma unroll
    for (unsigned i = 0; i < sizeof(N) / 4; ++i) x.w[i] = __builtin_amdgcn_update_dpp(0, x.w[i], CTRL, 0xF, 0xF, true);
    return __builtin_bit_cast(N, x);
}
template <typename N>
__device__ __forceinline__ N of_lane(N v, int lane)
{
    Words<N> x = __builtin_bit_cast(Words<N>, v);
#pragma unroll
    for (unsigned i = 0; i < sizeof(N) / 4; ++i) x.w[i] = __builtin_amdgcn_readlane(x.w[i], lane);
    return __builtin_bit_cast(N, x);
}

}  // namespace

#endif  // PS_VEC_H
