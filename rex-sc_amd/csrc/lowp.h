// Element types of the operators that take float32, float16 or bfloat16 tensors, and what they share.  Arithmetic is
// float32 throughout: a 16-bit tensor is widened on the load and rounded once, half to even, on the store.
#pragma once
#include "rexsc_common.h"

namespace rexsc {

typedef _Float16 f16_t;
typedef __bf16 bf16_t;

inline size_t dtype_size(int dtype) { return dtype == REXSC_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == REXSC_F32 || dtype == REXSC_F16 || dtype == REXSC_BF16; }

// Calls the statement with T = the element type of a dtype code that has passed dtype_ok().
#define REXSC_DTYPE_SWITCH(dtype, ...)                                              \
    do {                                                                            \
        if ((dtype) == REXSC_F32) { typedef float T; __VA_ARGS__; }                 \
        else if ((dtype) == REXSC_F16) { typedef ::rexsc::f16_t T; __VA_ARGS__; }   \
        else { typedef ::rexsc::bf16_t T; __VA_ARGS__; }                            \
    } while (0)

template <typename T, int V> struct VecOf { typedef T type __attribute__((ext_vector_type(V))); };
template <typename T> struct VecOf<T, 1> { typedef T type; };
// The same, aligned to its element only: one load or store of as many bytes wherever it lies.
template <typename T, int V> struct LooseVecOf { typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T)))); };

// The first n of the V elements from p on, zeros behind them.
template <typename T, int V>
__device__ __forceinline__ typename VecOf<T, V>::type load_some(const T *p, int n)
{
    typename VecOf<T, V>::type v{};
    if (n >= V) v = *(const typename LooseVecOf<T, V>::type *)p;
    else if (n > 0) {
#pragma unroll
        for (int i = 0; i < V - 1; i++)
            if (i < n) v[i] = p[i];
    }
    return v;
}
// The same where `before` elements in front of p may be read: where fewer than V are left, the vector that ends with the
// last one is read and shifted down, one load all the same.
template <typename T, int V>
__device__ __forceinline__ typename VecOf<T, V>::type load_some(const T *p, int n, int before)
{
    static_assert(V * sizeof(T) == 16, "shifted as a 128-bit integer");
    typename VecOf<T, V>::type v{};
    const int back = n < V ? V - n : 0;
    if (n > 0 && back <= before) {
        v = *(const typename LooseVecOf<T, V>::type *)(p - back);
        if (back) v = __builtin_bit_cast(typename VecOf<T, V>::type, __builtin_bit_cast(unsigned __int128, v) >> (back * 8 * (int)sizeof(T)));
    } else if (n > 0) {
#pragma unroll
        for (int i = 0; i < V - 1; i++)
            if (i < n) v[i] = p[i];
    }
    return v;
}
// Stores the first n of V elements.
template <typename T, int V>
__device__ __forceinline__ void store_some(T *p, typename VecOf<T, V>::type v, int n)
{
    if (n >= V) *(typename LooseVecOf<T, V>::type *)p = v;
    else if (n > 0) {
#pragma unroll
        for (int i = 0; i < V - 1; i++)
            if (i < n) p[i] = v[i];
    }
}

// V consecutive elements, widened.  p is aligned to V * sizeof(T).
template <int V, typename T>
__device__ __forceinline__ void load_vec(float (&out)[V], const T *p)
{
    const typename VecOf<T, V>::type v = *(const typename VecOf<T, V>::type *)p;
    if constexpr (V == 1) out[0] = (float)v;
    else {
#pragma unroll
        for (int i = 0; i < V; i++) out[i] = (float)v[i];
    }
}

template <int V, typename T>
__device__ __forceinline__ void store_vec(T *p, const float (&in)[V])
{
    typename VecOf<T, V>::type v;
    if constexpr (V == 1) v = (T)in[0];
    else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = (T)in[i];
    }
    *(typename VecOf<T, V>::type *)p = v;
}

// One element of a tensor whose type is known at run time only (wave-uniform branch): biases.
__device__ __forceinline__ float load_any(const void *p, int dtype, size_t i)
{
    if (dtype == REXSC_F32) return ((const float *)p)[i];
    if (dtype == REXSC_F16) return (float)((const f16_t *)p)[i];
    return (float)((const bf16_t *)p)[i];
}
__device__ __forceinline__ void store_any(void *p, int dtype, size_t i, float v)
{
    if (dtype == REXSC_F32) ((float *)p)[i] = v;
    else if (dtype == REXSC_F16) ((f16_t *)p)[i] = (f16_t)v;
    else ((bf16_t *)p)[i] = (bf16_t)v;
}

// Maximum over the 64 lanes, the result in every lane.
__device__ __forceinline__ unsigned wave_max(unsigned v)
{
#pragma unroll
    for (int s = 32; s; s >>= 1) {
        const unsigned o = (unsigned)__shfl_xor((int)v, s, 64);
        v = v > o ? v : o;
    }
    return v;
}

// |x| as an unsigned integer: ordered like the magnitude, with infinity above every number and NaN above infinity,
// so that a maximum over it never loses a NaN.
__device__ __forceinline__ unsigned mag_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// Column sums of partial results: out[c] = sum_r part[r][c] for `cols` columns of `rows` float32 rows at distance
// `ld`, and out2[c] = sum_r part[r][cols + c] (either may be NULL), in a fixed order, rounded to out_dtype.  Launched by
// the operators that accumulate a weight's or bias's gradient per block first (no atomics: the same inputs give the
// same bits).
int launch_column_sums(const float *part, size_t rows, size_t cols, size_t ld, void *out, void *out2, int out_dtype,
                       hipStream_t stream);

} // namespace rexsc
