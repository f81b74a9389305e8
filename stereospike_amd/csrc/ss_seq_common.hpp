// ss_seq_common.hpp — shared device helpers of the ss_seq_*.hip units (sequence operators).
#pragma once
#include <hip/hip_runtime.h>
#include <hip/hip_fp16.h>
#include <hip/hip_bf16.h>
#include <stdint.h>
#include <math.h>
#include <type_traits>

#include "ss_sequence.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x16 __attribute__((ext_vector_type(16)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x4 __attribute__((ext_vector_type(4)));
typedef unsigned short u16x8 __attribute__((ext_vector_type(8)));

// storage type of an activation of element type DT, and its conversions (narrowing rounds to nearest even)
template <int DT> struct Elem { typedef float type; };
template <> struct Elem<SS_SEQ_F16> { typedef unsigned short type; };
template <> struct Elem<SS_SEQ_BF16> { typedef unsigned short type; };
template <int DT> using elem_t = typename Elem<DT>::type;

template <int DT> __device__ __forceinline__ float widen(elem_t<DT> v)
{
    if constexpr (DT == SS_SEQ_F32) return v;
    else if constexpr (DT == SS_SEQ_F16) return (float)__builtin_bit_cast(_Float16, v);
    else return __uint_as_float((unsigned)v << 16);
}
template <int DT> __device__ __forceinline__ elem_t<DT> narrow(float v)
{
    if constexpr (DT == SS_SEQ_F32) return v;
    else if constexpr (DT == SS_SEQ_F16) return __builtin_bit_cast(unsigned short, (_Float16)v);
    else return __builtin_bit_cast(unsigned short, (__bf16)v);
}

// N consecutive elements as one access of N * sizeof bytes
template <int DT, int N> struct alignas(N * sizeof(elem_t<DT>)) Pack { elem_t<DT> v[N]; };

__device__ __forceinline__ float wave_sum(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ float wave_max(float v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmaxf(v, __shfl_xor(v, o));
    return v;
}
__device__ __forceinline__ double wave_sum(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}
__device__ __forceinline__ double wave_max(double v)
{
#pragma unroll
    for (int o = 32; o; o >>= 1) v = fmax(v, __shfl_xor(v, o));
    return v;
}

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? SS_SEQ_OK : SS_SEQ_ELAUNCH; }

}  // namespace
