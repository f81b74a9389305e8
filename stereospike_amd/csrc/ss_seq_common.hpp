// ss_seq_common.hpp — shared device helpers of the ss_seq_*.hip units (sequence operators).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include <math.h>
#include <type_traits>

#include "ss_sequence.h"

namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
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

// Over the 64 lanes, by every lane: within rows of 16 by DPP (no LDS pipe), the four rows by reading a lane of each.
template <int CTRL> __device__ __forceinline__ float dpp(float v) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false)); }
template <int CTRL> __device__ __forceinline__ double dpp(double v)
{
    return __hiloint2double(__builtin_amdgcn_update_dpp(0, __double2hiint(v), CTRL, 0xF, 0xF, false), __builtin_amdgcn_update_dpp(0, __double2loint(v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float lane_of(float v, int l) { return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), l)); }
__device__ __forceinline__ double lane_of(double v, int l) { return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(v), l), __builtin_amdgcn_readlane(__double2loint(v), l)); }
template <typename V, typename F> __device__ __forceinline__ V wave_reduce(V v, F&& f)
{
    v = f(v, dpp<0xB1>(v));                                // quad_perm 1 0 3 2
    v = f(v, dpp<0x4E>(v));                                // quad_perm 2 3 0 1
    v = f(v, dpp<0x141>(v));                               // row_half_mirror
    v = f(v, dpp<0x140>(v));                               // row_mirror
    return f(f(lane_of(v, 0), lane_of(v, 16)), f(lane_of(v, 32), lane_of(v, 48)));
}
template <typename V> __device__ __forceinline__ V wave_sum(V v) { return wave_reduce(v, [](V x, V y) { return x + y; }); }
template <typename V> __device__ __forceinline__ V wave_max(V v) { return wave_reduce(v, [](V x, V y) { return x > y ? x : y; }); }

inline bool aligned(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }
inline int launched() { return hipGetLastError() == hipSuccess ? SS_SEQ_OK : SS_SEQ_ELAUNCH; }

}  // namespace
