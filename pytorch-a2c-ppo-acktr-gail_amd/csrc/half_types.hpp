// Element types of the mixed-precision operators (linear_act.hip, gated_scan.hip, adamw.hip): bf16, fp16 and fp32 storage, fp32
// arithmetic.  A conversion to 16 bits rounds to nearest even.
#pragma once
#include "common.hpp"
#include "../../include/acktr_hip.h"

namespace acktr {

typedef float f32v4 __attribute__((ext_vector_type(4)));

template <class T, int N>
struct VecOf { typedef T type __attribute__((ext_vector_type(N))); };
template <class T, int N>
using vec_t = typename VecOf<T, N>::type;
// the same in memory at any element's address: one wide access, which the hardware splits where it has to
template <class T, int N>
struct UnalignedVecOf { typedef T type __attribute__((ext_vector_type(N), aligned(sizeof(T)))); };
template <class T, int N>
using uvec_t = typename UnalignedVecOf<T, N>::type;

template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }

static inline long elem_bytes(int dtype) { return dtype == ACKTR_F32 ? 4 : 2; }
static inline bool dtype_ok(int dtype) { return dtype == ACKTR_F32 || dtype == ACKTR_BF16 || dtype == ACKTR_F16; }

// calls f(T{}) with the element type of a dtype code
template <class F>
static inline auto with_dtype(int dtype, F&& f) {
    if (dtype == ACKTR_BF16) return f(__bf16{});
    if (dtype == ACKTR_F16) return f(_Float16{});
    return f(float{});
}

}  // namespace acktr
