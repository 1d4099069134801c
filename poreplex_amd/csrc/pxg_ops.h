// pxg_ops.h -- what the operators on the caller's device memory share (k_decay*.hip, k_distill.hip): the three element
// types and their conversions.  Unlike the signal path these sources are compiled with fused multiply-adds where the
// compiler sees them: their results are held to an error, not to bits.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>
#include "../../include/pxg.h"

typedef __bf16 pxg_bf16;
typedef _Float16 pxg_f16;
typedef float pxg_f32x4 __attribute__((ext_vector_type(4)));

template <typename T> __device__ __forceinline__ float pxg_to_f32(T x) { return (float)x; }
template <typename T> __device__ __forceinline__ T pxg_from_f32(float x) { return (T)x; }       // round to nearest even
