// Shared by the operators over rows of channels (linear.hip, dropout.hip, groupnorm.hip): float32 / float16 runs of a row held as
// float32 in registers, and the activations fused into them.
#pragma once
#include "common.h"

typedef _Float16 f16;

namespace {

// ---- activations, their derivatives: values in float32 ---------------------------------------------------------------------------
__device__ __forceinline__ float act_value(float z, int act) {
	if (act == PZ_ACT_RELU) return z < 0.f ? 0.f : z;                                   // (NaN stays NaN)
	if (act == PZ_ACT_GELU) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
	if (act == PZ_ACT_SILU) return z / (1.f + expf(-z));
	return z;
}

__device__ __forceinline__ float act_slope(float z, int act) {
	if (act == PZ_ACT_RELU) return z > 0.f ? 1.f : 0.f;
	if (act == PZ_ACT_GELU) return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * expf(-0.5f * z * z);
	if (act == PZ_ACT_SILU) {
		const float s = 1.f / (1.f + expf(-z));
		return s * (1.f + z * (1.f - s));
	}
	return 1.f;
}

// ---- COUNT consecutive values of a row, float32 in registers ----------------------------------------------------------------------
// `whole`: all COUNT of them exist and the address is a multiple of 16 bytes; else the first `left` one by one
template <typename T, int COUNT>
__device__ __forceinline__ void load_run(const T *p, bool whole, int left, float (&v)[COUNT]) {
	if (whole) {
		typedef T vec __attribute__((ext_vector_type(COUNT)));
		const vec x = *reinterpret_cast<const vec *>(p);
#pragma unroll
		for (int e = 0; e < COUNT; ++e) v[e] = (float)x[e];
	} else {
#pragma unroll
		for (int e = 0; e < COUNT; ++e) v[e] = e < left ? (float)p[e] : 0.f;
	}
}

template <typename T, int COUNT>
__device__ __forceinline__ void store_run(T *p, bool whole, int left, const float (&v)[COUNT]) {
	if (whole) {
		typedef T vec __attribute__((ext_vector_type(COUNT)));
		vec x;
#pragma unroll
		for (int e = 0; e < COUNT; ++e) x[e] = (T)v[e];
		*reinterpret_cast<vec *>(p) = x;
	} else {
#pragma unroll
		for (int e = 0; e < COUNT; ++e)
			if (e < left) p[e] = (T)v[e];
	}
}

}  // namespace
