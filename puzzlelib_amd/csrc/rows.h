// Shared by the operators over rows of channels (linear.hip, dropout.hip, groupnorm.hip): float32 / float16 runs of a row held as
// float32 in registers, and the activations fused into them.
#pragma once
#include "common.h"

#include <type_traits>

typedef _Float16 f16;

namespace {

// a launch has fewer than 2^32 threads
inline bool launchable(size_t blocks, unsigned threads) { return blocks < (1ull << 32) / threads; }

// ---- activations, their derivatives: values in float32 ---------------------------------------------------------------------------
__device__ __forceinline__ float exp_of(float x) { return __builtin_amdgcn_exp2f(x * 1.44269504088896341f); }

// The normal distribution's tail, Phi(-a) for a >= 0, with e = exp(-a^2 / 2): e * R(a), where R(a) = erfcx(a / sqrt 2) / 2 is smooth and
// falls like 1 / a, so that a polynomial in t = 1 / (1 + 0.3 a) holds it. The coefficients are a least-maximum fit of the relative error
// over 0 <= a <= 13 (1.2e-7; beyond, e vanishes in float32). 18 instructions and no branch, where erff takes both of its branches in a
// wave: an epilogue of 65536 values a CU is not hidden behind anything.
__device__ __forceinline__ float normal_tail(float a, float e) {
	const float t = __builtin_amdgcn_rcpf(fmaf(0.3f, a, 1.f));
	float r = 0.0361948135f;
	r = fmaf(r, t, -0.15937814f);
	r = fmaf(r, t, 0.21011811f);
	r = fmaf(r, t, -0.0571671165f);
	r = fmaf(r, t, 0.130416329f);
	r = fmaf(r, t, 0.0993471597f);
	r = fmaf(r, t, 0.120845525f);
	r = fmaf(r, t, 0.119623263f);
	return r * t * e;
}

__device__ __forceinline__ float act_value(float z, int act) {
	if (act == PZ_ACT_RELU) return z < 0.f ? 0.f : z;                                   // (NaN stays NaN)
	if (act == PZ_ACT_GELU) {
		const float q = normal_tail(fabsf(z), exp_of(-0.5f * z * z));
		return z * (z < 0.f ? q : 1.f - q);
	}
	if (act == PZ_ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + exp_of(-z));
	return z;
}

// INF: z may be infinite, where the slopes are 0 and 1 and z times nothing is not; from 100 on they are that in float32. (The median forgets a
// NaN, the exponential beside it does not.)
template <bool INF = false>
__device__ __forceinline__ float act_slope(float z, int act) {
	const float f = INF ? __builtin_amdgcn_fmed3f(z, -100.f, 100.f) : z;
	if (act == PZ_ACT_RELU) return z > 0.f ? 1.f : 0.f;
	if (act == PZ_ACT_GELU) {
		const float e = exp_of(-0.5f * z * z), q = normal_tail(fabsf(z), e);
		return fmaf(f * 0.39894228040143268f, e, z < 0.f ? q : 1.f - q);
	}
	if (act == PZ_ACT_SILU) {
		const float s = __builtin_amdgcn_rcpf(1.f + exp_of(-z));
		return s * fmaf(f, 1.f - s, 1.f);
	}
	return 1.f;
}

// f(activation as a constant): the choice once in front of a loop. Left inside, a branch per value keeps the values' chains from overlapping (group norm
// backward, 64 x 1024 x 512 float16 with SiLU: 80 instead of 71 us; linear 8192 x 2048 x 8192 with GELU 320 instead of 306).
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
	if (act == PZ_ACT_NONE) f(std::integral_constant<int, PZ_ACT_NONE>{});
	else if (act == PZ_ACT_RELU) f(std::integral_constant<int, PZ_ACT_RELU>{});
	else if (act == PZ_ACT_GELU) f(std::integral_constant<int, PZ_ACT_GELU>{});
	else f(std::integral_constant<int, PZ_ACT_SILU>{});
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
