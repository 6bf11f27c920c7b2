// Dropout whose mask is computed, never stored: y = residual + x * keep / (1 - p), element i kept by word i of a counter-based generator
// (philox.h). The forward and the backward pass are the same call with the same key: 2 bytes in, 2 out per float16 element, where the
// stored form (rng.hip's fill, then PZ_OP_DROPOUT) moves 4 + 4 bytes of words per element besides.
#include "philox.h"
#include "rows.h"

namespace {

// 16 bytes of T a lane: COUNT consecutive elements, so a lane evaluates whole quads of the generator. Bound by memory: 8192 x 8192 float16
// with a residual 70 us (402 MB, 5.7 TB/s); 256 x 1024 float32 2.5 us, the launch.
template <typename T>
__global__ void __launch_bounds__(256) dropout_kernel(const T *x, const T *residual, T *y, size_t count, DropKey key, int dropping, int vec) {
	constexpr int COUNT = 16 / sizeof(T);
	const size_t first = ((size_t)blockIdx.x * 256 + threadIdx.x) * COUNT;
	if (first >= count) return;
	const int left = count - first < COUNT ? (int)(count - first) : COUNT;
	const bool whole = vec && left == COUNT;
	const unsigned bits = dropping ? drop_bits<COUNT>(key, first) : ~0u;
	float v[COUNT];
	load_run(x + first, whole, left, v);
#pragma unroll
	for (int e = 0; e < COUNT; ++e) v[e] = bits >> e & 1u ? v[e] / key.keep : 0.f;
	if (residual) {
		float r[COUNT];
		load_run(residual + first, whole, left, r);
#pragma unroll
		for (int e = 0; e < COUNT; ++e) v[e] += r[e];
	}
	store_run(y + first, whole, left, v);
}

template <typename T>
int run(const void *x, const void *residual, void *y, size_t count, const pz_dropout_mask *mask, hipStream_t st) {
	constexpr int COUNT = 16 / sizeof(T);
	const int vec = (((uintptr_t)x | (uintptr_t)residual | (uintptr_t)y) & 15) == 0;
	const size_t blocks = (count + 256 * COUNT - 1) / (256 * COUNT);
	PZ_REQUIRE(launchable(blocks, 256), "pz_dropout: %zu elements are too many", count);
	dropout_kernel<T><<<(unsigned)blocks, 256, 0, st>>>((const T *)x, (const T *)residual, (T *)y, count,
	                                                    DropKey{mask->seed, mask->call, mask->threshold, mask->keep}, drops(mask), vec);
	PZ_LAUNCH_CHECK();
	return PZ_OK;
}

}  // namespace

extern "C" int pz_dropout(int dtype, const void *x, const void *residual, void *y, size_t count, const pz_dropout_mask *mask, pz_stream_t stream) {
	PZ_REQUIRE(dtype == PZ_F32 || dtype == PZ_F16, "pz_dropout: unknown dtype %d", dtype);
	PZ_REQUIRE(mask && mask->keep > 0.f && mask->keep <= 1.f, "pz_dropout: a mask with a keep probability in (0, 1]");
	if (count == 0) return PZ_OK;
	PZ_REQUIRE(x && y, "pz_dropout: null tensor");
	return dtype == PZ_F16 ? run<f16>(x, residual, y, count, mask, pz::as_stream(stream)) : run<float>(x, residual, y, count, mask, pz::as_stream(stream));
}
