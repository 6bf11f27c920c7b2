// Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy as 1, 2, 3", 2011): words of a counter under a key. Word i of
// call #k of a generator is philox(key = seed, counter = {i / 4, k})[i % 4] — a fill (rng.hip) writes them, a dropout whose mask is
// never stored (dropout.hip, linear.hip) evaluates the very same words where it needs them.
#pragma once
#include "common.h"

__device__ __forceinline__ uint4 philox4x32_10(uint4 ctr, uint2 key) {
	constexpr uint32_t M0 = 0xD2511F53u, M1 = 0xCD9E8D57u, W0 = 0x9E3779B9u, W1 = 0xBB67AE85u;
#pragma unroll
	for (int r = 0; r < 10; ++r) {
		const uint32_t hi0 = __umulhi(M0, ctr.x), lo0 = M0 * ctr.x;
		const uint32_t hi1 = __umulhi(M1, ctr.z), lo1 = M1 * ctr.z;
		ctr = make_uint4(hi1 ^ ctr.y ^ key.x, lo1, hi0 ^ ctr.w ^ key.y, lo0);
		key.x += W0;
		key.y += W1;
	}
	return ctr;
}

// The mask of a dropout by its key: element i is kept where word i < threshold, and kept elements are divided by `keep`
struct DropKey {
	uint64_t seed, call;
	uint32_t threshold;
	float keep;
};

// A mask of p = 0 keeps everything and is no mask at all: below its threshold of 2^32 - 1 every word lies but one
inline bool drops(const pz_dropout_mask *mask) { return mask && !(mask->threshold == 0xffffffffu && mask->keep == 1.f); }

// words of elements 4 * quad ... 4 * quad + 3
__device__ __forceinline__ uint4 drop_words(const DropKey &d, uint64_t quad) {
	return philox4x32_10(make_uint4((uint32_t)quad, (uint32_t)(quad >> 32), (uint32_t)d.call, (uint32_t)(d.call >> 32)),
	                     make_uint2((uint32_t)d.seed, (uint32_t)(d.seed >> 32)));
}

// bit e: element `first + e` is kept, e < COUNT (a multiple of 4). A first element inside a quad takes one evaluation more.
template <int COUNT>
__device__ __forceinline__ unsigned drop_bits(const DropKey &d, uint64_t first) {
	const unsigned skip = (unsigned)(first & 3);
	uint64_t bits = 0;
#pragma unroll
	for (int q = 0; q < COUNT / 4; ++q) {
		const uint4 w = drop_words(d, (first >> 2) + q);
		bits |= (uint64_t)((w.x < d.threshold ? 1u : 0u) | (w.y < d.threshold ? 2u : 0u) | (w.z < d.threshold ? 4u : 0u) |
		                   (w.w < d.threshold ? 8u : 0u)) << (4 * q);
	}
	if (skip) {
		const uint4 w = drop_words(d, (first >> 2) + COUNT / 4);
		bits |= (uint64_t)((w.x < d.threshold ? 1u : 0u) | (w.y < d.threshold ? 2u : 0u) | (w.z < d.threshold ? 4u : 0u) |
		                   (w.w < d.threshold ? 8u : 0u)) << COUNT;
	}
	return (unsigned)(bits >> skip);
}
