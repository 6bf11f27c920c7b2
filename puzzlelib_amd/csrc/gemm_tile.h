// The operand loader of the fp32 matrix products (gemm.hip, linear.hip): one tile of rows x BK reduction steps, through registers
// into LDS, reduction-major.
#pragma once
#include "common.h"

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

namespace {

constexpr int BK = 16;
constexpr unsigned kOOB = 0xfffffff0u;      // buffer-load byte offset beyond every matrix: the hardware returns 0

// Loads one operand tile (ROWS x BK, ROWS = BM or BN) into registers and parks it in LDS as [k][row].
// KMAJOR: the source is stored [k][row] (row contiguous); else [row][k] (k contiguous). VEC: 16-byte buffer loads. PAD: the row stride
// in LDS is ROWS + PAD floats.
template <int NT, int ROWS, bool KMAJOR, bool VEC, int BK = ::BK, int PAD = 32>
struct Loader {
	static constexpr int LD = ROWS + PAD;
	static constexpr int NV = ROWS * BK / 4 / NT;             // float4 per thread per tile
	static_assert(NV >= 1 && NV * NT * 4 == ROWS * BK, "operand tile / thread count");
	f32x4 reg[NV];
	unsigned voff[NV];               // VEC: byte offset of this thread's quad in k-tile 0 of the launch (kOOB: row outside)
	int kq[NV];                      // VEC: its first k inside a k-tile

	__device__ __forceinline__ void init(int ld, int row0, int nrows, int kbeg, int tid) {
		if (!VEC) return;
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			const int v = tid + NT * i;
			int r, k;
			if (KMAJOR) { r = (v % (ROWS / 4)) * 4, k = v / (ROWS / 4); }
			else        { r = v % ROWS, k = (v / ROWS) * 4; }
			const int gr = row0 + r;
			kq[i] = k;
			// a quad that starts inside the matrix and runs over its edge (KMAJOR, rows not a multiple of 4) reads the next
			// k-row's first elements or zeros beyond the descriptor: rows >= nrows only meet outputs that are not stored
			const size_t e = KMAJOR ? (size_t)(kbeg + k) * ld + gr : (size_t)gr * ld + kbeg + k;
			voff[i] = gr < nrows ? (unsigned)(e * 4) : kOOB;
		}
	}

	__device__ __forceinline__ void load(const float *__restrict__ src, __amdgpu_buffer_rsrc_t rs, int ld, int row0, int nrows, int k0,
	                                     int kend, int tid) {
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			if (VEC) {
				const unsigned vo = k0 + kq[i] < kend ? voff[i] : kOOB;
				reg[i] = __builtin_bit_cast(f32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, vo, 0, 0));
				voff[i] += KMAJOR ? (unsigned)(BK * ld) * 4u : (unsigned)BK * 4u;      // (kOOB stays beyond every matrix < 4 GiB - 64 K)
				continue;
			}
			const int v = tid + NT * i;
			int r, k;
			if (KMAJOR) { r = (v % (ROWS / 4)) * 4, k = v / (ROWS / 4); }       // 4 consecutive rows of one k
			else        { r = v % ROWS, k = (v / ROWS) * 4; }                     // 4 consecutive k of one row
			const int gr = row0 + r, gk = k0 + k;
			f32x4 x = {0.f, 0.f, 0.f, 0.f};
			if (KMAJOR) {
				if (gk < kend) {
					const float *p = src + (size_t)gk * ld + gr;
#pragma unroll
					for (int e = 0; e < 4; ++e) if (gr + e < nrows) x[e] = p[e];
				}
			} else {
				if (gr < nrows) {
					const float *p = src + (size_t)gr * ld + gk;
#pragma unroll
					for (int e = 0; e < 4; ++e) if (gk + e < kend) x[e] = p[e];
				}
			}
			reg[i] = x;
		}
	}

	__device__ __forceinline__ void park(float *lds, int tid) const {
#pragma unroll
		for (int i = 0; i < NV; ++i) {
			const int v = tid + NT * i;
			if (KMAJOR) {
				const int r = (v % (ROWS / 4)) * 4, k = v / (ROWS / 4);
				*reinterpret_cast<f32x4 *>(&lds[k * LD + r]) = reg[i];
			} else {
				const int r = v % ROWS, k = (v / ROWS) * 4;
#pragma unroll
				for (int e = 0; e < 4; ++e) lds[(k + e) * LD + r] = reg[i][e];
			}
		}
	}
};

}  // namespace
