// Matrix product with its epilogue: y = residual + dropout(act(x W + b)), and the backward pass (dx, dW, db). float32 and float16
// operands, float32 sums; bias and its gradient are float32. A layer of the package's Linear -> Activation -> Dropout -> Add chain
// (Modules/Linear.py:36-54, Activation.py:52-60, Dropout.py:33-72, Add.py:15-26) in one launch instead of five passes.
//
// Every product is C[m][n] = sum_k A(m, k) B(k, n) with A stored [m][k] or [k][m] and B stored [k][n] or [n][k]; the forward pass is
// x W, the backward pass dz W^T and x^T dz with dz = dy * keep / (1 - p) * act'(z) written once by linear_gate_kernel, which also
// leaves the column sums that become db.
#include "philox.h"
#include "rows.h"

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef __fp16 tr16x4 __attribute__((ext_vector_type(4)));

namespace {

// ---- what happens to a finished sum -------------------------------------------------------------------------------------------------
enum { EPI_FORWARD = 0, EPI_ACCUMULATE = 1 };        // y = residual + dropout(act(s + b)) | c = beta * c + alpha * s

struct Epilogue {
	void *out;                       // T, or float32 when out_f32
	void *preact;                    // T: s + b, optional
	const void *residual;            // T, optional
	const float *bias;               // optional
	long ldo, ldp, ldr;              // row pitches in elements
	int m, n;
	int kind, act, dropping, out_f32;
	float alpha, beta, inv_keep;
	int vec;                         // every pitch and base of the tensors above takes runs of COUNT (16 bytes of T, 32 of float32)
	DropKey drop;
};

// COUNT finished sums of a row, whose first is element `index` of the (m, n) tensor; the callers say how runs are loaded and stored
template <int COUNT, typename LoadOld, typename LoadResidual, typename StorePreact, typename StoreOut>
__device__ __forceinline__ void finish(const Epilogue &e, float (&s)[COUNT], const float (&bias)[COUNT], uint64_t index, LoadOld load_old,
                                       LoadResidual load_residual, StorePreact store_preact, StoreOut store_out) {
	if (e.kind == EPI_ACCUMULATE) {
#pragma unroll
		for (int i = 0; i < COUNT; ++i) s[i] *= e.alpha;
		if (e.beta != 0.f) {
			float old[COUNT];
			load_old(old);
#pragma unroll
			for (int i = 0; i < COUNT; ++i) s[i] += e.beta * old[i];
		}
		store_out(s);
		return;
	}
#pragma unroll
	for (int i = 0; i < COUNT; ++i) s[i] += bias[i];
	if (e.preact) store_preact(s);
	with_act(e.act, [&](auto act) {
#pragma unroll
		for (int i = 0; i < COUNT; ++i) s[i] = act_value(s[i], act);
	});
	if (e.dropping) {
		const unsigned bits = drop_bits<COUNT>(e.drop, index);
#pragma unroll
		for (int i = 0; i < COUNT; ++i) s[i] = bits >> i & 1u ? s[i] * e.inv_keep : 0.f;
	}
	if (e.residual) {
		float r[COUNT];
		load_residual(r);
#pragma unroll
		for (int i = 0; i < COUNT; ++i) s[i] += r[i];
	}
	store_out(s);
}

template <int COUNT>
__device__ __forceinline__ void load_bias(const Epilogue &e, int col, float (&bias)[COUNT]) {
#pragma unroll
	for (int i = 0; i < COUNT; ++i) bias[i] = 0.f;
	if (e.kind == EPI_FORWARD && e.bias && col < e.n) load_run(e.bias + col, e.vec && col + COUNT <= e.n, e.n - col, bias);
}

// the run at (row, col), any part of which may lie beyond the matrix
template <typename T, int COUNT>
__device__ __forceinline__ void finish_at(const Epilogue &e, int row, int col, float (&s)[COUNT], const float (&bias)[COUNT]) {
	const int left = e.n - col;
	if (row >= e.m || left <= 0) return;
	const bool whole = e.vec && left >= COUNT;
	const size_t at = (size_t)row * e.ldo + col;
	finish(
	    e, s, bias, (uint64_t)row * e.n + col,
	    [&](float (&v)[COUNT]) { e.out_f32 ? load_run((const float *)e.out + at, whole, left, v) : load_run((const T *)e.out + at, whole, left, v); },
	    [&](float (&v)[COUNT]) { load_run((const T *)e.residual + (size_t)row * e.ldr + col, whole, left, v); },
	    [&](const float (&v)[COUNT]) { store_run((T *)e.preact + (size_t)row * e.ldp + col, whole, left, v); },
	    [&](const float (&v)[COUNT]) { e.out_f32 ? store_run((float *)e.out + at, whole, left, v) : store_run((T *)e.out + at, whole, left, v); });
}

// the runs at (row, col), (row + step, col), ...: all inside, all aligned. Addresses move by additions.
template <typename T, int COUNT>
struct Column {
	char *out;
	T *preact;
	const T *residual;
	long out_step, preact_step, residual_step;
	uint64_t index, index_step;

	__device__ __forceinline__ void init(const Epilogue &e, int row, int col, int step) {
		const int size = e.out_f32 ? 4 : sizeof(T);
		out = (char *)e.out + ((size_t)row * e.ldo + col) * size, out_step = step * e.ldo * size;
		preact = (T *)e.preact + (size_t)row * e.ldp + col, preact_step = step * e.ldp;
		residual = (const T *)e.residual + (size_t)row * e.ldr + col, residual_step = step * e.ldr;
		index = (uint64_t)row * e.n + col, index_step = (uint64_t)step * e.n;
	}

	__device__ __forceinline__ void next(const Epilogue &e, float (&s)[COUNT], const float (&bias)[COUNT]) {
		finish(
		    e, s, bias, index,
		    [&](float (&v)[COUNT]) { e.out_f32 ? load_run((const float *)out, true, COUNT, v) : load_run((const T *)out, true, COUNT, v); },
		    [&](float (&v)[COUNT]) { load_run(residual, true, COUNT, v); }, [&](const float (&v)[COUNT]) { store_run(preact, true, COUNT, v); },
		    [&](const float (&v)[COUNT]) { e.out_f32 ? store_run((float *)out, true, COUNT, v) : store_run((T *)out, true, COUNT, v); });
		out += out_step, preact += preact_step, residual += residual_step, index += index_step;
	}
};

struct Product {
	const void *a, *b;
	float *slabs;                    // partial sums [split][m][slab_n] when splits > 1
	int slab_n;                      // n up to whole runs
	long lda, ldb;
	int reach_a, reach_b;            // stored rows within 32 bits of a tile's start (reach_of)
	int m, n, k;
	int tiles_m, tiles_n, splits, ksteps_per_split;
	size_t a_bytes, b_bytes;         // extents of the operands
	Epilogue epi;
};

// Tiles in groups of kGroup rows of tiles, groups dealt out so that the blocks of one XCD (block id mod 8) work on neighbouring tiles:
// its L2 then holds the few operand strips they share
constexpr int kGroup = 4;

__device__ __forceinline__ void tile_of(const Product &g, int &tm, int &tn) {
	const int tiles = g.tiles_m * g.tiles_n, xcd = blockIdx.x % pz::kNumXCD, at = blockIdx.x / pz::kNumXCD;
	const int each = tiles / pz::kNumXCD, more = tiles % pz::kNumXCD;
	const int id = xcd * each + min(xcd, more) + at;
	const int group = id / (kGroup * g.tiles_n), rest = id % (kGroup * g.tiles_n);
	const int rows = min(kGroup, g.tiles_m - group * kGroup);
	tm = group * kGroup + rest % rows;
	tn = rest / rows;
}

// A wave's accumulators -> rows. The matrix instruction took the operand of the n side first, so a lane holds, of each 16 x 16 tile, 4
// consecutive columns 4 (lane >> 4) of row lane & 15. They go through LDS in slabs of 32 rows (the wave's own, no barrier), so that consecutive lanes store consecutive runs
// of a row: whole 128-byte lines instead of pieces of 16 bytes.
template <typename T, int ROWS, int COLS>
struct Drain {
	static constexpr int COUNT = 16 / sizeof(T);                 // values a lane stores at once
	static constexpr int PITCH = COLS + 4;                       // (+4: the rows of a store start 4 banks apart)
	static constexpr int FLOATS = 32 * PITCH;

	template <int TM, int TN>
	static __device__ __forceinline__ void park(const f32x4 (&acc)[TM][TN], int i, float *lds, int lane) {
#pragma unroll
		for (int h = 0; h < 2; ++h)
#pragma unroll
			for (int j = 0; j < TN; ++j)
				*reinterpret_cast<f32x4 *>(lds + (h * 16 + (lane & 15)) * PITCH + j * 16 + (lane >> 4) * 4) = acc[2 * i + h][j];
	}

	template <typename ACC>
	static __device__ __forceinline__ void run(const Product &g, const ACC &acc, float *lds, int row0, int col0, int split, int lane) {
		constexpr int RUNS = COLS / COUNT, STEP = 64 / RUNS;             // runs in a row, rows a wave handles at once
		static_assert(64 % RUNS == 0, "runs of a row over lanes");
		const int run = lane % RUNS, first = lane / RUNS, col = col0 + run * COUNT;
		const bool inside = g.epi.vec && row0 + ROWS <= g.m && col0 + COLS <= g.n;
		float bias[COUNT];
		load_bias(g.epi, col, bias);
		Column<T, COUNT> column;
		column.init(g.epi, row0 + first, col, STEP);
#pragma unroll
		for (int i = 0; i < ROWS / 32; ++i) {
			park(acc, i, lds, lane);
			__builtin_amdgcn_wave_barrier();
#pragma unroll 2
			for (int r = first; r < 32; r += STEP) {
				float s[COUNT];
#pragma unroll
				for (int v = 0; v < COUNT; v += 4) {
					const f32x4 x = *reinterpret_cast<const f32x4 *>(lds + r * PITCH + run * COUNT + v);
#pragma unroll
					for (int e = 0; e < 4; ++e) s[v + e] = x[e];
				}
				const int row = row0 + i * 32 + r;
				if (g.splits > 1) {
					if (row < g.m && col < g.n) store_run(g.slabs + ((size_t)split * g.m + row) * g.slab_n + col, true, COUNT, s);
				} else if (inside) {
					column.next(g.epi, s, bias);
				} else {
					finish_at<T>(g.epi, row, col, s, bias);
				}
			}
			__builtin_amdgcn_wave_barrier();
		}
	}
};

// ---- the product: operands straight into LDS, v_mfma_f32_16x16x32_f16 or v_mfma_f32_16x16x4_f32 -----------------------------------------
// LDS holds two tiles of 128 bytes of reduction steps (64 float16, 32 float32): of a row whose contiguous axis is k that is one L2 request.
// A wave keeps the n side's fragments of half a tile in registers and walks over its rows, so that a tile's place in LDS frees in pieces:
// the n side and the first half of the m side's rows ("half 0") in the tile's middle, the other rows at its end. What the tile after
// the next one puts there is asked for at once and not needed for one and a half tiles — about 1.5 us, the time a line takes that no L2
// holds. Per-step costs matter as much as waits: 8192 x 8192 x 2048 in float16 runs into the card's power limit (1.9 of 2.4 GHz, the matrix
// pipes busy 60 % of the cycles). 16 x 16 instructions move half the accumulator bytes of 32 x 32 ones and hold a higher clock: 248
// instead of 263 us.
// A fragment is 16 bytes a lane: row lane & 15, steps (lane >> 4) C ... + C - 1 of 4 C, C = 16 / sizeof(T). In float16 that is one matrix
// instruction's operand; in float32 element e feeds the e-th of four instructions, each of which sums the steps 4 q + e — any four will
// do, as long as both operands take the same ones.
template <typename T>
constexpr int kSteps = 128 / sizeof(T);

__device__ __forceinline__ unsigned lds_address(const void *p) {
	return (unsigned)(size_t)(__attribute__((address_space(3))) const void *)p;
}

// 16 bytes per lane from `voff` of the buffer to lds + 16 * lane, no register in between; outside the buffer: zeros. The caller waits
// (vmcnt) before anyone reads them.
__device__ __forceinline__ void dma16(__amdgpu_buffer_rsrc_t rs, unsigned lds, unsigned voff) {
	asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(voff), "s"(rs) : "memory");
}

// all but the last LEFT of this wave's dma16 have landed (they do in order), its LDS reads are back, and so for every wave behind the barrier
template <int LEFT>
__device__ __forceinline__ void meet() {
	asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// ROWS rows of one operand x 128 bytes of steps, staged by WAVES waves: rows row0 + (q / RUN) 2 RUN + half RUN + q mod RUN, q < ROWS — half of
// the rows of every wave, or all rows (RUN = ROWS, half 0). LDS has 64 banks of 4 bytes; a read is spread so that 16 neighbouring lanes
// of a ds_read_b128, 32 of a ds_read_b64 or 64 of a ds_read_b32 touch each bank once.
// KMAJOR = false: [row][k] in memory, so 128 bytes of k per row in LDS, two rows to all banks; the 16-byte pieces of row r stand at
//   piece ^ (r / 2 mod 8), so the fragment's 16 rows at one piece land on 16 different places.
// KMAJOR = true: [k][row] in memory, so a row of ROWS values per k in LDS, in pieces of 16 rows; the pieces of step k stand at
//   piece ^ turn(k). Float16 fragments are read with ds_read_b64_tr_b16, which hands 16 lanes the 4 x 16 block of 4 steps x 16 rows
//   transposed: 32 lanes take one piece of each of 8 steps (k mod 4 and k / 8 mod 2 tell them apart). Float32 fragments are read element
//   by element: 64 lanes take one piece of each of 4 steps (k / 4 mod 4).
template <typename T, int ROWS, int RUN, bool KMAJOR, int WAVES>
struct Stage {
	static constexpr int SIZE = sizeof(T), HK = kSteps<T>, C = 16 / SIZE;
	static constexpr int VALUES = ROWS * HK;
	static constexpr int PIECES = ROWS / 8 / WAVES;            // dma16 per wave and tile
	static_assert(PIECES >= 1 && PIECES * WAVES * 8 == ROWS, "tile / waves");

	__device__ __forceinline__ static int turn(int k) {
		if (SIZE == 4) return k >> 2 & (ROWS == 32 ? 1 : 3);
		return ROWS == 32 ? k >> 3 & 1 : ROWS == 64 ? (k >> 1 & 1) | (k >> 3 & 1) << 1 : (k & 3) | (k >> 3 & 1) << 2;      // (64 rows: two steps to all banks, 32: four)
	}
	__device__ __forceinline__ static int spot(int r) { return r >> 1 & 7; }

	// past every buffer's end: zeros. Of a tile's stored rows the first `reach` lie within 32 bits of its start, the operand's own among
	// them (check_reach); the others, of which a tile of few rows has many, must not wrap onto those.
	static constexpr unsigned NOWHERE = 0xfffffff0u;

	long bytes, step;                // what is left of the operand from the next tile on (negative: nothing); advance per tile
	const char *p;                   // the next tile
	long shift;                      // from half 0 to half 1
	unsigned off[PIECES];            // a lane's byte offsets from there
	int kpiece[PIECES];              // KMAJOR = false: first k of the lane's pieces

	__device__ __forceinline__ void init(const void *src, size_t extent, long ld, int reach, int row0, int kbeg, int wave, int lane) {
		const size_t start = KMAJOR ? ((size_t)kbeg * ld + row0) * SIZE : ((size_t)row0 * ld + kbeg) * SIZE;
		p = (const char *)src + start;
		bytes = (long)(extent - start);
		step = KMAJOR ? HK * ld * SIZE : HK * SIZE;
		shift = KMAJOR ? RUN * SIZE : RUN * ld * SIZE;
		const unsigned pitch = (unsigned)ld * SIZE;
#pragma unroll
		for (int i = 0; i < PIECES; ++i) {
			const int o = ((wave * PIECES + i) * 64 + lane) * 16;                // place in the LDS tile
			if (KMAJOR) {
				const int k = o / (ROWS * SIZE), at = o % (ROWS * SIZE) / 16, q = ((at / SIZE) ^ turn(k)) * 16 + at % SIZE * C;
				off[i] = k < reach ? k * pitch + (q / RUN * (2 * RUN) + q % RUN) * SIZE : NOWHERE;
			} else {
				const int q = o / 128, piece = (o / 16 % 8) ^ spot(q);
				kpiece[i] = piece * C;
				const int row = q / RUN * (2 * RUN) + q % RUN;
				off[i] = row < reach ? row * pitch + piece * 16 : NOWHERE;
			}
		}
	}

	// piece i of k steps [k, k + HK) to LDS address `lds`. Steps from kend on are zeros (or another split's, never multiplied).
	__device__ __forceinline__ void issue(int i, unsigned lds, int k, int kend, int wave, int half) {
		const long left = bytes - half * shift;
		const int high = (int)(left >> 32);                                  // (32-bit tests: they stay in the scalar unit)
		const unsigned span = high > 0 ? 0xfffff000u : high < 0 ? 0u : min((unsigned)left, 0xfffff000u);
		const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void *)(p + half * shift), 0, span, 0x00020000);
		dma16(rs, lds + (wave * PIECES + i) * 1024, KMAJOR || k + kpiece[i] < kend ? off[i] : NOWHERE);
	}

	__device__ __forceinline__ void advance() { p += step, bytes -= step; }

	// fragment s of rows row0 + (lane & 15)
	__device__ __forceinline__ static f32x4 fragment(const T *tile, int row0, int s, int lane) {
		const int j = lane & 15;
		if (!KMAJOR) {
			const int r = row0 + j, piece = s * 4 + (lane >> 4);
			return *reinterpret_cast<const f32x4 *>(tile + r * HK + ((piece ^ spot(r)) * C));
		}
		if (SIZE == 4) {
			f32x4 f;
#pragma unroll
			for (int e = 0; e < 4; ++e) {
				const int k = s * 16 + (lane >> 4) * 4 + e;
				f[e] = (float)tile[k * ROWS + ((row0 / 16) ^ turn(k)) * 16 + j];
			}
			return f;
		}
		// lane j of the 16 that share 8 steps points at step (j >> 2), rows 4 (j & 3) ... + 3 of their 4 x 16 block
		const int k = s * 32 + (lane >> 4) * 8 + (j >> 2);
		union { f32x4 v; tr16x4 h[2]; } f;
#pragma unroll
		for (int half = 0; half < 2; ++half) {
			const int kk = k + half * 4;
			const T *at = tile + kk * ROWS + ((row0 / 16) ^ turn(kk)) * 16 + (j & 3) * 4;
			f.h[half] = __builtin_amdgcn_ds_read_tr16_b64_v4f16((__attribute__((address_space(3))) tr16x4 *)at);
		}
		return f.v;
	}
};

// acc[j] += a b[j]; in float32 the instructions on one accumulator stand N apart
template <typename T, int N>
__device__ __forceinline__ void multiply_add(f32x4 (&acc)[N], const f32x4 &a, const f32x4 (&b)[N]) {
	if (sizeof(T) == 2) {
#pragma unroll
		for (int j = 0; j < N; ++j)
			acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, b[j]), __builtin_bit_cast(f16x8, a), acc[j], 0, 0, 0);
	} else {
#pragma unroll
		for (int e = 0; e < 4; ++e)
#pragma unroll
			for (int j = 0; j < N; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[j][e], a[e], acc[j], 0, 0, 0);
	}
}

// Bound by the matrix pipe: float16 8192 x 8192 x 2048 with dropout and residual 235 us (1170 TFLOP/s), 8192 x 2048 x 8192 with GELU and the
// kept pre-activation 279 us (985; the epilogue writes 268 MB and evaluates 65536 GELUs a CU), float32 4096^3 with ReLU and residual 958 us
// (143 TFLOP/s). Single rows are bound by the weights: 1 x 4096 x 16384 float16 23-25 us (5.4 TB/s), then the join.
template <typename T, int BM, int BN, int WM, int WN, bool TA, bool TB>
__global__ void __launch_bounds__(64 * WM * WN) linear_kernel(Product g) {
	constexpr int HK = kSteps<T>, WAVES = WM * WN, TM = BM / (16 * WM), TN = BN / (16 * WN);
	using SA = Stage<T, BM / 2, BM / WM / 2, TA, WAVES>;            // a half of the rows
	using SB = Stage<T, BN, BN, !TB, WAVES>;
	using Out = Drain<T, BM / WM, BN / WN>;
	constexpr int TILE = 2 * SA::VALUES + SB::VALUES, SLABS = WAVES * Out::FLOATS * 4 / (int)sizeof(T);
	constexpr int NH = SA::PIECES, NB = SB::PIECES;              // dma16 per wave: a half of the m side, the n side
	__shared__ __attribute__((aligned(1024))) T lds[2 * TILE > SLABS ? 2 * TILE : SLABS];

	const int lane = threadIdx.x & 63;
	const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
	const int wm = wave / WN, wn = wave % WN;
	int tm, tn;
	tile_of(g, tm, tn);
	const int m0 = tm * BM, n0 = tn * BN;
	const int split = blockIdx.z;
	const int kbeg = split * g.ksteps_per_split * HK;
	const int kend = min(g.k, kbeg + g.ksteps_per_split * HK);

	f32x4 acc[TM][TN];
#pragma unroll
	for (int i = 0; i < TM; ++i)
#pragma unroll
		for (int j = 0; j < TN; ++j) acc[i][j] = (f32x4){0.f, 0.f, 0.f, 0.f};

	SA sa;
	SB sb;
	sa.init(g.a, g.a_bytes, g.lda, g.reach_a, m0, kbeg, wave, lane);
	sb.init(g.b, g.b_bytes, g.ldb, g.reach_b, n0, kbeg, wave, lane);
	const unsigned at = lds_address(lds);
	auto ask_a = [&](int tile, int half, int i) {
		sa.issue(i, at + ((tile & 1) * TILE + half * SA::VALUES) * (int)sizeof(T), kbeg + tile * HK, kend, wave, half);
		if (half == 1 && i == NH - 1) sa.advance();
	};
	auto ask_b = [&](int tile, int i) {
		sb.issue(i, at + ((tile & 1) * TILE + 2 * SA::VALUES) * (int)sizeof(T), kbeg + tile * HK, kend, wave, 0);
		if (i == NB - 1) sb.advance();
	};
	// a tile is 2 TM steps, TM for each half of the rows: step y multiplies the fragment of 16 rows at one reduction half s with TN fragments
	// of the other operand. The halves s turn back in a half's middle (0 1 1 0, then 1 0 0 1 in the next tile), so that each set of the
	// other operand's fragments is free, and the next one fetched, half a tile's quarter before its use. Each step also issues a share
	// of what else there is to issue; left alone, the scheduler collects that between the steps, where the matrix pipe stands.
	constexpr int STEPS = 2 * TM, AHEAD = 3;
	static_assert(TM % 4 == 0 && TN <= 4, "shares of a step");
	f32x4 av[4], bv[2][TN];
	auto side = [](int odd, int y) { return odd ^ y / TM ^ y % TM / (TM / 2); };
	auto fetch_a = [&](int tile, int odd, int y) {
		av[y % 4] = SA::fragment(lds + (tile & 1) * TILE + y / TM * SA::VALUES, wm * (BM / WM / 2) + y % (TM / 2) * 16, side(odd, y), lane);
	};
	auto fetch_b = [&](int tile, int s, int j) {
		if (j < TN) bv[s][j] = SB::fragment(lds + (tile & 1) * TILE + 2 * SA::VALUES, wn * (BN / WN) + j * 16, s, lane);
	};
	auto multiply = [&](auto parity, int t) {
		constexpr int odd = decltype(parity)::value;
#pragma unroll
		for (int y = 0; y < STEPS; ++y) {
			// behind step TM - 3 every wave has read half 0 and the n side of this tile, and half 1 is there; behind step 2 TM - 3 it has read
			// half 1, and half 0 and the n side of the next tile are there. What was asked for since may still be on its way.
			const bool middle = y >= TM - AHEAD && y < TM, end = y >= STEPS - AHEAD, border = y == TM - AHEAD || y == STEPS - AHEAD;
			auto fetch = [&]() { y + AHEAD < STEPS ? fetch_a(t, odd, y + AHEAD) : fetch_a(t + 1, odd ^ 1, y + AHEAD - STEPS); };
			if (!border) fetch();
			if (y < 2) fetch_b(t, odd ^ 1, 2 * y), fetch_b(t, odd ^ 1, 2 * y + 1);
			const int i = y / TM * (TM / 2) + y % (TM / 2);
			multiply_add<T>(acc[i], av[y % 4], bv[side(odd, y)]);
			if (border) {
				meet<2 * NH + NB>();
				fetch();
			}
			if (end && y < STEPS - 1) {
				const int j = 2 * (y - (STEPS - AHEAD));
				fetch_b(t + 1, odd ^ 1, j), fetch_b(t + 1, odd ^ 1, j + 1);
			}
			if (middle) {
				constexpr int SHARE = (NH + NB + AHEAD - 1) / AHEAD;
				const int from = (y - (TM - AHEAD)) * SHARE;
#pragma unroll
				for (int q = from; q < from + SHARE && q < NH + NB; ++q) q < NH ? ask_a(t + 2, 0, q) : ask_b(t + 2, q - NH);
			}
			if (end) {
				constexpr int SHARE = (NH + AHEAD - 1) / AHEAD;
				const int from = (y - (STEPS - AHEAD)) * SHARE;
#pragma unroll
				for (int q = from; q < from + SHARE && q < NH; ++q) ask_a(t + 2, 1, q);
			}
			__builtin_amdgcn_sched_barrier(0);
		}
	};

	const int tiles = (kend - kbeg + HK - 1) / HK;
#pragma unroll
	for (int t = 0; t < 2; ++t) {
#pragma unroll
		for (int i = 0; i < NH; ++i) ask_a(t, 0, i);
#pragma unroll
		for (int i = 0; i < NB; ++i) ask_b(t, i);
#pragma unroll
		for (int i = 0; i < NH; ++i) ask_a(t, 1, i);
	}
	meet<3 * NH + NB>();
#pragma unroll
	for (int j = 0; j < TN; ++j) fetch_b(0, 0, j);
#pragma unroll
	for (int y = 0; y < AHEAD; ++y) fetch_a(0, 0, y);
	for (int t = 0; t < tiles; t += 2) {
		multiply(std::integral_constant<int, 0>{}, t);
		if (t + 1 < tiles) multiply(std::integral_constant<int, 1>{}, t + 1);
	}
	meet<0>();                       // the slabs below lie over the tiles
	Out::run(g, acc, reinterpret_cast<float *>(lds) + wave * Out::FLOATS, m0 + wm * (BM / WM), n0 + wn * (BN / WN), split, lane);
}

// ---- partial sums of a product split along k, added in order, then the epilogue ------------------------------------------------------
// A launch of its own instead of a last workgroup that waits: the order of the sums is fixed and no counter has to be cleared. Bound by the
// launch (4-6 us at 37 x 4099 and 256 x 2048); the slabs come from the L2s and the memory-side cache.
template <typename T>
__global__ void __launch_bounds__(256) linear_join_kernel(Product g) {
	constexpr int COUNT = 16 / sizeof(T);
	const int runs = g.slab_n / COUNT;
	const size_t idx = (size_t)blockIdx.x * 256 + threadIdx.x, each = (size_t)g.m * g.slab_n;
	if (idx >= (size_t)runs * g.m) return;
	const int row = (int)(idx / runs), col = (int)(idx % runs) * COUNT;
	const float *p = g.slabs + (size_t)row * g.slab_n + col;
	float s[COUNT], bias[COUNT];
	load_bias(g.epi, col, bias);
	load_run(p, true, COUNT, s);
#pragma unroll 4
	for (int i = 1; i < g.splits; ++i) {
		float more[COUNT];
		load_run(p + i * each, true, COUNT, more);
#pragma unroll
		for (int e = 0; e < COUNT; ++e) s[e] += more[e];
	}
	finish_at<T>(g.epi, row, col, s, bias);
}

// ---- operands whose rows do not start on 16 bytes: a copy whose pitch is a multiple of 8 elements, the rest of each row zero -----------
// (the product's loads put 16 bytes a lane straight into LDS and take nothing less; both operands in one launch: 37 x 1001 with 1001 x 4099
// float16 6.6 us, 2.5 TB/s)
struct Aligned {
	const void *src;
	void *dst;                       // null: the operand stays where it is
	int rows, cols, pitch;
	long ld;
};

template <typename T>
__global__ void __launch_bounds__(256) linear_align_kernel(Aligned a, Aligned b, unsigned a_blocks) {
	constexpr int COUNT = 16 / sizeof(T);
	typedef T vec __attribute__((ext_vector_type(COUNT), aligned(sizeof(T))));
	const bool second = blockIdx.x >= a_blocks;
	const Aligned &o = second ? b : a;
	const int runs = o.pitch / COUNT;
	const size_t idx = (size_t)(blockIdx.x - (second ? a_blocks : 0)) * 256 + threadIdx.x;
	if (idx >= (size_t)runs * o.rows) return;
	const int row = (int)(idx / runs), col = (int)(idx % runs) * COUNT;
	const T *p = (const T *)o.src + (size_t)row * o.ld + col;
	float v[COUNT];
	if (col + COUNT <= o.cols) {
		const vec x = *reinterpret_cast<const vec *>(p);                  // (whole elements, no better alignment)
#pragma unroll
		for (int e = 0; e < COUNT; ++e) v[e] = (float)x[e];
	} else {
		load_run(p, false, o.cols - col, v);
	}
	store_run((T *)o.dst + (size_t)row * o.pitch + col, true, COUNT, v);
}

// ---- dz = dy * keep / (1 - p) * act'(z), and partial column sums -----------------------------------------------------------------------
// dz is held in the operands' type, the only one that the matrix instructions of the two products take at their full rate; db sums it before
// that rounding. In float16 it is held as dz * held_part * (1 - p), which dy's own range always has room for: 1 / (1 - p) and an activation's
// slope above 1 would take dz = 65504 / (1 - p) * 1.13 to infinity although dx and dW are in range. The products' sums are multiplied by
// what is missing, in float32. So without a curved activation nothing is rounded (dy or zero), and behind GELU or SiLU dz carries one
// rounding: half a step of 2^-11 relative (8192 x 2048 x 8192 with GELU: dx 2.9e-4 off the 64-bit result, root mean square, where 2.1e-4 is
// the rounding of dx itself), or 2^-25 absolute where it is below 2^-14, as far as dy can be off. A second product with what the rounding
// left would double the pass: 507 us.
float held_part(int dtype, int act) { return dtype == PZ_F16 && (act == PZ_ACT_GELU || act == PZ_ACT_SILU) ? 0.875f : 1.f; }      // (slopes up to 1.13)

struct Gate {
	const void *dy, *preact;
	void *dz;                        // optional: without it only the sums are made
	float *sums;                     // [row blocks][n], optional
	long lddy, ldp, lddz;
	int m, n, act, dropping, vec, rows_per_block;
	float inv_keep, held;            // dz is stored as held * (1 - p) of its value
	DropKey drop;
};

// block = 4 waves x (64 lanes x 16 bytes of columns), rows dealt out over the waves. Once for both products, which read dz several times
// over; bound by its bytes: 8192 x 8192 float16 with GELU 90 us (402 MB, 4.5 TB/s).
template <typename T>
__global__ void __launch_bounds__(256) linear_gate_kernel(Gate g) {
	constexpr int COUNT = 16 / sizeof(T);
	__shared__ float part[4][64][COUNT + 1];
	const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
	const int col = (blockIdx.x * 64 + lane) * COUNT, left = g.n - col;
	const int row0 = blockIdx.y * g.rows_per_block, row1 = min(g.m, row0 + g.rows_per_block);
	float sum[COUNT];
#pragma unroll
	for (int e = 0; e < COUNT; ++e) sum[e] = 0.f;

	if (left > 0) {
		const bool whole = g.vec && left >= COUNT;
		for (int row = row0 + wave; row < row1; row += 4) {
			float d[COUNT];
			load_run((const T *)g.dy + (size_t)row * g.lddy + col, whole, left, d);
			// (the words are drawn while the loads are on their way)
			const unsigned bits = g.dropping ? drop_bits<COUNT>(g.drop, (uint64_t)row * g.n + col) : ~0u;
			if (g.act != PZ_ACT_NONE) {
				float z[COUNT];
				load_run((const T *)g.preact + (size_t)row * g.ldp + col, whole, left, z);
				with_act(g.act, [&](auto act) {
#pragma unroll
					for (int e = 0; e < COUNT; ++e) d[e] *= act_slope<true>(z[e], act);      // (a z beyond its type was stored as an infinity)
				});
			}
			if (g.dropping) {                                            // (last: nothing comes through a dropped element, whatever dy and z hold)
#pragma unroll
				for (int e = 0; e < COUNT; ++e) d[e] = bits >> e & 1u ? d[e] : 0.f;
			}
#pragma unroll
			for (int e = 0; e < COUNT; ++e) sum[e] += d[e], d[e] *= g.held;
			if (g.dz) store_run((T *)g.dz + (size_t)row * g.lddz + col, true, COUNT, d);     // (pitch of 8s: what lies beyond n are the zeros loaded)
		}
	}
	if (!g.sums) return;
#pragma unroll
	for (int e = 0; e < COUNT; ++e) part[wave][lane][e] = sum[e];
	__syncthreads();
	for (int i = threadIdx.x; i < 64 * COUNT; i += 256) {
		const int l = i / COUNT, e = i % COUNT, c = (blockIdx.x * 64 + l) * COUNT + e;
		if (c < g.n) g.sums[(size_t)blockIdx.y * g.n + c] = (part[0][l][e] + part[1][l][e] + part[2][l][e] + part[3][l][e]) * g.inv_keep;
	}
}

// db = beta * db + alpha * (sums of the row blocks, in a fixed order, float64). 64 columns a workgroup, 16 row blocks at a time: 8192
// columns 4.6 us.
__global__ void __launch_bounds__(1024) linear_bias_grad_kernel(const float *__restrict__ sums, int blocks, int n, float *__restrict__ db,
                                                                 float alpha, float beta) {
	__shared__ double part[16][64];
	const int lane = threadIdx.x & 63, row = threadIdx.x >> 6, c = blockIdx.x * 64 + lane;
	double s = 0.0;
	if (c < n)
		for (int i = row; i < blocks; i += 16) s += sums[(size_t)i * n + c];
	part[row][lane] = s;
	__syncthreads();
	if (row > 0 || c >= n) return;
	for (int i = 1; i < 16; ++i) s += part[i][lane];
	db[c] = (beta == 0.f ? 0.f : beta * db[c]) + alpha * (float)s;
}

// ---- host ------------------------------------------------------------------------------------------------------------------------------
constexpr size_t kAlign = 256;
size_t rounded(size_t nbytes) { return (nbytes + kAlign - 1) / kAlign * kAlign; }
int padded(int n) { return (n + 7) / 8 * 8; }

// what a product takes from the workspace: copies of operands that are not aligned, slabs of a split
struct Plan {
	int bm, bn, bk, splits, ksteps_per_split, tiles_m, tiles_n;
	bool copy_a, copy_b;
	size_t a_bytes, b_bytes, slab_bytes;
	size_t bytes() const { return a_bytes + b_bytes + slab_bytes; }
};

struct Operands {
	const void *a, *b;
	long lda, ldb;
	int m, n, k;
	bool ta, tb;
	int wide_a, wide_b;              // readable length of a stored row: its elements, and zeros behind them
};

// 16-byte loads: rows that start on 16 bytes and are whole pieces long
bool aligned(const void *p, long ld, int wide, int size) {
	const int piece = 16 / size;
	return (uintptr_t)p % 16 == 0 && ld % piece == 0 && wide % piece == 0;
}

Plan plan_product(int dtype, const Operands &o) {
	Plan p{};
	if (o.m == 0 || o.n == 0) return p;                                 // (no output, nothing runs)
	const int size = dtype == PZ_F16 ? 2 : 4;
	p.bk = dtype == PZ_F16 ? kSteps<f16> : kSteps<float>;
	p.bm = o.m > 64 ? 128 : 64, p.bn = o.n > 64 ? 128 : 64;
	// narrower tiles where square ones give a CU one workgroup at most (2048^3: float16 33 -> 30 us, float32 147 -> 137; 4096 x 512 x 512
	// 27 -> 13), or half of one where the reduction runs over rows (dW of 2048 x 1024 x 4096: 65 us both ways instead of 69)
	if (p.bm == 128 && (long)pz::ceil_div(o.m, 128) * pz::ceil_div(o.n, 128) <= pz::kNumCU / (o.ta ? 2 : 1)) p.bn = 64;
	const long tiles256 = (long)pz::ceil_div(o.m, 256) * pz::ceil_div(o.n, 256);
	if (o.k >= (dtype == PZ_F16 ? 256 : 1024) && tiles256 >= pz::kNumCU) p.bm = p.bn = 256;
	p.tiles_m = pz::ceil_div(o.m, p.bm), p.tiles_n = pz::ceil_div(o.n, p.bn);
	const long tiles = (long)p.tiles_m * p.tiles_n;
	// k is split until every CU has a workgroup: two each cost more in slabs than they hide (1 x 4096 x 16384 32 against 29 us), and a split
	// keeps four steps of the loop (two, in float16: 46 against 30 us for the backward pass of 256 x 2048 x 1000)
	const int ksteps = pz::ceil_div(o.k, p.bk), least = 4;
	int splits = 1;
	if (tiles < pz::kNumCU) {
		splits = (int)(pz::kNumCU / tiles);
		splits = splits > ksteps / least ? ksteps / least : splits;
		splits = splits < 1 ? 1 : splits > 64 ? 64 : splits;
	}
	p.ksteps_per_split = ksteps > 0 ? pz::ceil_div(ksteps, splits) : 1;
	p.splits = ksteps > 0 ? pz::ceil_div(ksteps, p.ksteps_per_split) : 1;
	p.copy_a = !aligned(o.a, o.lda, o.wide_a, size);
	p.copy_b = !aligned(o.b, o.ldb, o.wide_b, size);
	p.a_bytes = p.copy_a ? rounded((size_t)(o.ta ? o.k : o.m) * padded(o.ta ? o.m : o.k) * size) : 0;
	p.b_bytes = p.copy_b ? rounded((size_t)(o.tb ? o.n : o.k) * padded(o.tb ? o.k : o.n) * size) : 0;
	p.slab_bytes = p.splits > 1 ? rounded((size_t)p.splits * o.m * padded(o.n) * sizeof(float)) : 0;
	return p;
}

template <typename T, bool TA, bool TB>
void launch(const Plan &p, const Product &g, dim3 grid, hipStream_t st) {
	if (p.bm == 256) linear_kernel<T, 256, 256, 2, 4, TA, TB><<<grid, 512, 0, st>>>(g);
	else if (p.bm == 128 && p.bn == 128) linear_kernel<T, 128, 128, 2, 2, TA, TB><<<grid, 256, 0, st>>>(g);
	else if (p.bm == 128) linear_kernel<T, 128, 64, 2, 2, TA, TB><<<grid, 256, 0, st>>>(g);
	else if (p.bn == 128) linear_kernel<T, 64, 128, 1, 4, TA, TB><<<grid, 256, 0, st>>>(g);
	else linear_kernel<T, 64, 64, 1, 1, TA, TB><<<grid, 64, 0, st>>>(g);
}

template <typename T>
void launch(const Plan &p, const Product &g, bool ta, bool tb, dim3 grid, hipStream_t st) {
	if (ta) launch<T, true, false>(p, g, grid, st);
	else if (tb) launch<T, false, true>(p, g, grid, st);
	else launch<T, false, false>(p, g, grid, st);
}

// how many rows of a pitch of ld elements a 32-bit byte offset reaches whole
int reach_of(long ld, int size) {
	const long rows = 0xfffff000l / size / ld;
	return rows < 0x7fffffff ? (int)rows : 0x7fffffff;
}

// a lane's place in a tile is a 32-bit offset from the tile's start: of up to bm rows where k runs along a row, of bk steps elsewhere
int check_reach(int dtype, const Operands &o, const char *who) {
	const Plan p = plan_product(dtype, o);
	auto reach = [&](bool copied, long ld, bool kmajor, int rows, int block) {
		const long held = kmajor ? (o.k < p.bk ? o.k : p.bk) : (rows < block ? rows : block);
		return held <= reach_of(copied ? padded(kmajor ? rows : o.k) : ld, dtype == PZ_F16 ? 2 : 4);
	};
	PZ_REQUIRE(o.m == 0 || o.n == 0 || (reach(p.copy_a, o.lda, o.ta, o.m, p.bm) && reach(p.copy_b, o.ldb, !o.tb, o.n, p.bn)),
	           "%s: rows of %ld and %ld elements are too far apart", who, o.lda, o.ldb);
	return PZ_OK;
}

size_t extent_of(int rows, int wide, long ld, int size) { return rows > 0 ? ((size_t)(rows - 1) * ld + wide) * size : 0; }

// C = epilogue(A B); ws: plan_product(...).bytes()
int product(int dtype, Operands o, const Epilogue &epi, char *ws, hipStream_t st) {
	if (o.m == 0 || o.n == 0) return PZ_OK;
	const Plan p = plan_product(dtype, o);
	const int size = dtype == PZ_F16 ? 2 : 4;
	if (p.copy_a || p.copy_b) {
		Aligned a{o.a, nullptr, 0, 0, 0, o.lda}, b{o.b, nullptr, 0, 0, 0, o.ldb};
		if (p.copy_a) a.dst = ws, a.rows = o.ta ? o.k : o.m, a.cols = o.ta ? o.m : o.k, a.pitch = padded(a.cols), o.a = ws, o.lda = a.pitch;
		if (p.copy_b) b.dst = ws + p.a_bytes, b.rows = o.tb ? o.n : o.k, b.cols = o.tb ? o.k : o.n, b.pitch = padded(b.cols), o.b = b.dst, o.ldb = b.pitch;
		auto blocks = [&](const Aligned &x) { return ((size_t)x.rows * (x.pitch * size / 16) + 255) / 256; };
		const size_t total = blocks(a) + blocks(b);
		PZ_REQUIRE(launchable(total, 256), "linear: an unaligned operand of %d x %d is too large", o.m, o.k);
		if (total > 0) {
			if (dtype == PZ_F16) linear_align_kernel<f16><<<(unsigned)total, 256, 0, st>>>(a, b, (unsigned)blocks(a));
			else linear_align_kernel<float><<<(unsigned)total, 256, 0, st>>>(a, b, (unsigned)blocks(a));
			PZ_LAUNCH_CHECK();
		}
	}

	Product g;
	g.a = o.a, g.b = o.b, g.lda = o.lda, g.ldb = o.ldb, g.reach_a = reach_of(o.lda, size), g.reach_b = reach_of(o.ldb, size);
	g.slabs = (float *)(ws + p.a_bytes + p.b_bytes);
	g.m = o.m, g.n = o.n, g.k = o.k, g.slab_n = padded(o.n);
	g.tiles_m = p.tiles_m, g.tiles_n = p.tiles_n, g.splits = p.splits, g.ksteps_per_split = p.ksteps_per_split;
	g.a_bytes = extent_of(o.ta ? o.k : o.m, p.copy_a ? (int)o.lda : o.wide_a, o.lda, size);
	g.b_bytes = extent_of(o.tb ? o.n : o.k, p.copy_b ? (int)o.ldb : o.wide_b, o.ldb, size);
	g.epi = epi;
	g.epi.m = o.m, g.epi.n = o.n;

	const dim3 grid((unsigned)(p.tiles_m * p.tiles_n), 1, (unsigned)p.splits);
	if (dtype == PZ_F16) launch<f16>(p, g, o.ta, o.tb, grid, st);
	else launch<float>(p, g, o.ta, o.tb, grid, st);
	PZ_LAUNCH_CHECK();
	if (p.splits > 1) {
		const size_t items = (size_t)o.m * (padded(o.n) * size / 16);         // (a split has fewer tiles than the chip has CUs)
		const unsigned blocks = (unsigned)((items + 255) / 256);
		if (dtype == PZ_F16) linear_join_kernel<f16><<<blocks, 256, 0, st>>>(g);
		else linear_join_kernel<float><<<blocks, 256, 0, st>>>(g);
		PZ_LAUNCH_CHECK();
	}
	return PZ_OK;
}

int check_desc(const pz_linear_desc *d, const char *who) {
	PZ_REQUIRE(d, "%s: null descriptor", who);
	PZ_REQUIRE(d->dtype == PZ_F32 || d->dtype == PZ_F16, "%s: unknown dtype %d", who, d->dtype);
	PZ_REQUIRE(d->act >= PZ_ACT_NONE && d->act <= PZ_ACT_SILU, "%s: unknown activation %d", who, d->act);
	PZ_REQUIRE(d->m >= 0 && d->n > 0 && d->k > 0, "%s: bad dimensions (%d, %d, %d)", who, d->m, d->n, d->k);
	// (32-bit indexes run up to two tiles and a workgroup's rows beyond the end)
	PZ_REQUIRE(d->m <= 0x7fffffff - (1 << 17) && d->n < (1 << 28) && d->k < (1 << 28), "%s: dimensions (%d, %d, %d) are too large", who, d->m, d->n, d->k);
	PZ_REQUIRE(d->ldx >= d->k && d->ldw >= (d->trans_w ? d->k : d->n) && d->ldy >= d->n, "%s: row pitch too small", who);
	return PZ_OK;
}

int check_mask(const pz_dropout_mask *mask, const char *who) {
	PZ_REQUIRE(!mask || (mask->keep > 0.f && mask->keep <= 1.f), "%s: keep probability %g", who, mask ? mask->keep : 0.f);
	return PZ_OK;
}

bool runs_ok(const void *p, long ld, int size) { return !p || ((uintptr_t)p % 16 == 0 && ld * size % 16 == 0); }

Operands forward_operands(const pz_linear_desc *d, const void *x, const void *w) {
	return Operands{x, w, d->ldx, d->ldw, d->m, d->n, d->k, false, d->trans_w != 0, d->k, d->trans_w ? d->k : d->n};
}

// the backward pass's workspace: dz (where dy cannot serve itself), row-block sums for db, then what the larger product takes
struct BackPlan {
	bool write_dz;
	int row_blocks, rows_per_block;
	size_t dz_bytes, sum_bytes, product_bytes;
	size_t bytes() const { return dz_bytes + sum_bytes + product_bytes; }
};

Operands data_operands(const pz_linear_desc *d, const void *dz, long lddz, int wide, const void *w) {      // dx[m][k] = dz W^T
	return Operands{dz, w, lddz, d->ldw, d->m, d->k, d->n, false, d->trans_w == 0, wide, d->trans_w ? d->k : d->n};
}

Operands weight_operands(const pz_linear_desc *d, const void *dz, long lddz, int wide, const void *x) {    // dW = x^T dz (or its transpose)
	if (d->trans_w) return Operands{dz, x, lddz, d->ldx, d->n, d->k, d->m, true, false, wide, d->k};
	return Operands{x, dz, d->ldx, lddz, d->k, d->n, d->m, true, false, d->k, wide};
}

BackPlan plan_backward(const pz_linear_desc *d, const void *dy, const void *x, const void *w, bool dropping, bool want_dx, bool want_dw, bool want_db) {
	BackPlan p;
	const int size = d->dtype == PZ_F16 ? 2 : 4;
	p.write_dz = (want_dx || want_dw) && (d->act != PZ_ACT_NONE || dropping || !aligned(dy, d->ldy, d->n, size));
	p.dz_bytes = p.write_dz ? rounded((size_t)d->m * padded(d->n) * size) : 0;
	const int strips = pz::ceil_div(d->n, 1024 / size);                  // (a workgroup takes 1 KiB of columns)
	p.rows_per_block = 128;                                              // fewer rows a block where there are few blocks
	while (p.rows_per_block > 4 && (long)strips * pz::ceil_div(d->m, p.rows_per_block) < 4 * pz::kNumCU) p.rows_per_block /= 2;
	while (pz::ceil_div(d->m, p.rows_per_block) > 65535) p.rows_per_block *= 2;
	p.row_blocks = pz::ceil_div(d->m, p.rows_per_block);
	p.sum_bytes = want_db ? rounded((size_t)p.row_blocks * d->n * sizeof(float)) : 0;
	// (dz in the workspace is aligned: any multiple of 256 stands for its address)
	const void *dz = p.write_dz ? (const void *)kAlign : dy;
	const long lddz = p.write_dz ? padded(d->n) : d->ldy;
	const int wide = p.write_dz ? padded(d->n) : d->n;
	const size_t dx_bytes = want_dx ? plan_product(d->dtype, data_operands(d, dz, lddz, wide, w)).bytes() : 0;
	const size_t dw_bytes = want_dw ? plan_product(d->dtype, weight_operands(d, dz, lddz, wide, x)).bytes() : 0;
	p.product_bytes = dx_bytes > dw_bytes ? dx_bytes : dw_bytes;
	return p;
}

DropKey key_of(const pz_dropout_mask *mask) {
	return mask ? DropKey{mask->seed, mask->call, mask->threshold, mask->keep} : DropKey{0, 0, 0, 1.f};
}

}  // namespace

extern "C" {

int pz_linear_fwd_workspace_bytes(const pz_linear_desc *d, const void *x, const void *w, size_t *nbytes) {
	if (int rc = check_desc(d, "pz_linear_fwd_workspace_bytes")) return rc;
	PZ_REQUIRE(nbytes, "pz_linear_fwd_workspace_bytes: null output");
	*nbytes = d->m > 0 ? plan_product(d->dtype, forward_operands(d, x, w)).bytes() : 0;
	return PZ_OK;
}

int pz_linear_fwd(const pz_linear_desc *d, const void *x, const void *w, const float *bias, const void *residual, const pz_dropout_mask *mask,
                  void *y, void *preact, void *workspace, size_t ws_bytes, pz_stream_t stream) {
	if (int rc = check_desc(d, "pz_linear_fwd")) return rc;
	if (int rc = check_mask(mask, "pz_linear_fwd")) return rc;
	if (!drops(mask)) mask = nullptr;
	if (d->m == 0) return PZ_OK;
	PZ_REQUIRE(x && w && y, "pz_linear_fwd: null tensor");
	PZ_REQUIRE((!residual || d->ldr >= d->n) && (!preact || d->ldp >= d->n), "pz_linear_fwd: row pitch too small");
	const Operands o = forward_operands(d, x, w);
	const size_t need = plan_product(d->dtype, o).bytes();
	if (int rc = check_reach(d->dtype, o, "pz_linear_fwd")) return rc;
	PZ_REQUIRE(need == 0 || (workspace && ws_bytes >= need), "pz_linear_fwd: workspace needs %zu bytes", need);

	const int size = d->dtype == PZ_F16 ? 2 : 4;
	Epilogue e{};
	e.out = y, e.preact = preact, e.residual = residual, e.bias = bias;
	e.ldo = d->ldy, e.ldp = d->ldp, e.ldr = d->ldr;
	e.kind = EPI_FORWARD, e.act = d->act, e.dropping = mask != nullptr, e.alpha = 1.f;
	e.vec = runs_ok(y, d->ldy, size) && runs_ok(preact, d->ldp, size) && runs_ok(residual, d->ldr, size) && runs_ok(bias, 4, 4);
	e.drop = key_of(mask), e.inv_keep = 1.f / e.drop.keep;
	return product(d->dtype, o, e, (char *)workspace, pz::as_stream(stream));
}

int pz_linear_bwd_workspace_bytes(const pz_linear_desc *d, const void *dy, const void *x, const void *w, int dropping, int want_dx, int want_dw,
                                  int want_db, size_t *nbytes) {
	if (int rc = check_desc(d, "pz_linear_bwd_workspace_bytes")) return rc;
	PZ_REQUIRE(nbytes, "pz_linear_bwd_workspace_bytes: null output");
	*nbytes = plan_backward(d, dy, x, w, dropping != 0, want_dx != 0, want_dw != 0, want_db != 0).bytes();
	return PZ_OK;
}

int pz_linear_bwd(const pz_linear_desc *d, const void *dy, const void *x, const void *w, const void *preact, const pz_dropout_mask *mask,
                  void *dx, void *dw, int dw_dtype, float *db, float alpha, float beta, void *workspace, size_t ws_bytes, pz_stream_t stream) {
	if (int rc = check_desc(d, "pz_linear_bwd")) return rc;
	if (int rc = check_mask(mask, "pz_linear_bwd")) return rc;
	if (!drops(mask)) mask = nullptr;
	PZ_REQUIRE(dw_dtype == PZ_F32 || dw_dtype == d->dtype, "pz_linear_bwd: weight gradients are float32 or the operands' type");
	PZ_REQUIRE(d->m == 0 || (dy && (!dx || w) && (!dw || x)), "pz_linear_bwd: null tensor");
	PZ_REQUIRE(d->m == 0 || d->act == PZ_ACT_NONE || (preact && d->ldp >= d->n), "pz_linear_bwd: the activation's gradient needs the pre-activation");
	PZ_REQUIRE(!dx || d->ldr >= d->k, "pz_linear_bwd: row pitch too small");
	const BackPlan p = plan_backward(d, dy, x, w, mask != nullptr, dx != nullptr, dw != nullptr, db != nullptr);
	const size_t need = p.bytes();

	hipStream_t st = pz::as_stream(stream);
	const int size = d->dtype == PZ_F16 ? 2 : 4;
	char *ws = (char *)workspace;
	float *sums = (float *)(ws + p.dz_bytes);
	const void *dz = p.write_dz ? (const void *)ws : dy;
	const long lddz = p.write_dz ? padded(d->n) : d->ldy;
	const int wide = p.write_dz ? padded(d->n) : d->n;
	const float held = held_part(d->dtype, d->act), inv_keep = mask ? 1.f / mask->keep : 1.f;
	const Operands data = data_operands(d, dz, lddz, wide, w), weight = weight_operands(d, dz, lddz, wide, x);
	if (int rc = dx ? check_reach(d->dtype, data, "pz_linear_bwd") : PZ_OK) return rc;
	if (int rc = dw ? check_reach(d->dtype, weight, "pz_linear_bwd") : PZ_OK) return rc;
	PZ_REQUIRE(need == 0 || (workspace && ws_bytes >= need), "pz_linear_bwd: workspace needs %zu bytes", need);

	if (d->m > 0 && (p.write_dz || db)) {
		Gate g{};
		g.dy = dy, g.preact = preact, g.dz = p.write_dz ? ws : nullptr, g.sums = db ? sums : nullptr;
		g.lddy = d->ldy, g.ldp = d->ldp, g.lddz = lddz;
		g.m = d->m, g.n = d->n, g.act = d->act, g.dropping = mask != nullptr, g.rows_per_block = p.rows_per_block;
		g.vec = runs_ok(dy, d->ldy, size) && (d->act == PZ_ACT_NONE || runs_ok(preact, d->ldp, size));
		g.drop = key_of(mask), g.inv_keep = inv_keep, g.held = held;
		const dim3 grid((unsigned)pz::ceil_div(d->n, 1024 / size), (unsigned)p.row_blocks);
		if (d->dtype == PZ_F16) linear_gate_kernel<f16><<<grid, 256, 0, st>>>(g);
		else linear_gate_kernel<float><<<grid, 256, 0, st>>>(g);
		PZ_LAUNCH_CHECK();
	}
	if (db) {
		linear_bias_grad_kernel<<<pz::ceil_div(d->n, 64), 1024, 0, st>>>(sums, p.row_blocks, d->n, db, alpha, beta);
		PZ_LAUNCH_CHECK();
	}
	ws += p.dz_bytes + p.sum_bytes;
	if (dx) {
		Epilogue e{};
		e.out = dx, e.ldo = d->ldr, e.kind = EPI_ACCUMULATE, e.alpha = inv_keep / held, e.vec = runs_ok(dx, d->ldr, size);
		if (int rc = product(d->dtype, data, e, ws, st)) return rc;
	}
	if (dw) {
		Epilogue e{};
		e.out = dw, e.ldo = d->trans_w ? d->k : d->n, e.kind = EPI_ACCUMULATE, e.alpha = alpha * (inv_keep / held), e.beta = beta, e.out_f32 = dw_dtype == PZ_F32;
		e.vec = runs_ok(dw, e.ldo, e.out_f32 ? 4 : 2) && (!e.out_f32 || e.ldo % (16 / size) == 0);
		if (int rc = product(d->dtype, weight, e, ws, st)) return rc;
	}
	return PZ_OK;
}

}  // extern "C"
