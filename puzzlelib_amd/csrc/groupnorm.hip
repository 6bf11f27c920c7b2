// Group normalisation with an activation, channels last: y = act(scale * (x - mean) * invvar + bias) over the pixels and channels of a
// group of a sample, and its backward pass. With m values to a group, xhat = (x - mean) * invvar and da = dy * act'(scale * xhat + bias):
//   dbias = sum da, dscale = sum da * xhat over samples and pixels;  dx = invvar * (scale * da - (A + xhat * B) / m)
//   with A = sum scale * da and B = sum scale * da * xhat over the group.
// Statistics are float32, the variance is that of the centred values (no difference of large squares).
#include "rows.h"

namespace {

struct Norm {
	const void *x, *dy;
	void *out;                       // y, or dx
	const float *scale, *bias;
	float *mean, *invvar;            // written forward (optional), read backward
	float *dscale, *dbias;
	int n, pixels, c, groups, width;
	int act;
	float epsilon;
};

__device__ __forceinline__ float or_else(const float *p, int i, float v) { return p ? p[i] : v; }

// ---- where the values of a workgroup lie ----------------------------------------------------------------------------------------------
// A workgroup holds `rows` rows of `width` consecutive values, `pitch` apart, as 16-byte vectors in registers: thread (tx, ty) the
// vectors at tx * V of the rows ty, ty + TY, ... — its channels never change, so scale, bias and statistics are fetched once. Either
//  - a row is a pixel's slab of channels (whole groups, at least a cache line where the shape gives one), pitch c; or
//  - the pixels lie back to back: a row is lcm(c, V) values (`reps` pixels), whatever c is; the last row may end early.
struct Slab {
	int width, tx, ty, reps, slabs, uniform;     // uniform: every vector lies inside one group
	int pitch;
	int rows, last_rows;                         // of a chunk, of the last one
	int last_values;                             // values of the last chunk (the last row may end early)
	float count, last_count;                     // values of a group in a chunk, in the last one
	int chunks;
	int sharing;                                 // slabs that share cache lines: workgroups b, b + 8, ... (one XCD, hence one L2) take them
	int wd, period;                              // values of a group and of all channels in a row's cells (below)
};

template <typename T>
struct Vec {
	static constexpr int V = 16 / sizeof(T);
	typedef T raw __attribute__((ext_vector_type(V), aligned(sizeof(T))));       // (any alignment of whole elements)
};

template <typename T>
__device__ __forceinline__ typename Vec<T>::raw load_vec(const T *p, int left) {
	constexpr int V = Vec<T>::V;
	typename Vec<T>::raw v;
	if (left >= V) return *reinterpret_cast<const typename Vec<T>::raw *>(p);
#pragma unroll
	for (int e = 0; e < V; ++e) v[e] = e < left ? p[e] : (T)0.f;
	return v;
}

template <typename T>
__device__ __forceinline__ void store_vec(T *p, int left, const float (&v)[Vec<T>::V]) {
	constexpr int V = Vec<T>::V;
	if (left >= V) {
		typename Vec<T>::raw x;
#pragma unroll
		for (int e = 0; e < V; ++e) x[e] = (T)v[e];
		*reinterpret_cast<typename Vec<T>::raw *>(p) = x;
	} else {
#pragma unroll
		for (int e = 0; e < V; ++e)
			if (e < left) p[e] = (T)v[e];
	}
}

// The vectors of a thread: rows ty, ty + TY, ...: `mine` of them, the last one with `last` values (V unless the data ends inside it).
// All arithmetic on the shape is 32-bit, its divisions the host's: 64-bit ones (150 instructions each) took most of a small call's time.
template <int V>
__device__ __forceinline__ void share(const Slab &s, int chunk, int tx, int ty, int most, int &mine, int &last) {
	const bool ends = chunk == s.chunks - 1;
	const int rows = ends ? s.last_rows : s.rows;
	mine = ty < min(s.ty, rows) ? min(most, (rows - ty + s.ty - 1) / s.ty) : 0;
	last = V;
	if (ends && mine > 0 && s.slabs == 1) {
		const int left = s.last_values - (ty + (mine - 1) * s.ty) * s.pitch - tx * V;
		if (left <= 0) mine -= 1;                    // (only the last row ends early: the one before it is whole)
		else if (left < V) last = left;
	}
}

// the workgroup's slab, chunk and sample
__device__ __forceinline__ void place(const Slab &s, int &slab, int &chunk, long &sample) {
	const unsigned item = (blockIdx.x / (8 * s.sharing) * 8 + blockIdx.x % 8) * s.sharing + blockIdx.x / 8 % s.sharing, rest = item / s.slabs;
	slab = item - rest * s.slabs;
	const unsigned at = rest / s.chunks;
	chunk = rest - at * s.chunks, sample = at;
}

// Sums of cells in LDS: red[row * across + cell], `rows` rows; output o takes the cells rep * period + o * wd ... + wd - 1, rep < reps, of
// every row. Each output is added by up to 64 lanes in a fixed order; out[o] = sum * factor. All threads call it; the caller has synchronised.
template <int NT>
__device__ void sum_cells(const float *red, int across, int rows, int reps, int period, int wd, int outputs, float factor, float *out) {
	int shift = 6;
	while (shift > 0 && (outputs << shift) > NT) --shift;
	const int lanes = 1 << shift, sub = threadIdx.x & (lanes - 1);
	for (int o0 = 0; o0 < outputs; o0 += NT >> shift) {
		const int o = o0 + (threadIdx.x >> shift);
		float s = 0.f;
		if (o < outputs) {
			const float *p = red + o * wd;
			if (rows > 1) {
				for (int r = sub; r < rows; r += lanes)
					for (int rep = 0; rep < reps; ++rep)
						for (int i = 0; i < wd; ++i) s += p[r * across + rep * period + i];
			} else {
				for (int rep = 0; rep < reps; ++rep)
					for (int i = sub; i < wd; i += lanes) s += p[rep * period + i];
			}
		}
		for (int l = lanes >> 1; l > 0; l >>= 1) s += __shfl_xor(s, l, 64);
		if (o < outputs && sub == 0) out[o] = s * factor;
	}
}

// scale or bias (`none` where there is none) of V channels from `first` on
template <int V>
__device__ __forceinline__ void load_floats(const float *p, int first, float none, float (&v)[V]) {
	typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
#pragma unroll
	for (int q = 0; q < V; q += 4) {
		const vec x = p ? *reinterpret_cast<const vec *>(p + first + q) : (vec){none, none, none, none};
#pragma unroll
		for (int e = 0; e < 4; ++e) v[q + e] = x[e];
	}
}

// channel and group (inside the slab) of the V values of a vector, f(e, channel, group); UNI: one group, no pixel border inside
template <int V, bool UNI, typename F>
__device__ __forceinline__ void each_channel(int first, int c, int width, F f) {
	if (UNI) {
		const int group = first / width;
#pragma unroll
		for (int e = 0; e < V; ++e) f(e, first + e, group);
	} else {
		int ch = first % c, group = ch / width, at = ch - group * width;
#pragma unroll
		for (int e = 0; e < V; ++e) {
			f(e, ch, group);
			if (++at == width) at = 0, ++group;
			if (++ch == c) ch = 0, group = 0;
		}
	}
}

constexpr int kMaxWidth = 2048;                  // values of a row of a slab

// ---- forward: statistics, and with FINISH the normalised values, from one read ---------------------------------------------------------
// Two passes over registers cost less than one with a running mean, and the centred sum loses nothing. 32 x 4096 x 512 float16 with SiLU:
// 79 us (3.4 TB/s): a CU holds one workgroup of 256 KiB, whose loads and stores do not overlap; chunks that are read twice take 90.
// 128 x 1 x 2048: one wave a slab, 7 us.
// PART (FINISH = false): {mean, sum of centred squares} of the chunk's groups, for norm_join_kernel.
template <typename T, int NT, int NV, bool UNI, bool FINISH>
__global__ void __launch_bounds__(NT) norm_slab_kernel(Norm g, Slab s, float2 *part) {
	constexpr int V = Vec<T>::V, CELLS = UNI ? 1 : V;
	__shared__ float red[NT * CELLS];
	constexpr int GROUPS = UNI ? NT : NT * V < kMaxWidth ? NT * V : kMaxWidth;      // (of a row of NT vectors at most; UNI: one to a vector at most)
	__shared__ float smean[GROUPS], sinv[GROUPS];
	const int ty = threadIdx.x / s.tx, tx = threadIdx.x - ty * s.tx, TY = s.ty;
	int slab, chunk;
	long sample;
	place(s, slab, chunk, sample);
	const int c0 = slab * s.width * (s.slabs > 1);
	const int groups = s.slabs > 1 ? s.width / g.width : g.groups, group0 = c0 / g.width;
	const size_t start = ((size_t)sample * g.pixels) * g.c + c0 + (size_t)chunk * s.rows * s.pitch;
	const T *x = (const T *)g.x + start;
	const float count = chunk == s.chunks - 1 ? s.last_count : s.count;

	typename Vec<T>::raw v[NV];
	int mine, last;
	share<V>(s, chunk, tx, ty, NV, mine, last);
#pragma unroll
	for (int k = 0; k < NV; ++k)
		if (k < mine) v[k] = load_vec(x + (ty + k * TY) * (size_t)s.pitch + tx * V, k + 1 < mine ? V : last);

	float acc[CELLS];
	auto cells = [&](auto value) {                                              // red <- per-thread sums of value(x, cell)
#pragma unroll
		for (int e = 0; e < CELLS; ++e) acc[e] = 0.f;
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k + 1 < mine || (k < mine && last == V)) {
#pragma unroll
				for (int e = 0; e < V; ++e) acc[UNI ? 0 : e] += value((float)v[k][e], e);
			} else if (k < mine) {
#pragma unroll
				for (int e = 0; e < V; ++e)
					if (e < last) acc[UNI ? 0 : e] += value((float)v[k][e], e);
			}
		}
		if (ty < TY) {
#pragma unroll
			for (int e = 0; e < CELLS; ++e) red[(ty * s.tx + tx) * CELLS + e] = acc[e];
		}
		__syncthreads();
	};

	cells([](float f, int) { return f; });
	sum_cells<NT>(red, s.tx * CELLS, TY, s.reps, s.period, s.wd, groups, 1.f / count, smean);
	__syncthreads();

	float mean[CELLS];
	each_channel<CELLS, UNI>(tx * V, g.c, g.width, [&](int e, int, int group) { mean[e] = smean[group]; });
	cells([&](float f, int e) {
		const float d = f - mean[UNI ? 0 : e];
		return d * d;
	});
	sum_cells<NT>(red, s.tx * CELLS, TY, s.reps, s.period, s.wd, groups, 1.f, sinv);
	__syncthreads();

	if (!FINISH) {
		for (int o = threadIdx.x; o < groups; o += NT)
			part[((size_t)sample * s.chunks + chunk) * g.groups + group0 + o] = make_float2(smean[o], sinv[o]);
		return;
	}
	for (int o = threadIdx.x; o < groups; o += NT) {
		const float inv = 1.f / sqrtf(sinv[o] / count + g.epsilon);
		sinv[o] = inv;
		if (g.mean) g.mean[(size_t)sample * g.groups + group0 + o] = smean[o];
		if (g.invvar) g.invvar[(size_t)sample * g.groups + group0 + o] = inv;
	}
	__syncthreads();
	if (mine == 0) return;

	float scale[V], bias[V];
	if (UNI) load_floats(g.scale, c0 + tx * V, 1.f, scale), load_floats(g.bias, c0 + tx * V, 0.f, bias);
	each_channel<V, UNI>(tx * V, g.c, g.width, [&](int e, int ch, int group) {
		if (!UNI) scale[e] = or_else(g.scale, c0 + ch, 1.f), bias[e] = or_else(g.bias, c0 + ch, 0.f);
		scale[e] *= sinv[group];
	});
	T *y = (T *)g.out + start;
	with_act(g.act, [&](auto act) {
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k >= mine) continue;
			float o[V];
#pragma unroll
			for (int e = 0; e < V; ++e) o[e] = act_value(((float)v[k][e] - mean[UNI ? 0 : e]) * scale[e] + bias[e], act);
			store_vec(y + (ty + k * TY) * (size_t)s.pitch + tx * V, k + 1 < mine ? V : last, o);
		}
	});
}

// mean and 1 / sqrt(var + epsilon) of a (sample, group) from its chunks' {mean, centred squares}: a wave each, float64 sums
__global__ void __launch_bounds__(256) norm_join_kernel(Norm g, Slab s, const float2 *part, float *mean, float *invvar) {
	const long at = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
	if (at >= (long)g.n * g.groups) return;
	const int lane = threadIdx.x & 63;
	const unsigned sample = (unsigned)at / g.groups, group = (unsigned)at - sample * g.groups;
	const double total = (double)g.pixels * g.width;
	auto each = [&](int k) { return (double)(k == s.chunks - 1 ? s.last_count : s.count); };
	auto sum = [](double v) {
		for (int l = 32; l > 0; l >>= 1) v += __shfl_xor(v, l, 64);
		return v;
	};
	double m = 0.0, q = 0.0;
	for (int k = lane; k < s.chunks; k += 64) m += each(k) * part[((size_t)sample * s.chunks + k) * g.groups + group].x;
	m = sum(m) / total;
	for (int k = lane; k < s.chunks; k += 64) {
		const float2 p = part[((size_t)sample * s.chunks + k) * g.groups + group];
		const double d = p.x - m;
		q += p.y + each(k) * d * d;
	}
	q = sum(q) / total;
	if (lane == 0) mean[at] = (float)m, invvar[at] = (float)(1.0 / sqrt(q + (double)g.epsilon));
}

// y from x and the statistics, a chunk of rows back to back, bound by memory
template <typename T, int NV, bool UNI>
__global__ void __launch_bounds__(256) norm_apply_kernel(Norm g, Slab s, const float *means, const float *invvars) {
	constexpr int V = Vec<T>::V, CELLS = UNI ? 1 : V;
	const int ty = threadIdx.x / s.tx, tx = threadIdx.x - ty * s.tx;
	int slab, chunk, mine, last;
	long sample;
	place(s, slab, chunk, sample);
	share<V>(s, chunk, tx, ty, NV, mine, last);
	const size_t start = (size_t)sample * g.pixels * g.c + (size_t)chunk * s.rows * s.pitch + (size_t)ty * s.pitch + tx * V;
	const T *x = (const T *)g.x + start;
	T *y = (T *)g.out + start;
	typename Vec<T>::raw v[NV];
#pragma unroll
	for (int k = 0; k < NV; ++k)
		if (k < mine) v[k] = load_vec(x + (size_t)k * s.ty * s.pitch, k + 1 < mine ? V : last);
	float mean[CELLS], scale[V], bias[V], inv = 0.f;
	if (UNI) load_floats(g.scale, tx * V, 1.f, scale), load_floats(g.bias, tx * V, 0.f, bias);
	each_channel<V, UNI>(tx * V, g.c, g.width, [&](int e, int ch, int group) {
		const size_t at = sample * g.groups + group;
		if (!UNI || e == 0) mean[UNI ? 0 : e] = means[at], inv = invvars[at];
		if (!UNI) scale[e] = or_else(g.scale, ch, 1.f), bias[e] = or_else(g.bias, ch, 0.f);
		scale[e] *= inv;
	});
	with_act(g.act, [&](auto act) {
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k >= mine) continue;
			float o[V];
#pragma unroll
			for (int e = 0; e < V; ++e) o[e] = act_value(((float)v[k][e] - mean[UNI ? 0 : e]) * scale[e] + bias[e], act);
			store_vec(y + (size_t)k * s.ty * s.pitch, k + 1 < mine ? V : last, o);
		}
	});
}

// ---- backward ---------------------------------------------------------------------------------------------------------------------------
// Sums over a chunk's pixels per channel, sums[((sample * chunks + chunk) * 2 + {0: da, 1: da xhat}) * c + channel], and with FINISH dx from
// the same registers. 64 x 1024 x 512 float16 with SiLU: 68 us (3.0 TB/s), two workgroups of 128 KiB a CU; chunks take 84.
// (512 threads: 128 registers, so that a CU holds two workgroups; 134 would leave one: 89 us)
template <typename T, int NT, int NV, bool UNI, bool FINISH>
__global__ void __launch_bounds__(NT, NT == 512 ? 4 : 1) norm_slab_bwd_kernel(Norm g, Slab s, float *sums) {
	constexpr int V = Vec<T>::V, CELLS = UNI ? 1 : V;
	__shared__ float red[2][NT * V];
	__shared__ float chan[2][NT * V < kMaxWidth ? NT * V : kMaxWidth];      // (a row has NT vectors at most)
	constexpr int GROUPS = UNI ? NT : NT * V < kMaxWidth ? NT * V : kMaxWidth;
	__shared__ float sa[GROUPS], sb[GROUPS];
	const int ty = threadIdx.x / s.tx, tx = threadIdx.x - ty * s.tx, TY = s.ty;
	int slab, chunk;
	long sample;
	place(s, slab, chunk, sample);
	const int c0 = slab * s.width * (s.slabs > 1);
	const int channels = s.slabs > 1 ? s.width : g.c, groups = channels / g.width, group0 = c0 / g.width;
	const size_t start = (size_t)sample * g.pixels * g.c + c0 + (size_t)chunk * s.rows * s.pitch;
	const T *x = (const T *)g.x + start, *dy = (const T *)g.dy + start;

	typename Vec<T>::raw v[NV], d[NV];
	int mine, last;
	share<V>(s, chunk, tx, ty, NV, mine, last);
#pragma unroll
	for (int k = 0; k < NV; ++k) {
		const size_t at = (ty + k * TY) * (size_t)s.pitch + tx * V;
		const int left = k + 1 < mine ? V : last;
		if (k < mine) v[k] = load_vec(x + at, left), d[k] = load_vec(dy + at, left);      // (beyond the end: zeros, which add nothing)
	}
	float mean[CELLS], inv[CELLS], scale[V], bias[V], da[V], db[V];
	if (UNI) load_floats(g.scale, c0 + tx * V, 1.f, scale), load_floats(g.bias, c0 + tx * V, 0.f, bias);
	each_channel<V, UNI>(tx * V, g.c, g.width, [&](int e, int ch, int group) {
		const size_t at = sample * g.groups + group0 + group;
		if (!UNI || e == 0) mean[UNI ? 0 : e] = g.mean[at], inv[UNI ? 0 : e] = g.invvar[at];
		if (!UNI) scale[e] = or_else(g.scale, c0 + ch, 1.f), bias[e] = or_else(g.bias, c0 + ch, 0.f);
		da[e] = db[e] = 0.f;
	});
	with_act(g.act, [&](auto act) {
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k >= mine) continue;
#pragma unroll
			for (int e = 0; e < V; ++e) {
				const float xhat = ((float)v[k][e] - mean[UNI ? 0 : e]) * inv[UNI ? 0 : e];
				const float t = (float)d[k][e] * act_slope(scale[e] * xhat + bias[e], act);
				da[e] += t, db[e] += t * xhat;
			}
		}
	});
	if (ty < TY) {
#pragma unroll
		for (int e = 0; e < V; ++e) red[0][(ty * s.tx + tx) * V + e] = da[e], red[1][(ty * s.tx + tx) * V + e] = db[e];
	}
	__syncthreads();
	for (int i = 0; i < 2; ++i) sum_cells<NT>(red[i], s.tx * V, TY, s.reps, g.c, 1, channels, 1.f, chan[i]);
	__syncthreads();
	for (int i = threadIdx.x; i < 2 * channels; i += NT)
		sums[(((size_t)sample * s.chunks + chunk) * 2 + i / channels) * g.c + c0 + i % channels] = chan[i / channels][i % channels];
	if (!FINISH) return;

	__syncthreads();
	for (int i = threadIdx.x; i < channels; i += NT) {
		const float f = or_else(g.scale, c0 + i, 1.f);
		chan[0][i] *= f, chan[1][i] *= f;
	}
	__syncthreads();
	const float one = 1.f / ((float)g.pixels * (float)g.width);
	sum_cells<NT>(chan[0], 0, 1, 1, 0, g.width, groups, one, sa);
	sum_cells<NT>(chan[1], 0, 1, 1, 0, g.width, groups, one, sb);
	__syncthreads();
	if (mine == 0) return;
	float a[CELLS], b[CELLS];
	each_channel<CELLS, UNI>(tx * V, g.c, g.width, [&](int e, int, int group) { a[e] = sa[group], b[e] = sb[group]; });
	T *dx = (T *)g.out + start;
	with_act(g.act, [&](auto act) {
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k >= mine) continue;
			float o[V];
#pragma unroll
			for (int e = 0; e < V; ++e) {
				const int u = UNI ? 0 : e;
				const float xhat = ((float)v[k][e] - mean[u]) * inv[u];
				const float t = scale[e] * ((float)d[k][e] * act_slope(scale[e] * xhat + bias[e], act));
				o[e] = inv[u] * (t - a[u] - xhat * b[u]);
			}
			store_vec(dx + (ty + k * TY) * (size_t)s.pitch + tx * V, k + 1 < mine ? V : last, o);
		}
	});
}

// The chunks' channel sums of a (sample, group), a workgroup each: added in a fixed order in float64 into totals[(sample * 2 + {0, 1}) * c +
// channel] (what norm_param_kernel reads: a row per sample instead of one per chunk), and with `scale` into A and B of the head,
// divided by m. 16 channels at a time, 16 chunks side by side (16 x 4096 x 256 float32, 128 chunks a sample: with it the backward pass took
// 73 us; with the parameters' kernel reading a row per chunk 85).
__global__ void __launch_bounds__(256) norm_join_bwd_kernel(Norm g, Slab s, const float *sums, float *totals, float2 *ab) {
	__shared__ double part[2][16][17];
	const long at = blockIdx.x, sample = at / g.groups;
	const int c0 = (int)(at - sample * g.groups) * g.width, lane = threadIdx.x & 15, row = threadIdx.x >> 4;
	double a = 0.0, b = 0.0;                                                    // (of lane's channels, in the threads of row 0)
	for (int strip = 0; strip < g.width; strip += 16) {
		const bool mine = strip + lane < g.width;
		const int ch = c0 + strip + lane;
		double p0 = 0.0, p1 = 0.0;
		if (mine) {
			const float *p = sums + ((size_t)sample * s.chunks + row) * 2 * g.c + ch;
#pragma unroll 4
			for (int chunk = row; chunk < s.chunks; chunk += 16, p += (size_t)32 * g.c) p0 += p[0], p1 += p[g.c];
		}
		part[0][row][lane] = p0, part[1][row][lane] = p1;
		__syncthreads();
		if (row == 0 && mine) {
			for (int r = 1; r < 16; ++r) p0 += part[0][r][lane], p1 += part[1][r][lane];
			totals[(size_t)sample * 2 * g.c + ch] = (float)p0, totals[((size_t)sample * 2 + 1) * g.c + ch] = (float)p1;
			const double f = or_else(g.scale, ch, 1.f);
			a += f * p0, b += f * p1;
		}
		__syncthreads();
	}
	if (row > 0) return;
	for (int l = 8; l > 0; l >>= 1) a += __shfl_xor(a, l, 16), b += __shfl_xor(b, l, 16);
	const double m = (double)g.pixels * g.width;
	if (lane == 0) ab[at] = make_float2((float)(a / m), (float)(b / m));
}

template <typename T, int NV, bool UNI>
__global__ void __launch_bounds__(256) norm_apply_bwd_kernel(Norm g, Slab s, const float2 *ab) {
	constexpr int V = Vec<T>::V, CELLS = UNI ? 1 : V;
	const int ty = threadIdx.x / s.tx, tx = threadIdx.x - ty * s.tx;
	int slab, chunk, mine, last;
	long sample;
	place(s, slab, chunk, sample);
	share<V>(s, chunk, tx, ty, NV, mine, last);
	const size_t start = (size_t)sample * g.pixels * g.c + (size_t)chunk * s.rows * s.pitch + (size_t)ty * s.pitch + tx * V;
	const T *x = (const T *)g.x + start, *dy = (const T *)g.dy + start;
	T *dx = (T *)g.out + start;
	typename Vec<T>::raw v[NV], d[NV];
#pragma unroll
	for (int k = 0; k < NV; ++k) {
		const size_t at = (size_t)k * s.ty * s.pitch;
		const int left = k + 1 < mine ? V : last;
		if (k < mine) v[k] = load_vec(x + at, left), d[k] = load_vec(dy + at, left);
	}
	float mean[CELLS], inv[CELLS], scale[V], bias[V];
	float2 sum[CELLS];
	if (UNI) load_floats(g.scale, tx * V, 1.f, scale), load_floats(g.bias, tx * V, 0.f, bias);
	each_channel<V, UNI>(tx * V, g.c, g.width, [&](int e, int ch, int group) {
		const size_t at = sample * g.groups + group;
		if (!UNI || e == 0) mean[UNI ? 0 : e] = g.mean[at], inv[UNI ? 0 : e] = g.invvar[at], sum[UNI ? 0 : e] = ab[at];
		if (!UNI) scale[e] = or_else(g.scale, ch, 1.f), bias[e] = or_else(g.bias, ch, 0.f);
	});
	with_act(g.act, [&](auto act) {
#pragma unroll
		for (int k = 0; k < NV; ++k) {
			if (k >= mine) continue;
			float o[V];
#pragma unroll
			for (int e = 0; e < V; ++e) {
				const int u = UNI ? 0 : e;
				const float xhat = ((float)v[k][e] - mean[u]) * inv[u];
				const float t = scale[e] * ((float)d[k][e] * act_slope(scale[e] * xhat + bias[e], act));
				o[e] = inv[u] * (t - sum[u].x - xhat * sum[u].y);
			}
			store_vec(dx + (size_t)k * s.ty * s.pitch, k + 1 < mine ? V : last, o);
		}
	});
}

// ---- any shape: one workgroup per (sample, group), three sweeps over its values ----------------------------------------------------------
// Threads take consecutive channels of consecutive pixels. Kept simple: it reads x three times. A thread adds m / 256 values one after the
// other, so it adds them in float64: in float32 4096 x 4100 values of 1.1 +- 0.001 gave a mean off by a quarter of their deviation.
// Rows come here that no workgroup holds: where neither slabs of whole groups fit (plan_norm), nor a row of all channels is at most kMaxWidth
// values and 256 vectors — float32 above 1024 channels, or a channel count whose vectors repeat later than that.
__device__ __forceinline__ double block_sum64(double v, double *smem) {
	for (int l = 32; l > 0; l >>= 1) v += __shfl_xor(v, l, 64);
	__syncthreads();
	if ((threadIdx.x & 63) == 0) smem[threadIdx.x >> 6] = v;
	__syncthreads();
	return smem[0] + smem[1] + smem[2] + smem[3];
}

template <typename T>
__global__ void __launch_bounds__(256) norm_fwd_kernel(Norm g) {
	__shared__ double red[4];
	const int group = blockIdx.x % g.groups, c0 = group * g.width;
	const long sample = blockIdx.x / g.groups;
	const T *x = (const T *)g.x + sample * g.pixels * g.c + c0;
	T *y = (T *)g.out + sample * g.pixels * g.c + c0;
	const long m = (long)g.pixels * g.width;

	double sum = 0.0;
	for (long i = threadIdx.x; i < m; i += 256) sum += (float)x[i / g.width * g.c + i % g.width];
	const float mean = (float)(block_sum64(sum, red) / (double)m);
	double square = 0.0;
	for (long i = threadIdx.x; i < m; i += 256) {
		const float d = (float)x[i / g.width * g.c + i % g.width] - mean;
		square += d * d;
	}
	const float invvar = (float)(1.0 / sqrt(block_sum64(square, red) / (double)m + (double)g.epsilon));
	if (threadIdx.x == 0) {
		if (g.mean) g.mean[blockIdx.x] = mean;
		if (g.invvar) g.invvar[blockIdx.x] = invvar;
	}
	for (long i = threadIdx.x; i < m; i += 256) {
		const int ch = (int)(i % g.width);
		const size_t at = (size_t)(i / g.width) * g.c + ch;
		y[at] = (T)act_value(or_else(g.scale, c0 + ch, 1.f) * (((float)x[at] - mean) * invvar) + or_else(g.bias, c0 + ch, 0.f), g.act);
	}
}

template <typename T>
__global__ void __launch_bounds__(256) norm_bwd_kernel(Norm g) {
	__shared__ double red[4];
	const int group = blockIdx.x % g.groups, c0 = group * g.width;
	const size_t base = (size_t)(blockIdx.x / g.groups) * g.pixels * g.c + c0;
	const T *x = (const T *)g.x + base, *dy = (const T *)g.dy + base;
	T *dx = (T *)g.out + base;
	const long m = (long)g.pixels * g.width;
	const float mean = g.mean[blockIdx.x], invvar = g.invvar[blockIdx.x];

	double sum_a = 0.0, sum_b = 0.0;
	for (long i = threadIdx.x; i < m; i += 256) {
		const int ch = (int)(i % g.width);
		const size_t at = (size_t)(i / g.width) * g.c + ch;
		const float scale = or_else(g.scale, c0 + ch, 1.f), xhat = ((float)x[at] - mean) * invvar;
		const float d = scale * ((float)dy[at] * act_slope(scale * xhat + or_else(g.bias, c0 + ch, 0.f), g.act));
		sum_a += d, sum_b += d * xhat;
	}
	const float a = (float)(block_sum64(sum_a, red) / (double)m), b = (float)(block_sum64(sum_b, red) / (double)m);
	for (long i = threadIdx.x; i < m; i += 256) {
		const int ch = (int)(i % g.width);
		const size_t at = (size_t)(i / g.width) * g.c + ch;
		const float scale = or_else(g.scale, c0 + ch, 1.f), xhat = ((float)x[at] - mean) * invvar;
		const float d = scale * ((float)dy[at] * act_slope(scale * xhat + or_else(g.bias, c0 + ch, 0.f), g.act));
		dx[at] = (T)(invvar * (d - a - xhat * b));
	}
}

// sums over the pixels of one sample, a thread per channel, in the layout of norm_slab_bwd_kernel
template <typename T>
__global__ void __launch_bounds__(256) norm_channel_kernel(Norm g, float *sums) {
	const long at = (long)blockIdx.x * 256 + threadIdx.x;
	if (at >= (long)g.n * g.c) return;
	const long sample = at / g.c;
	const int ch = (int)(at % g.c);
	const T *x = (const T *)g.x + sample * g.pixels * g.c + ch, *dy = (const T *)g.dy + sample * g.pixels * g.c + ch;
	const size_t stat = sample * g.groups + ch / g.width;
	const float mean = g.mean[stat], invvar = g.invvar[stat], scale = or_else(g.scale, ch, 1.f), bias = or_else(g.bias, ch, 0.f);
	double s = 0.0, b = 0.0;
	for (int p = 0; p < g.pixels; ++p) {
		const float xhat = ((float)x[(size_t)p * g.c] - mean) * invvar;
		const float d = (float)dy[(size_t)p * g.c] * act_slope(scale * xhat + bias, g.act);
		b += d, s += d * xhat;
	}
	sums[(sample * 2) * g.c + ch] = (float)b;
	sums[(sample * 2 + 1) * g.c + ch] = (float)s;
}

// dbias, dscale: the samples' sums, added in a fixed order in float64. A workgroup takes 16 channels, 64 rows at a time:
// 64 samples of 512 channels 4 us.
__global__ void __launch_bounds__(1024) norm_param_kernel(const float *sums, int rows, int c, float *dscale, float *dbias) {
	__shared__ double part[2][64][16];
	const int lane = threadIdx.x & 15, row = threadIdx.x >> 4, ch = blockIdx.x * 16 + lane;
	double s = 0.0, b = 0.0;
	if (ch < c) {
#pragma unroll 4
		for (int i = row; i < rows; i += 64) {
			b += sums[(size_t)i * 2 * c + ch];
			s += sums[((size_t)i * 2 + 1) * c + ch];
		}
	}
	part[0][row][lane] = b, part[1][row][lane] = s;
	__syncthreads();
	for (int half = 32; half > 0; half >>= 1) {
		if (row < half) part[0][row][lane] += part[0][row + half][lane], part[1][row][lane] += part[1][row + half][lane];
		__syncthreads();
	}
	if (row > 0 || ch >= c) return;
	if (dbias) dbias[ch] = (float)part[0][0][lane];
	if (dscale) dscale[ch] = (float)part[1][0][lane];
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------
int check(const pz_groupnorm_desc *d, const char *who) {
	PZ_REQUIRE(d, "%s: null descriptor", who);
	PZ_REQUIRE(d->dtype == PZ_F32 || d->dtype == PZ_F16, "%s: unknown dtype %d", who, d->dtype);
	PZ_REQUIRE(d->act >= PZ_ACT_NONE && d->act <= PZ_ACT_SILU, "%s: unknown activation %d", who, d->act);
	PZ_REQUIRE(d->n >= 0 && d->pixels >= 0 && d->c > 0 && d->groups > 0 && d->c % d->groups == 0, "%s: bad dimensions (%d, %d, %d) in %d groups", who,
	           d->n, d->pixels, d->c, d->groups);
	PZ_REQUIRE((long)d->n * d->groups < (1l << 31) && (long)d->n * d->c < (1l << 32) - 256 && d->c < (1 << 26), "%s: %d samples of %d channels are too many", who, d->n, d->c);
	PZ_REQUIRE(d->epsilon >= 0.f, "%s: epsilon %g", who, d->epsilon);
	return PZ_OK;
}

Norm args_of(const pz_groupnorm_desc *d) {
	Norm g{};
	g.n = d->n, g.pixels = d->pixels, g.c = d->c, g.groups = d->groups, g.width = d->c / d->groups;
	g.act = d->act, g.epsilon = d->epsilon;
	return g;
}

long gcd(long a, long b) { return b == 0 ? a : gcd(b, a % b); }

enum { WAY_PLAIN, WAY_ONE, WAY_CHUNKS };

struct Plan {
	int way, nt, nv;                 // WAY_ONE: threads and vectors a thread of the kernel that holds a sample's slab
	Slab slab;                       // WAY_CHUNKS: of the statistics
	Slab apply;                      // WAY_CHUNKS: of the second read
	size_t part_bytes, stat_bytes;
};

// vectors a thread holds at most: 16 forward (64 registers), 8 + 8 backward
constexpr int kForwardVectors = 16, kBackwardVectors = 8;

Slab back_to_back(const pz_groupnorm_desc *d, int v, int threads, int vectors) {
	Slab s{};
	const int width = d->c / d->groups, period = (int)(d->c / gcd(d->c, v) * v);          // lcm
	s.width = s.pitch = period, s.tx = period / v, s.ty = threads / s.tx, s.reps = period / d->c, s.slabs = s.sharing = 1;
	s.uniform = s.reps == 1 && width % v == 0;
	s.wd = s.uniform ? width / v : width, s.period = s.uniform ? d->c / v : d->c;
	const long values = (long)d->pixels * d->c, rows = (values + period - 1) / period, held = (long)s.ty * vectors;
	s.rows = (int)(rows < held ? rows : held);
	s.chunks = (int)((rows + s.rows - 1) / s.rows);
	const long before = (long)(s.chunks - 1) * s.rows;
	s.last_rows = (int)(rows - before), s.last_values = (int)(values - before * period);
	s.count = (float)((long)s.rows * period / d->c * width), s.last_count = (float)((long)s.last_values / d->c * width);
	return s;
}

Plan plan_norm(const pz_groupnorm_desc *d, bool backward) {
	Plan p{};
	const int v = d->dtype == PZ_F16 ? 8 : 4, size = d->dtype == PZ_F16 ? 2 : 4, width = d->c / d->groups;
	const long period = d->c / gcd(d->c, v) * v;
	const int vectors = backward ? kBackwardVectors : kForwardVectors;
	if (d->n == 0 || d->pixels == 0) return p;

	// whole groups of a channel count that vectors divide: the widest slab of a cache line or half of one of which a CU holds two workgroups
	// (one loads while the other stores); where none fits, one workgroup of twice the size. Quarter lines do not pay: 115 instead of 87 us
	// for 32 x 4096 x 512 float16
	const long unit = width / gcd(width, v) * v;
	const bool uniform = width % v == 0;
	if (d->c % v == 0 && d->c % unit == 0 && unit <= kMaxWidth) {
		for (const int most : {512, 1024}) {
			for (const long bytes : {128l, 64l}) {
				long slab = unit;
				while (slab * size < bytes && slab < d->c) {
					do slab += unit;
					while (d->c % slab != 0);
				}
				if (slab > kMaxWidth) continue;
				const int tx = (int)(slab / v);
				for (const int nt : {64, 256, 512, 1024})
					for (const int nv : {4, vectors}) {
						if (nt > (uniform ? most : 256) || (nt == 64 && nv > 4) || tx > nt || (long)(nt / tx) * nv < d->pixels) continue;
						// few large workgroups leave most of the chip idle: chunks, although they read twice (16 workgroups of 256 KiB: 25 us,
						// chunks 20)
						if (nt > 256 && (long)d->n * (d->c / slab) < pz::kNumCU / 2) continue;
						p.way = WAY_ONE, p.nt = nt, p.nv = nv;
						Slab s{};
						s.width = (int)slab, s.tx = tx, s.ty = nt / tx, s.reps = 1, s.slabs = (int)(d->c / slab), s.uniform = uniform, s.pitch = d->c;
						s.rows = s.last_rows = d->pixels, s.last_values = (int)(d->pixels * slab), s.chunks = 1;
						s.count = s.last_count = (float)((long)d->pixels * width);
						s.sharing = (int)(128 / (slab * size));
						if (s.sharing < 1 || (long)d->n * s.slabs % (8 * s.sharing) != 0) s.sharing = 1;
						s.wd = uniform ? width / v : width, s.period = 0;
						if (s.slabs == 1) s.period = uniform ? d->c / v : d->c;
						p.slab = s;
						return p;
					}
			}
		}
	}
	if (period > kMaxWidth || period / v > 256) return p;                                   // WAY_PLAIN
	for (const int nt : {64, 256})
		for (const int nv : {4, vectors}) {
			if (period / v > nt || (nt == 64 && nv > 4)) continue;
			const Slab s = back_to_back(d, v, nt, nv);
			if (s.chunks > 1) continue;
			p.way = WAY_ONE, p.nt = nt, p.nv = nv, p.slab = s;
			return p;
		}
	p.way = WAY_CHUNKS, p.nt = 256, p.nv = vectors;
	p.slab = back_to_back(d, v, 256, vectors);
	p.apply = back_to_back(d, v, 256, 8);
	p.part_bytes = backward ? 0 : (size_t)d->n * p.slab.chunks * d->groups * sizeof(float2);
	p.stat_bytes = (size_t)d->n * d->groups * sizeof(float2);
	return p;
}

// the backward pass's workspace: channel sums per sample, per chunk of a sample with WAY_CHUNKS, then A and B of the head
size_t total_bytes(const pz_groupnorm_desc *d) { return (size_t)d->n * 2 * d->c * sizeof(float); }
size_t chunk_bytes(const pz_groupnorm_desc *d, const Plan &p) { return p.way == WAY_CHUNKS ? total_bytes(d) * p.slab.chunks : 0; }

template <typename T, int NT, int NV, bool UNI, bool FINISH>
void slab_fwd(const Norm &g, const Plan &p, float2 *part, hipStream_t st) {
	norm_slab_kernel<T, NT, NV, UNI, FINISH><<<(unsigned)((long)g.n * p.slab.chunks * p.slab.slabs), NT, 0, st>>>(g, p.slab, part);
}

template <typename T>
int forward(const pz_groupnorm_desc *d, const Norm &g, char *ws, hipStream_t st) {
	const Plan p = plan_norm(d, false);
	if (p.way == WAY_PLAIN) {
		PZ_REQUIRE(launchable((long)d->n * d->groups, 256), "pz_groupnorm_fwd: too many workgroups");
		norm_fwd_kernel<T><<<d->n * d->groups, 256, 0, st>>>(g);
		PZ_LAUNCH_CHECK();
		return PZ_OK;
	}
	PZ_REQUIRE(launchable((long)d->n * p.slab.chunks * p.slab.slabs, p.nt), "pz_groupnorm_fwd: too many workgroups");
	if (p.way == WAY_ONE) {
		if (p.slab.uniform) {
			if (p.nt == 64) slab_fwd<T, 64, 4, true, true>(g, p, nullptr, st);
			else if (p.nt == 1024) slab_fwd<T, 1024, 16, true, true>(g, p, nullptr, st);
			else if (p.nt == 512) slab_fwd<T, 512, 16, true, true>(g, p, nullptr, st);
			else if (p.nv == 4) slab_fwd<T, 256, 4, true, true>(g, p, nullptr, st);
			else slab_fwd<T, 256, 16, true, true>(g, p, nullptr, st);
		} else if (p.nt == 64) slab_fwd<T, 64, 4, false, true>(g, p, nullptr, st);
		else if (p.nv == 4) slab_fwd<T, 256, 4, false, true>(g, p, nullptr, st);
		else slab_fwd<T, 256, 16, false, true>(g, p, nullptr, st);
		PZ_LAUNCH_CHECK();
		return PZ_OK;
	}
	float2 *part = (float2 *)ws;
	float *stats = (float *)(ws + p.part_bytes);
	float *mean = g.mean ? g.mean : stats, *invvar = g.invvar ? g.invvar : stats + (size_t)d->n * d->groups;
	PZ_REQUIRE(launchable((long)d->n * p.apply.chunks, 256), "pz_groupnorm_fwd: too many workgroups");
	if (p.slab.uniform) slab_fwd<T, 256, 16, true, false>(g, p, part, st);
	else slab_fwd<T, 256, 16, false, false>(g, p, part, st);
	PZ_LAUNCH_CHECK();
	norm_join_kernel<<<pz::ceil_div((long)d->n * d->groups, 4), 256, 0, st>>>(g, p.slab, part, mean, invvar);
	PZ_LAUNCH_CHECK();
	const unsigned blocks = (unsigned)((long)d->n * p.apply.chunks);
	if (p.apply.uniform) norm_apply_kernel<T, 8, true><<<blocks, 256, 0, st>>>(g, p.apply, mean, invvar);
	else norm_apply_kernel<T, 8, false><<<blocks, 256, 0, st>>>(g, p.apply, mean, invvar);
	PZ_LAUNCH_CHECK();
	return PZ_OK;
}

template <typename T, int NT, int NV, bool UNI, bool FINISH>
void slab_bwd(const Norm &g, const Plan &p, float *sums, hipStream_t st) {
	norm_slab_bwd_kernel<T, NT, NV, UNI, FINISH><<<(unsigned)((long)g.n * p.slab.chunks * p.slab.slabs), NT, 0, st>>>(g, p.slab, sums);
}

template <typename T>
int backward(const pz_groupnorm_desc *d, const Norm &g, const Plan &p, float *sums, hipStream_t st) {
	float *chunks = (float *)((char *)sums + total_bytes(d));
	float2 *ab = (float2 *)((char *)chunks + chunk_bytes(d, p));
	PZ_REQUIRE(p.way == WAY_ONE || launchable((long)d->n * d->groups, 256), "pz_groupnorm_bwd: too many workgroups");
	if (p.way == WAY_PLAIN) {
		norm_channel_kernel<T><<<pz::ceil_div((long)d->n * d->c, 256), 256, 0, st>>>(g, sums);
		PZ_LAUNCH_CHECK();
		norm_bwd_kernel<T><<<d->n * d->groups, 256, 0, st>>>(g);
		PZ_LAUNCH_CHECK();
		return PZ_OK;
	}
	PZ_REQUIRE(launchable((long)d->n * p.slab.chunks * p.slab.slabs, p.nt), "pz_groupnorm_bwd: too many workgroups");
	if (p.way == WAY_ONE) {
		if (p.slab.uniform) {
			if (p.nt == 64) slab_bwd<T, 64, 4, true, true>(g, p, sums, st);
			else if (p.nt == 1024) slab_bwd<T, 1024, 8, true, true>(g, p, sums, st);
			else if (p.nt == 512) slab_bwd<T, 512, 8, true, true>(g, p, sums, st);
			else p.nv == 4 ? slab_bwd<T, 256, 4, true, true>(g, p, sums, st) : slab_bwd<T, 256, 8, true, true>(g, p, sums, st);
		} else if (p.nt == 64) slab_bwd<T, 64, 4, false, true>(g, p, sums, st);
		else p.nv == 4 ? slab_bwd<T, 256, 4, false, true>(g, p, sums, st) : slab_bwd<T, 256, 8, false, true>(g, p, sums, st);
		PZ_LAUNCH_CHECK();
		return PZ_OK;
	}
	PZ_REQUIRE(launchable((long)d->n * p.apply.chunks, 256), "pz_groupnorm_bwd: too many workgroups");
	if (p.slab.uniform) slab_bwd<T, 256, 8, true, false>(g, p, chunks, st);
	else slab_bwd<T, 256, 8, false, false>(g, p, chunks, st);
	PZ_LAUNCH_CHECK();
	norm_join_bwd_kernel<<<(unsigned)((long)d->n * d->groups), 256, 0, st>>>(g, p.slab, chunks, sums, ab);
	PZ_LAUNCH_CHECK();
	const unsigned blocks = (unsigned)((long)d->n * p.apply.chunks);
	if (p.apply.uniform) norm_apply_bwd_kernel<T, 8, true><<<blocks, 256, 0, st>>>(g, p.apply, ab);
	else norm_apply_bwd_kernel<T, 8, false><<<blocks, 256, 0, st>>>(g, p.apply, ab);
	PZ_LAUNCH_CHECK();
	return PZ_OK;
}

}  // namespace

extern "C" {

int pz_groupnorm_workspace_bytes(const pz_groupnorm_desc *d, int backward, size_t *nbytes) {
	if (int rc = check(d, "pz_groupnorm_workspace_bytes")) return rc;
	PZ_REQUIRE(nbytes, "pz_groupnorm_workspace_bytes: null output");
	const Plan p = plan_norm(d, backward != 0);
	*nbytes = backward ? total_bytes(d) + chunk_bytes(d, p) + p.stat_bytes : p.part_bytes + p.stat_bytes;
	return PZ_OK;
}

int pz_groupnorm_fwd(const pz_groupnorm_desc *d, const void *x, const float *scale, const float *bias, void *y, float *savemean, float *saveinvvar,
                     void *workspace, size_t ws_bytes, pz_stream_t stream) {
	if (int rc = check(d, "pz_groupnorm_fwd")) return rc;
	if (d->n == 0 || d->pixels == 0) return PZ_OK;
	size_t need = 0;
	if (int rc = pz_groupnorm_workspace_bytes(d, 0, &need)) return rc;
	PZ_REQUIRE(x && y, "pz_groupnorm_fwd: null tensor");
	PZ_REQUIRE(need == 0 || (workspace && ws_bytes >= need), "pz_groupnorm_fwd: workspace needs %zu bytes", need);
	Norm g = args_of(d);
	g.x = x, g.out = y, g.scale = scale, g.bias = bias, g.mean = savemean, g.invvar = saveinvvar;
	hipStream_t st = pz::as_stream(stream);
	return d->dtype == PZ_F16 ? forward<f16>(d, g, (char *)workspace, st) : forward<float>(d, g, (char *)workspace, st);
}

int pz_groupnorm_bwd(const pz_groupnorm_desc *d, const void *dy, const void *x, const float *scale, const float *bias, const float *savemean,
                     const float *saveinvvar, void *dx, float *dscale, float *dbias, void *workspace, size_t ws_bytes, pz_stream_t stream) {
	if (int rc = check(d, "pz_groupnorm_bwd")) return rc;
	hipStream_t st = pz::as_stream(stream);
	const bool empty = d->n == 0 || d->pixels == 0;
	size_t need = 0;
	if (int rc = pz_groupnorm_workspace_bytes(d, 1, &need)) return rc;
	PZ_REQUIRE(empty || (dy && x && dx && savemean && saveinvvar), "pz_groupnorm_bwd: null tensor");
	PZ_REQUIRE(empty || (workspace && ws_bytes >= need), "pz_groupnorm_bwd: workspace needs %zu bytes", need);
	Norm g = args_of(d);
	g.x = x, g.dy = dy, g.out = dx, g.scale = scale, g.bias = bias, g.mean = (float *)savemean, g.invvar = (float *)saveinvvar;
	const Plan p = plan_norm(d, true);
	float *sums = (float *)workspace;
	if (!empty)
		if (int rc = d->dtype == PZ_F16 ? backward<f16>(d, g, p, sums, st) : backward<float>(d, g, p, sums, st)) return rc;
	if (dscale || dbias) {
		norm_param_kernel<<<pz::ceil_div(d->c, 16), 1024, 0, st>>>(sums, empty ? 0 : d->n, d->c, dscale, dbias);
		PZ_LAUNCH_CHECK();
	}
	return PZ_OK;
}

}  // extern "C"
