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

// One workgroup per (sample, group), three sweeps over its values: any shape. Threads take consecutive channels of consecutive pixels.
template <typename T>
__global__ void __launch_bounds__(256) norm_fwd_kernel(Norm g) {
	__shared__ float red[16];
	const int group = blockIdx.x % g.groups, c0 = group * g.width;
	const long sample = blockIdx.x / g.groups;
	const T *x = (const T *)g.x + sample * g.pixels * g.c + c0;
	T *y = (T *)g.out + sample * g.pixels * g.c + c0;
	const long m = (long)g.pixels * g.width;

	float sum = 0.f;
	for (long i = threadIdx.x; i < m; i += 256) sum += (float)x[i / g.width * g.c + i % g.width];
	const float mean = block_sum(sum, red) / (float)m;
	float square = 0.f;
	for (long i = threadIdx.x; i < m; i += 256) {
		const float d = (float)x[i / g.width * g.c + i % g.width] - mean;
		square += d * d;
	}
	const float invvar = 1.f / sqrtf(block_sum(square, red) / (float)m + g.epsilon);
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
	__shared__ float red[16];
	const int group = blockIdx.x % g.groups, c0 = group * g.width;
	const size_t base = (size_t)(blockIdx.x / g.groups) * g.pixels * g.c + c0;
	const T *x = (const T *)g.x + base, *dy = (const T *)g.dy + base;
	T *dx = (T *)g.out + base;
	const long m = (long)g.pixels * g.width;
	const float mean = g.mean[blockIdx.x], invvar = g.invvar[blockIdx.x];

	float a = 0.f, b = 0.f;
	for (long i = threadIdx.x; i < m; i += 256) {
		const int ch = (int)(i % g.width);
		const size_t at = (size_t)(i / g.width) * g.c + ch;
		const float scale = or_else(g.scale, c0 + ch, 1.f), xhat = ((float)x[at] - mean) * invvar;
		const float d = scale * ((float)dy[at] * act_slope(scale * xhat + or_else(g.bias, c0 + ch, 0.f), g.act));
		a += d, b += d * xhat;
	}
	a = block_sum(a, red) / (float)m;
	b = block_sum(b, red) / (float)m;
	for (long i = threadIdx.x; i < m; i += 256) {
		const int ch = (int)(i % g.width);
		const size_t at = (size_t)(i / g.width) * g.c + ch;
		const float scale = or_else(g.scale, c0 + ch, 1.f), xhat = ((float)x[at] - mean) * invvar;
		const float d = scale * ((float)dy[at] * act_slope(scale * xhat + or_else(g.bias, c0 + ch, 0.f), g.act));
		dx[at] = (T)(invvar * (d - a - xhat * b));
	}
}

// sums over the pixels of one sample, a thread per channel: part[(sample * 2 + {0: da, 1: da * xhat}) * c + channel]
template <typename T>
__global__ void __launch_bounds__(256) norm_channel_kernel(Norm g, float *part) {
	const int ch = blockIdx.x * 256 + threadIdx.x;
	if (ch >= g.c) return;
	const size_t sample = blockIdx.y, at = sample * g.groups + ch / g.width;
	const T *x = (const T *)g.x + sample * g.pixels * g.c + ch, *dy = (const T *)g.dy + sample * g.pixels * g.c + ch;
	const float mean = g.mean[at], invvar = g.invvar[at], scale = or_else(g.scale, ch, 1.f), bias = or_else(g.bias, ch, 0.f);
	float s = 0.f, b = 0.f;
	for (int p = 0; p < g.pixels; ++p) {
		const float xhat = ((float)x[(size_t)p * g.c] - mean) * invvar;
		const float d = (float)dy[(size_t)p * g.c] * act_slope(scale * xhat + bias, g.act);
		b += d, s += d * xhat;
	}
	part[(sample * 2) * g.c + ch] = b;
	part[(sample * 2 + 1) * g.c + ch] = s;
}

// dbias, dscale: the samples' sums, added in order
__global__ void __launch_bounds__(256) norm_param_kernel(const float *part, int rows, int c, float *dscale, float *dbias) {
	const int ch = blockIdx.x * 256 + threadIdx.x;
	if (ch >= c) return;
	float s = 0.f, b = 0.f;
	for (int i = 0; i < rows; ++i) {
		b += part[((size_t)i * 2) * c + ch];
		s += part[((size_t)i * 2 + 1) * c + ch];
	}
	if (dbias) dbias[ch] = b;
	if (dscale) dscale[ch] = s;
}

int check(const pz_groupnorm_desc *d, const char *who) {
	PZ_REQUIRE(d, "%s: null descriptor", who);
	PZ_REQUIRE(d->dtype == PZ_F32 || d->dtype == PZ_F16, "%s: unknown dtype %d", who, d->dtype);
	PZ_REQUIRE(d->act >= PZ_ACT_NONE && d->act <= PZ_ACT_SILU, "%s: unknown activation %d", who, d->act);
	PZ_REQUIRE(d->n >= 0 && d->pixels >= 0 && d->c > 0 && d->groups > 0 && d->c % d->groups == 0, "%s: bad dimensions (%d, %d, %d) in %d groups", who,
	           d->n, d->pixels, d->c, d->groups);
	PZ_REQUIRE((long)d->n * d->groups < (1l << 31) && d->n <= 65535, "%s: %d samples of %d groups are too many", who, d->n, d->groups);
	return PZ_OK;
}

Norm args_of(const pz_groupnorm_desc *d) {
	Norm g{};
	g.n = d->n, g.pixels = d->pixels, g.c = d->c, g.groups = d->groups, g.width = d->c / d->groups;
	g.act = d->act, g.epsilon = d->epsilon;
	return g;
}

}  // namespace

extern "C" {

int pz_groupnorm_workspace_bytes(const pz_groupnorm_desc *d, int backward, size_t *nbytes) {
	if (int rc = check(d, "pz_groupnorm_workspace_bytes")) return rc;
	PZ_REQUIRE(nbytes, "pz_groupnorm_workspace_bytes: null output");
	*nbytes = backward ? (size_t)d->n * 2 * d->c * sizeof(float) : 0;
	return PZ_OK;
}

int pz_groupnorm_fwd(const pz_groupnorm_desc *d, const void *x, const float *scale, const float *bias, void *y, float *savemean, float *saveinvvar,
                     void *workspace, size_t ws_bytes, pz_stream_t stream) {
	if (int rc = check(d, "pz_groupnorm_fwd")) return rc;
	if (d->n == 0 || d->pixels == 0) return PZ_OK;
	PZ_REQUIRE(x && y, "pz_groupnorm_fwd: null tensor");
	Norm g = args_of(d);
	g.x = x, g.out = y, g.scale = scale, g.bias = bias, g.mean = savemean, g.invvar = saveinvvar;
	hipStream_t st = pz::as_stream(stream);
	if (d->dtype == PZ_F16) norm_fwd_kernel<f16><<<d->n * d->groups, 256, 0, st>>>(g);
	else norm_fwd_kernel<float><<<d->n * d->groups, 256, 0, st>>>(g);
	PZ_LAUNCH_CHECK();
	return PZ_OK;
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
	float *part = (float *)workspace;
	if (!empty) {
		if (dscale || dbias) {
			const dim3 grid((unsigned)pz::ceil_div(d->c, 256), (unsigned)d->n);
			if (d->dtype == PZ_F16) norm_channel_kernel<f16><<<grid, 256, 0, st>>>(g, part);
			else norm_channel_kernel<float><<<grid, 256, 0, st>>>(g, part);
			PZ_LAUNCH_CHECK();
		}
		if (d->dtype == PZ_F16) norm_bwd_kernel<f16><<<d->n * d->groups, 256, 0, st>>>(g);
		else norm_bwd_kernel<float><<<d->n * d->groups, 256, 0, st>>>(g);
		PZ_LAUNCH_CHECK();
	}
	if (dscale || dbias) {
		norm_param_kernel<<<pz::ceil_div(d->c, 256), 256, 0, st>>>(part, empty ? 0 : d->n, d->c, dscale, dbias);
		PZ_LAUNCH_CHECK();
	}
	return PZ_OK;
}

}  // extern "C"
