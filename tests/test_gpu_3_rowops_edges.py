"""
The operators over rows of channels on the device, beyond tests/test_gpu_3_rowops.py (whose plain forms in 64 bits and bounds it uses):
values at the ends of the types' ranges, row pitches whose multiples pass 32 bits, the tiles and slabs of large problems, streams.
"""
import numpy as np
import pytest

from puzzlelib_amd import lib
import test_gpu_3_rowops as rowops
from test_gpu_3_rowops import ACTS, NORMS, U32, Case, act, gpu, keep, productBound, put, slope, within, words

pytestmark = pytest.mark.gpu


# ------------------------------------------------------------------------------------------------ linear: values
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("name", ACTS)
def test_nothing_comes_through_a_dropped_element(bnd, dtype, name):
	"""pre-activations and gradients that are no numbers, in dropped places only: the gradients are those of finite values there, bit for bit"""
	c = Case(bnd, dtype, 40, 72, 136, seed=31)
	mask = bnd.DropoutMask(3, 8, 0.5)
	dropped = keep(mask, c.dy.shape) == 0
	z = np.random.RandomState(8).randn(*c.dy.shape).astype(dtype)
	dy, bad = c.dy.copy(), z.copy()
	places = np.flatnonzero(dropped)
	for values, at in ((bad, 0), (dy, 2)):
		for i, v in enumerate((np.nan, np.inf, -np.inf)):
			values.reshape(-1)[places[at + i::11]] = v

	def grads(dy, z):
		out = bnd.blas.linearBackward(gpu(bnd, dy), gpu(bnd, c.x), gpu(bnd, c.W), act=bnd.FusedAct[name], preact=gpu(bnd, z), dropout=mask)
		return [g.get() for g in out]

	for got, want in zip(grads(dy, bad), grads(np.where(dropped, dtype(0), c.dy), z)):
		assert np.isfinite(want).all() and np.array_equal(got, want)


@pytest.mark.parametrize("name,p,top", [("none", 0.875, 65504.0), ("relu", 0.75, 60000.0), ("gelu", 0.0, 65504.0), ("gelu", 0.875, 65504.0), ("silu", 0.5, 65504.0)])
def test_gradients_at_the_end_of_float16(bnd, name, p, top):
	"""dz = dy * act' / (1 - p) lies beyond float16, dx and dW do not"""
	m, k, n = 33, 72, 40
	c = Case(bnd, np.float16, m, k, n, seed=33)
	c.dy = (np.sign(c.dy.astype(np.float64)) * top).astype(np.float16)
	c.W, c.x = (c.W.astype(np.float32) / 512).astype(np.float16), (c.x.astype(np.float32) / 512).astype(np.float16)
	z = np.full((m, n), 1.5, np.float16)                                         # (slopes 1.128 and 1.04)
	mask = bnd.DropoutMask(6, 7, p) if p else None
	kept = keep(mask, (m, n)) * np.ones((m, n))
	dz = c.dy.astype(np.float64) * kept * slope(z.astype(np.float64), name)
	assert np.abs(dz).max() > 65504.0
	dx, dW, db = bnd.blas.linearBackward(
		gpu(bnd, c.dy), gpu(bnd, c.x), gpu(bnd, c.W), act=bnd.FusedAct[name], preact=gpu(bnd, z), dropout=mask
	)
	# without a curved activation dz is dy or zero times one factor: no rounding of its own. Behind one: half a step, and the slope's
	# own few roundings (exp and two products of values up to 1.13)
	curved = name in ("gelu", "silu")
	off = np.abs(dz) * ((2.0 ** -11 if curved else 0.0) + 32 * U32)
	x64, W64 = c.x.astype(np.float64), c.W.astype(np.float64)
	assert np.abs(dz @ W64.T).max() < 60000 and np.abs(x64.T @ dz).max() < 60000
	within(dx.get(), dz @ W64.T, productBound(dz, W64.T, n) + off @ np.abs(W64.T), "dx")
	within(dW.get(), x64.T @ dz, productBound(x64.T, dz, m) + np.abs(x64.T) @ off, "dW")
	within(db.get(), dz.sum(axis=0), off.sum(axis=0) + (m + 4) * U32 * np.abs(dz).sum(axis=0), "db")


@pytest.mark.parametrize("name", ["relu", "gelu", "silu"])
def test_pre_activations_beyond_float16(bnd, name):
	"""x W + b beyond 65504 either way: what the forward pass leaves is infinite, the output below is 0 and so is the slope; above it is 1"""
	m, k, n = 8, 16, 24
	x, W = np.full((m, k), 250.0, np.float16), np.full((k, n), 30.0, np.float16)
	W[:, ::2] = -30.0                                                              # z = +-120000
	y, z = bnd.blas.linear(gpu(bnd, x), gpu(bnd, W), act=bnd.FusedAct[name], preact=True)
	assert np.isneginf(z.get()[:, ::2]).all() and np.isposinf(z.get()[:, 1::2]).all() and np.all(y.get()[:, ::2] == 0)
	dy = np.random.RandomState(35).randn(m, n).astype(np.float16)
	dx, dW, db = bnd.blas.linearBackward(gpu(bnd, dy), gpu(bnd, x), gpu(bnd, W), act=bnd.FusedAct[name], preact=z)
	dz = np.where(np.arange(n) % 2 == 1, dy.astype(np.float64), 0.0)
	stored = 2.0 ** -11 * np.abs(dz) + 2.0 ** -24
	W64, x64 = W.astype(np.float64), x.astype(np.float64)
	within(dx.get(), dz @ W64.T, productBound(dz, W64.T, n) + stored @ np.abs(W64.T), "dx")
	within(dW.get(), x64.T @ dz, productBound(x64.T, dz, m) + np.abs(x64.T) @ stored, "dW")
	within(db.get(), dz.sum(axis=0), (m + 4) * U32 * np.abs(dz).sum(axis=0), "db")
	# NaN is not taken for either
	nan = gpu(bnd, np.full((m, n), np.nan, np.float16))
	assert name == "relu" or np.isnan(bnd.blas.linearBackward(gpu(bnd, dy), gpu(bnd, x), gpu(bnd, W), act=bnd.FusedAct[name], preact=nan)[2].get()).all()


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_a_mask_of_p_0_keeps_everything(bnd, dtype):
	"""word 1979 of call 117436 of seed 2026 is 2^32 - 1, the one word that does not lie below the threshold of p = 0"""
	seed, call, at, m, n = 2026, 117436, 1979, 32, 128
	assert words(seed, call, at + 1)[at] == 0xffffffff
	mask = bnd.DropoutMask(seed, call, 0.0)
	c = Case(bnd, dtype, m, 40, n, seed=34)
	args = gpu(bnd, c.x), gpu(bnd, c.W)
	plain = bnd.blas.linear(*args)
	assert plain.get().reshape(-1)[at] != 0 and np.array_equal(bnd.blas.linear(*args, dropout=mask).get(), plain.get())
	with_mask, without = (bnd.blas.linearBackward(gpu(bnd, c.dy), *args, dropout=d) for d in (mask, None))
	assert all(np.array_equal(a.get(), b.get()) for a, b in zip(with_mask, without))
	y = bnd.GPUArray.empty((m, n), dtype=dtype)
	bnd.counterDropoutKer(dtype)(y, plain, mask)
	assert np.array_equal(y.get(), plain.get())
	# through the C entries as well, whatever hands them the key
	lib.pz_dropout(lib.F32 if dtype == np.float32 else lib.F16, plain.rptr, None, y.optr, y.size, lib.byref(mask.key), None)
	assert np.array_equal(y.get(), plain.get())
	desc = lib.LinearDesc(lib.F32 if dtype == np.float32 else lib.F16, 0, 0, m, n, 40, 40, n, n, n, n)
	lib.pz_linear_fwd(lib.byref(desc), args[0].rptr, args[1].rptr, None, None, lib.byref(mask.key), y.optr, None, None, 0, None)
	assert np.array_equal(y.get(), plain.get())
	# one in 2^32 is what the stored form drops there; the smallest p that drops anything does too
	least = bnd.DropoutMask(seed, call, 2.0 ** -32)
	bnd.counterDropoutKer(dtype)(y, plain, least)
	assert y.get().reshape(-1)[at] == 0


def curve(z, name):
	"""value, slope in 64 bits, and what their evaluation in float32 may be off, as a bound of its own: u = 2^-24 a rounding, 2 u an exp2, a
	reciprocal or a rounded constant"""
	from scipy.special import erfc
	u, a = U32, np.abs(z)
	if name == "gelu":
		# tail = R e with e = exp(-z^2 / 2): the exponent z^2 / 2 log2(e) carries three roundings, which move e by 3 u z^2 / 2; R is a fit of
		# 1.2e-7 at a reciprocal, evaluated in eight steps whose terms add up to twice their sum at most
		tail, phi = 0.5 * erfc(a / np.sqrt(2.0)), np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)
		cdf = np.where(z < 0, tail, 1.0 - tail)
		rel = 1.2e-7 + (1.5 * z * z + 24) * u
		off = tail * rel + np.where(z < 0, 0.0, u)
		return z * cdf, a * off + 2 * u * np.abs(z * cdf), cdf + z * phi, off + a * phi * (rel + 4 * u) + 2 * u * (cdf + a * phi)
	# exp(-z): the exponent carries two roundings, 2 u |z|; s = 1 / (1 + exp(-z)) moves by that times 1 - s
	s, c = 1.0 / (1.0 + np.exp(-z)), 1.0 / (1.0 + np.exp(z))                      # (c = 1 - s)
	off = s * (c * (2 * a + 2) * u + 4 * u)
	return z * s, a * off + 2 * u * a * s, s * (1.0 + z * c), off * (1.0 + a * c) + s * (a * (off + u) + 2 * u * (1.0 + a * c))


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("name,far", [("gelu", 12.0), ("silu", 80.0)])
def test_activation_tails(bnd, dtype, name, far):
	"""the fused activations and their slopes over their whole range, through products with the identity: relative to the value itself, so that
	a tail of zeros does not pass"""
	k = 64
	z = np.concatenate((np.linspace(-far, far, 40 * k), np.linspace(-6.0, -2.0, 20 * k), np.linspace(-1.0, 1.0, 4 * k))).astype(dtype)
	z = np.concatenate((z, [0.0, -0.0, 1e-7, -1e-7], np.zeros(k - 4))).astype(dtype).reshape(-1, k)
	z64 = z.astype(np.float64)
	value, voff, der, doff = curve(z64, name)
	one = gpu(bnd, np.eye(k, dtype=dtype))
	y, pre = bnd.blas.linear(gpu(bnd, z), one, act=bnd.FusedAct[name], preact=True)
	assert np.array_equal(pre.get(), z)
	within(y.get(), value, voff, name)
	dx, _, db = bnd.blas.linearBackward(gpu(bnd, np.ones_like(z)), gpu(bnd, z), one, act=bnd.FusedAct[name], preact=pre)
	held = 0.0 if dtype == np.float32 else 2.0 ** -11 * np.abs(der) + 2.0 ** -24
	within(dx.get(), der, doff + held + 2 * U32 * np.abs(der), name + "'")
	within(db.get(), der.sum(axis=0), doff.sum(axis=0) + (z.shape[0] + 2) * U32 * np.abs(der).sum(axis=0), "sum of " + name + "'")


# ------------------------------------------------------------------------------------------------ linear: the tiles of large products
@pytest.fixture(scope="module")
def operands():
	"""one set of operands a type: (m, 4104), (4104, 4104) and gradients, of which each test takes a corner"""
	made = {}

	def get(dtype):
		if dtype not in made:
			rng = np.random.Generator(np.random.Philox(71))
			made[dtype] = [rng.standard_normal((4104, 4104), dtype=np.float32).astype(dtype) for _ in range(3)]
		return made[dtype]
	yield get
	made.clear()


# 256 x 256 tiles where there are 256 of them (k of 1024 on in float32, 256 in float16), 128 x 128 ones where more than 256 of those are; the
# last tile of every axis is ragged, and 2101 lies off 16 bytes
FORWARD = [(np.float32, 4000, 1100, 3908), (np.float16, 4000, 328, 3912), (np.float32, 2100, 516, 2108), (np.float16, 2100, 200, 2104), (np.float16, 2101, 201, 2101)]


@pytest.mark.parametrize("dtype,m,k,n", FORWARD)
@pytest.mark.parametrize("transpW", [False, True])
def test_large_tiles_forward(bnd, operands, dtype, m, k, n, transpW):
	a, b, c = operands(dtype)
	x, W, r = a[:m, :k], (b[:n, :k] if transpW else b[:k, :n]), c[:m, :n]
	bias = a[-1, :n].astype(np.float32)
	mask = bnd.DropoutMask(72, 1 << 33, 0.25)
	out, pre = bnd.blas.linear(gpu(bnd, x), gpu(bnd, W), gpu(bnd, bias), act=bnd.FusedAct.relu, dropout=mask, residual=gpu(bnd, r), preact=True, transpW=transpW)
	rows = np.unique(np.concatenate((np.arange(0, m, 53), [m - 1])))
	x64, W64 = x[rows].astype(np.float64), (W.T if transpW else W).astype(np.float64)
	z = x64 @ W64 + bias
	zb = productBound(x64, W64, k) + U32 * np.abs(z)
	within(pre.get()[rows], z, zb, "preact")
	kept = keep(mask, (m, n))[rows]
	y = act(z, "relu") * kept
	within(out.get()[rows], y + r[rows], zb * kept + 3 * U32 * (np.abs(y) + np.abs(r[rows].astype(np.float64))), "y")


BACKWARD = [(np.float32, 4000, 3908, 4100), (np.float16, 4000, 3912, 4104), (np.float32, 2100, 2108, 2116), (np.float16, 2100, 2104, 2120), (np.float16, 2101, 2099, 2101)]


@pytest.mark.parametrize("dtype,m,k,n", BACKWARD)
@pytest.mark.parametrize("transpW", [False, True])
def test_large_tiles_backward(bnd, operands, dtype, m, k, n, transpW):
	"""dx of m x k with n terms to a sum, dW of k x n with m: both in the tiles above, reduced along and across the rows"""
	a, b, c = operands(dtype)
	x, W, dy = a[:m, :k], (b[:n, :k] if transpW else b[:k, :n]), c[:m, :n]
	mask = bnd.DropoutMask(73, 2, 0.5)
	dx, dW, db = bnd.blas.linearBackward(gpu(bnd, dy), gpu(bnd, x), gpu(bnd, W), dropout=mask, transpW=transpW)
	dz = dy.astype(np.float64) * keep(mask, (m, n))                              # (dy doubled or nothing: no rounding)
	W64 = (W.T if transpW else W).astype(np.float64)
	rows = np.unique(np.concatenate((np.arange(0, m, 131), [m - 1])))
	got = dx.get()[rows]
	within(got, dz[rows] @ W64.T, productBound(dz[rows], W64.T, n), "dx")
	cols = np.unique(np.concatenate((np.arange(0, k, 127), [k - 1])))
	got = (dW.get().T if transpW else dW.get())[cols]
	xt = x[:, cols].T.astype(np.float64)
	within(got, xt @ dz, productBound(xt, dz, m), "dW")
	within(db.get(), dz.sum(axis=0), (m + 2) * U32 * np.abs(dz).sum(axis=0), "db")


# ------------------------------------------------------------------------------------------------ linear: few rows, far apart
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("rows,pitch", [(3, 1 << 28), (8, (1 << 27) - 8192), (2, 1 << 28)])
def test_a_tile_of_few_rows_far_apart(bnd, dtype, rows, pitch):
	"""A tile takes 32 (float16: 64) rows of an operand whose rows run along the reduction; the product of their number and such a pitch
	passes 32 bits, and there are rows of neither operand at the places that would wrap onto row 0. dW from x and dy, then x W with W in the buffer, all as
	columns of one buffer that holds NaN in between."""
	rng = np.random.RandomState(41)
	k, n = 16, 24
	x, dy, W = rng.randn(rows, k).astype(dtype), rng.randn(rows, n).astype(dtype), rng.randn(rows, n).astype(dtype)
	buf = bnd.GPUArray.empty((rows * pitch, ), dtype=dtype)
	buf.gpudata.fillD32(0x7fc07e00)                                 # NaN in either type
	cols = {"x": 0, "dy": 1024, "W": 4096}
	for name, ary in (("x", x), ("dy", dy), ("W", W)):
		put(buf, pitch, cols[name], ary)
	grid = buf.reshape(rows, pitch)
	view = lambda name, width: grid[:, cols[name]:cols[name] + width]

	x64, dy64, W64 = (a.astype(np.float64) for a in (x, dy, W))
	_, dW, db = bnd.blas.linearBackward(view("dy", n), view("x", k), gpu(bnd, np.zeros((k, n), dtype)), wantInput=False)
	within(dW.get(), x64.T @ dy64, productBound(x64.T, dy64, rows), "dW")
	within(db.get(), dy64.sum(axis=0), (rows + 2) * U32 * np.abs(dy64).sum(axis=0), "db")
	a = rng.randn(5, rows).astype(dtype)
	y = bnd.blas.linear(gpu(bnd, a), view("W", n))
	within(y.get(), a.astype(np.float64) @ W64, productBound(a.astype(np.float64), W64, rows), "y")
	# what stands in row 0 comes in once: an infinity does not meet the zeros behind the last column of a
	put(buf, pitch, cols["W"], np.full((1, n), np.inf, dtype))
	y = bnd.blas.linear(gpu(bnd, np.abs(a)), view("W", n)).get()
	assert np.isposinf(y).all()


# ------------------------------------------------------------------------------------------------ group norm
def test_groupnorm_of_many_values_to_a_group(bnd):
	"""4096 x 4100 values to one group, close together and far from zero: every value's rounding would fall the same way in a long float32 sum"""
	shape, u = (1, 4096, 4100), U32
	rng = np.random.RandomState(61)
	x = (1.1 + 1e-3 * rng.randn(*shape)).astype(np.float32)
	dy = (1.1 + 1e-3 * rng.randn(*shape)).astype(np.float32)
	gx = gpu(bnd, x)
	y, gm, gv = bnd.dnn.groupNormNd(gx, None, None, 1)
	x64, dy64 = x.astype(np.float64), dy.astype(np.float64)
	mean, var = x64.mean(), x64.var()
	invvar = 1.0 / np.sqrt(var + 1e-5)
	# the mean and 1 / sqrt are rounded once; a centred value is off by a rounding and the mean's, so that the variance moves by twice that
	dmean = u * mean
	dinv = invvar * 4 * (dmean * invvar + u)
	within(gm.get(), np.full((1, 1), mean), 0.0, "mean")
	within(gv.get(), np.full((1, 1), invvar), dinv, "invvar")
	xhat = (x64 - mean) * invvar
	within(y.get(), xhat, np.abs(xhat) * (dinv / invvar + 3 * u) + 2 * dmean * invvar, "y")

	m32, i32 = np.full((1, 1), mean, np.float32), np.full((1, 1), invvar, np.float32)
	xh = (x64 - np.float64(m32[0, 0])) * np.float64(i32[0, 0])
	a, b = dy64.mean(), (dy64 * xh).mean()
	dx = np.float64(i32[0, 0]) * (dy64 - a - xh * b)
	# xhat: a rounding of the difference (up to |x| in size, exact here: both lie within a factor of two) and one of the product; products and
	# differences of values up to dy
	off = 4 * u * (np.abs(dy64) + np.abs(xh * b) + np.abs(xh))
	got, _, _ = bnd.dnn.groupNormNdBackward(gpu(bnd, dy), gx, None, None, gpu(bnd, m32), gpu(bnd, i32), 1)
	within(got.get(), dx, np.float64(i32[0, 0]) * off, "dx")


# A slab is 128 bytes of channels wide, or 64 (two workgroups then share a line), where a workgroup of 512 or 1024 threads holds all pixels of it:
# up to 1024 (128 bytes, 512 threads), 2048 (64 bytes), 4096 (64 bytes, 1024 threads) forward, half as many backward; whole groups of 128
# bytes take 1024 threads at once. At least 128 such slabs, or the pixels are cut into chunks. Last: more samples than slabs of a power of two.
LARGE = [((16, 999, 512), 32), ((8, 1999, 512), 32), ((8, 3999, 512), 32), ((16, 1777, 512), 8), ((16, 333, 512), 32), ((8, 777, 512), 32), ((16, 901, 512), 8),
		 ((43, 700, 192), 12)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", LARGE)
def test_groupnorm_large_slabs(bnd, dtype, shape, groups):
	if dtype == np.float32:
		shape = shape[:2] + (shape[2] // 2, )                                       # (the same bytes a row)
	rowops.test_groupnorm(bnd, dtype, shape, groups // 2 if dtype == np.float32 else groups, "silu")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", LARGE)
@pytest.mark.parametrize("name", ["relu", "silu"])
def test_groupnorm_backward_large_slabs(bnd, dtype, shape, groups, name):
	if dtype == np.float32:
		shape = shape[:2] + (shape[2] // 2, )
	rowops.test_groupnorm_backward(bnd, dtype, shape, groups // 2 if dtype == np.float32 else groups, name)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", NORMS)
def test_groupnorm_backward_gelu(bnd, dtype, shape, groups):
	rowops.test_groupnorm_backward(bnd, dtype, shape, groups, "gelu")


# rows of all channels that no workgroup holds, next to the ones that one just does: float32 above 1024 channels, float16 above 2048
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", [((2, 70, 1024), 1), ((1, 90, 1028), 1), ((2, 400, 1280), 32), ((1, 50, 2056), 1), ((2, 300, 2560), 32), ((3, 40, 4096), 1)])
def test_groupnorm_many_channels(bnd, dtype, shape, groups):
	rowops.test_groupnorm(bnd, dtype, shape, groups, "silu")
	rowops.test_groupnorm_backward(bnd, dtype, shape, groups, "silu")


# ------------------------------------------------------------------------------------------------ streams
def test_casts_costs_and_user_kernels_on_a_stream_around_a_product(bnd):
	"""what a mixed-precision step would put beside its float16 product on a borrowed stream: each launch waits for the one whose result it takes"""
	rng = np.random.RandomState(51)
	m, k, n = 512, 384, 640
	W = (rng.randn(k, n) / 16).astype(np.float16)
	gW = gpu(bnd, W)
	stream = bnd.Driver.Stream()
	twice = bnd.ElementwiseKernel([("float *", "out"), ("const float *", "data")], "out[i] = 2.0f * data[i]", "twiceKer")
	E = lambda shape, dtype: bnd.GPUArray.empty(shape, dtype=dtype)
	for call in range(3):
		x = rng.randn(m, k).astype(np.float32)
		master, h, y32, t, g, err = E((m, k), np.float32), E((m, k), np.float16), E((m, n), np.float32), E((m, n), np.float32), E((m, n), np.float32), gpu(bnd, np.zeros((1, ), np.float32))
		master.set(gpu(bnd, x), stream=stream)
		bnd.castFP32toFP16(h, master, stream=stream)
		y = bnd.blas.linear(h, gW)
		bnd.castFP16toFP32(y32, y, stream=stream)
		twice(t, y32, stream=stream)
		bnd.smoothL1Ker(t, y32, err, g, 1.0, 1.0, stream=stream)
		z = bnd.blas.linear(y, gpu(bnd, np.eye(n, dtype=np.float16)))                   # another product while the stream still works
		want = y.get().astype(np.float32)
		x16 = x.astype(np.float16).astype(np.float64)
		assert np.array_equal(h.get().astype(np.float64), x16)
		within(y.get(), x16 @ W, productBound(x16, W.astype(np.float64), k), "y")
		assert np.array_equal(y32.get(), want) and np.array_equal(t.get(stream=stream), 2.0 * want) and np.array_equal(z.get(), y.get())
		assert np.isfinite(err.get()).all() and np.isfinite(g.get()).all()
