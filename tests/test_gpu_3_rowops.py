"""
The operators over rows of channels on the device — blas.linear / linearBackward, counterDropoutKer, dnn.groupNormNd /
groupNormNdBackward — against plain numpy in 64 bits: float32 and float16, every layout of the weights, lengths from one row,
odd sizes, row pitches, in-place forms, empty tensors; gradients against the formulas' and against differences.

Tolerances. A rounding is off by at most half a step: u = 2^-24 (float32), 2^-11 (float16) relative to the value. `within` allows one
rounding of the output besides the bound that each test derives from the roundings in front of it; sums of m terms carry at most m
roundings of their partial sums, whatever the order.
"""
import numpy as np
import pytest

pytestmark = pytest.mark.gpu

U = {np.dtype(np.float32): 2.0 ** -24, np.dtype(np.float16): 2.0 ** -11}
TINY = {np.dtype(np.float32): 1e-37, np.dtype(np.float16): 2.0 ** -25}       # half the smallest step of the type


def gpu(bnd, a):
	return bnd.GPUArray.toGpu(np.ascontiguousarray(a))


# ------------------------------------------------------------------------------------------------ plain forms in 64 bits
def erf(x):
	from math import erf as one
	return np.vectorize(one, otypes=[np.float64])(x)


def act(z, name):
	if name == "relu":
		return np.where(z > 0, z, 0.0)
	if name == "gelu":
		return 0.5 * z * (1.0 + erf(z / np.sqrt(2.0)))
	if name == "silu":
		return z / (1.0 + np.exp(-z))
	return z


def slope(z, name):
	if name == "relu":
		return (z > 0).astype(np.float64)
	if name == "gelu":
		return 0.5 * (1.0 + erf(z / np.sqrt(2.0))) + z * np.exp(-0.5 * z * z) / np.sqrt(2.0 * np.pi)
	if name == "silu":
		s = 1.0 / (1.0 + np.exp(-z))
		return s * (1.0 + z * (1.0 - s))
	return np.ones_like(z)


def wordsFrom(seed, call, quad, quads):
	"""Philox4x32-10 in numpy: the words of call `call` from word 4 * quad on"""
	mask = np.uint64(0xffffffff)
	q = np.arange(quad, quad + quads, dtype=np.uint64)
	c = [q & mask, q >> np.uint64(32), np.full_like(q, call & 0xffffffff), np.full_like(q, call >> 32)]
	k = [seed & 0xffffffff, seed >> 32]
	for _ in range(10):
		a, b = c[0] * np.uint64(0xD2511F53), c[2] * np.uint64(0xCD9E8D57)
		c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & mask, (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & mask]
		k = [(k[0] + 0x9E3779B9) & 0xffffffff, (k[1] + 0xBB67AE85) & 0xffffffff]
	return np.stack(c, axis=1).reshape(-1)


def words(seed, call, count):
	return wordsFrom(seed, call, 0, (count + 3) // 4)[:count]


def keep(mask, shape):
	if mask is None:
		return 1.0
	kept = words(mask.seed, mask.call, int(np.prod(shape))) < np.uint64(int((1.0 - mask.p) * 0xffffffff))
	return kept.reshape(shape) / (1.0 - mask.p)


def within(actual, desired, bound, what):
	"""|actual - desired| <= bound + one rounding of the output"""
	assert actual.shape == desired.shape, "%s: %s vs %s" % (what, actual.shape, desired.shape)
	u = U[actual.dtype]
	err = np.abs(actual.astype(np.float64) - desired)
	limit = bound * (1.0 + 2.0 * u) + u * np.abs(desired) + TINY[actual.dtype]
	bad = ~(err <= limit)
	assert not bad.any(), "%s: %d of %d off, worst %.3g of its bound, at %s" % (
		what, bad.sum(), bad.size, float(np.nanmax(err / limit)), np.argwhere(bad)[:3].tolist()
	)


U32 = 2.0 ** -24


def productBound(a, b, terms):
	"""A sum of `terms` exact products (float16) or rounded ones (float32) accumulated in float32: every partial sum and product is
	rounded once, so the error is at most (terms + 1) u32 sum |a||b| in any order; +1 ulp where the order folds partial sums again."""
	return (terms + 2) * U32 * (np.abs(a) @ np.abs(b))


# an activation moves an error of its argument by at most its steepest slope (1.13 for gelu, 1.1 for silu); its own evaluation in
# float32 is a few roundings of values of the argument's size — for the float16 forms a polynomial of relative error 2^-14 or better
LIPSCHITZ = 1.13


def actBound(z, name, dtype):
	if name in ("none", "relu"):
		return 0.0
	return np.abs(z) * (16 * U32 if dtype == np.float32 else 2.0 ** -14)


ACTS = ("none", "relu", "gelu", "silu")


class Case:
	def __init__(self, bnd, dtype, m, k, n, seed=0, transpW=False, rows=None):
		rng = np.random.RandomState(seed)
		self.bnd, self.dtype = bnd, np.dtype(dtype)
		self.x = rng.randn(m, k).astype(dtype)
		self.W = (rng.randn(*((n, k) if transpW else (k, n))) / np.sqrt(k)).astype(dtype)
		self.b = (0.1 * rng.randn(n)).astype(np.float32)
		self.r = rng.randn(m, n).astype(dtype)
		self.dy = rng.randn(m, n).astype(dtype)
		self.transpW = transpW
		self.x64 = self.x.astype(np.float64)
		self.W64 = (self.W.T if transpW else self.W).astype(np.float64)

	def forward(self, name="none", mask=None, residual=False, bias=True):
		"""(z, its bound, y, its bound)"""
		k = self.x.shape[1]
		z = self.x64 @ self.W64 + (self.b if bias else 0.0)
		zb = productBound(self.x64, self.W64, k) + U32 * np.abs(z)
		kp = keep(mask, z.shape)
		y = act(z, name) * kp
		yb = (zb * LIPSCHITZ + actBound(z, name, self.dtype)) * kp + 2 * U32 * np.abs(y)
		if residual:
			y = y + self.r.astype(np.float64)
			yb = yb + U32 * np.abs(y)
		return z, zb, y, yb


SIZES = [(1, 64, 64), (1, 65, 67), (2, 8, 1), (3, 1, 5), (7, 130, 96), (16, 256, 512), (33, 129, 257), (64, 64, 64), (65, 72, 130),
		 (128, 192, 256), (200, 100, 72), (257, 320, 264), (129, 1000, 60), (5, 2056, 1048)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("m,k,n", SIZES)
@pytest.mark.parametrize("transpW", [False, True])
def test_linear_sizes(bnd, dtype, m, k, n, transpW):
	c = Case(bnd, dtype, m, k, n, seed=m + k + n, transpW=transpW)
	z, zb, y, yb = c.forward()
	out = bnd.blas.linear(gpu(bnd, c.x), gpu(bnd, c.W), gpu(bnd, c.b), transpW=transpW)
	assert out.dtype == c.dtype
	within(out.get(), y, yb, "y")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("p", [0.0, 0.25])
@pytest.mark.parametrize("m,k,n", [(70, 136, 200), (70, 136, 203), (1, 40, 77)])
def test_linear_epilogue(bnd, dtype, name, p, m, k, n):
	c = Case(bnd, dtype, m, k, n, seed=5)
	mask = bnd.DropoutMask(0x1234567890abcdef, 11, p)
	z, zb, y, yb = c.forward(name, mask if p else None, residual=True)
	out, preact = bnd.blas.linear(
		gpu(bnd, c.x), gpu(bnd, c.W), gpu(bnd, c.b), act=bnd.FusedAct[name], dropout=mask, residual=gpu(bnd, c.r), preact=True
	)
	within(preact.get(), z, zb, "preact")
	within(out.get(), y, yb, "y")
	# no bias, no residual, nothing kept
	z, zb, y, yb = c.forward(name, bias=False)
	within(bnd.blas.linear(gpu(bnd, c.x), gpu(bnd, c.W), act=bnd.FusedAct[name]).get(), y, yb, "bare")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("m,k,n", [(1024, 1024, 1024), (2048, 320, 2304), (300, 4104, 296), (4096, 256, 4096)])
def test_linear_large_tiles(bnd, dtype, m, k, n):
	"""the tiles and splits that only larger products take; rows sampled"""
	c = Case(bnd, dtype, m, k, n, seed=9)
	mask = bnd.DropoutMask(7, 1 << 40, 0.1)
	out = bnd.blas.linear(gpu(bnd, c.x), gpu(bnd, c.W), gpu(bnd, c.b), act=bnd.FusedAct.relu, dropout=mask, residual=gpu(bnd, c.r)).get()
	kp = keep(mask, (m, n))
	rows = np.unique(np.concatenate((np.arange(0, m, 37), [m - 1])))
	c.x64, c.r = c.x64[rows], c.r[rows]
	z, zb, y, yb = c.forward("relu", None, residual=False)
	y, yb = y * kp[rows] + c.r.astype(np.float64), yb * kp[rows] + 4 * U32 * (np.abs(y) * kp[rows] + np.abs(c.r))
	within(out[rows], y, yb, "y")


def backwardOracle(c, name, mask, z):
	"""dz in 64 bits and the bound of what the kernels hold for it: in float16 one rounding"""
	kp = keep(mask, c.dy.shape)
	dz = c.dy.astype(np.float64) * kp * slope(z, name)
	eps = 24 * U32 if c.dtype == np.float32 else 2.0 ** -13
	gate = np.abs(c.dy.astype(np.float64)) * kp * (1.13 * eps if name in ("gelu", "silu") else 4 * U32)
	stored = gate if c.dtype == np.float32 or (name == "none" and mask is None) else gate + 2.0 ** -11 * np.abs(dz) + 2.0 ** -25
	return dz, gate, stored


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("p", [0.0, 0.5])
@pytest.mark.parametrize("m,k,n,transpW", [(40, 72, 136, False), (40, 72, 136, True), (67, 33, 129, False), (67, 33, 129, True), (1, 64, 40, False),
											(300, 264, 520, False)])
def test_linear_backward(bnd, dtype, name, p, m, k, n, transpW):
	c = Case(bnd, dtype, m, k, n, seed=3, transpW=transpW)
	mask = bnd.DropoutMask(99, 5, p) if p else None
	z = np.random.RandomState(8).randn(m, n).astype(dtype)
	dz, gate, stored = backwardOracle(c, name, mask, z.astype(np.float64))
	dx, dW, db = bnd.blas.linearBackward(
		gpu(bnd, c.dy), gpu(bnd, c.x), gpu(bnd, c.W), act=bnd.FusedAct[name], preact=gpu(bnd, z), dropout=mask, transpW=transpW
	)
	assert dx.dtype == dW.dtype == c.dtype and db.dtype == np.float32
	within(dx.get(), dz @ c.W64.T, productBound(dz, c.W64.T, n) + stored @ np.abs(c.W64.T) * 1.01, "dx")
	want, bound = c.x64.T @ dz, productBound(c.x64.T, dz, m) + np.abs(c.x64.T) @ stored * 1.01
	within(dW.get(), want.T if transpW else want, bound.T if transpW else bound, "dW")
	within(db.get(), dz.sum(axis=0), gate.sum(axis=0) + (m + 2) * U32 * np.abs(dz).sum(axis=0), "db")


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("wide", [False, True])
def test_linear_backward_accumulates(bnd, dtype, wide):
	"""dst = momentum * dst + scale * d into float32 gradients (or the operands' type), one of the outputs alone"""
	m, k, n = 50, 88, 61
	c = Case(bnd, dtype, m, k, n, seed=4)
	wtype = np.float32 if wide else dtype
	rng = np.random.RandomState(1)
	w0, b0 = rng.randn(k, n).astype(wtype), rng.randn(n).astype(np.float32)
	dw, db = gpu(bnd, w0), gpu(bnd, b0)
	w0, b0 = w0.astype(np.float64), b0.astype(np.float64)
	args = (gpu(bnd, c.dy), gpu(bnd, c.x), gpu(bnd, c.W))
	none, dw2, db2 = bnd.blas.linearBackward(*args, wgrad=dw, bgrad=db, scale=0.5, momentum=0.75, wantInput=False)
	assert none is None and dw2 is dw and db2 is db
	dz = c.dy.astype(np.float64)
	bound = productBound(c.x64.T, dz, m)
	within(dw.get(), 0.75 * w0 + 0.5 * (c.x64.T @ dz), 0.5 * bound + 3 * U32 * (np.abs(w0) + np.abs(c.x64.T @ dz)), "dW")
	within(db.get(), 0.75 * b0 + 0.5 * dz.sum(axis=0), (m + 4) * U32 * (np.abs(dz).sum(axis=0) + np.abs(b0)), "db")
	dx, nw, nb = bnd.blas.linearBackward(*args, wantParams=False)
	assert nw is None and nb is None
	within(dx.get(), dz @ c.W64.T, productBound(dz, c.W64.T, n), "dx alone")
	_, dw3, nb = bnd.blas.linearBackward(*args, withbias=False, wantInput=False)
	assert nb is None
	within(dw3.get(), c.x64.T @ dz, bound, "dW without a bias")


def test_linear_gradients_against_differences(bnd):
	"""the directional derivative of sum(g * y) in float32: central differences of the forward pass, step h: error h^2/6 f''' + u f / h"""
	m, k, n = 12, 20, 24
	c = Case(bnd, np.float32, m, k, n, seed=21)
	mask = bnd.DropoutMask(1, 2, 0.25)
	rng = np.random.RandomState(2)
	for name in ("gelu", "silu"):
		actId = bnd.FusedAct[name]

		def f(x, W, b, r):
			y = bnd.blas.linear(gpu(bnd, x), gpu(bnd, W), gpu(bnd, b), act=actId, dropout=mask, residual=gpu(bnd, r)).get()
			return float((y.astype(np.float64) * c.dy).sum())

		_, z = bnd.blas.linear(gpu(bnd, c.x), gpu(bnd, c.W), gpu(bnd, c.b), act=actId, dropout=mask, preact=True)
		dx, dW, db = bnd.blas.linearBackward(gpu(bnd, c.dy), gpu(bnd, c.x), gpu(bnd, c.W), act=actId, preact=z, dropout=mask)
		grads = [dx.get(), dW.get(), db.get(), c.dy]
		at = [c.x, c.W, c.b, c.r]
		for i in range(4):
			d = rng.randn(*at[i].shape).astype(np.float32)
			d /= np.linalg.norm(d)
			h = 2.0 ** -6
			plus, minus = list(at), list(at)
			plus[i], minus[i] = at[i] + np.float32(h) * d, at[i] - np.float32(h) * d
			# the points in float32 are off the line by u |point|; along it their distance is what they say
			step = float(((plus[i].astype(np.float64) - minus[i]) * d).sum())
			numeric = (f(*plus) - f(*minus)) / step
			exact = float((grads[i].astype(np.float64) * d).sum())
			# third derivatives of gelu / silu stay below 1.7 and the direction has norm 1; |dy| sums to about m n
			assert abs(numeric - exact) <= 2e-3 * (1.0 + abs(exact)), (name, i, numeric, exact)


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_linear_row_pitches_in_place_and_axes(bnd, dtype):
	m, k, n = 37, 64, 96
	rng = np.random.RandomState(6)
	big = rng.randn(m, 3 * 128).astype(dtype)
	W = (rng.randn(k, 2 * n) / 8).astype(dtype)
	x, Wv = big[:, 128:128 + k], W[:, n:]
	gbig, gW = gpu(bnd, big), gpu(bnd, W)
	res = rng.randn(m, 200).astype(dtype)
	gres = gpu(bnd, res)
	view = gres[:, 8:8 + n]
	y = x.astype(np.float64) @ Wv.astype(np.float64) + res[:, 8:8 + n]
	bound = productBound(x.astype(np.float64), Wv.astype(np.float64), k) + 2 * U32 * np.abs(y)
	out = bnd.blas.linear(gbig[:, 128:128 + k], gW[:, n:], residual=view, out=view)          # in place, inside wider rows
	assert out is view
	now = gres.get()
	within(now[:, 8:8 + n], y, bound, "columns in place")
	assert np.array_equal(now[:, :8], res[:, :8]) and np.array_equal(now[:, 8 + n:], res[:, 8 + n:]), "neighbours were written"
	# a row pitch and a start that no 16-byte load can use
	odd = bnd.blas.linear(gbig[:, 1:1 + k], gW[:, 3:3 + 5])
	xo, Wo = big[:, 1:1 + k].astype(np.float64), W[:, 3:8].astype(np.float64)
	within(odd.get(), xo @ Wo, productBound(xo, Wo, k), "odd view")
	# leading axes
	cube = bnd.blas.linear(gpu(bnd, big[:36]).reshape(4, 9, 384), gpu(bnd, (rng.randn(384, 8) / 16).astype(dtype)))
	assert cube.shape == (4, 9, 8)
	# side by side columns of one buffer
	left, right = gres[:, :n], gres[:, 100:100 + n]
	rl = now[:, :n].astype(np.float64)
	Wq = (rng.randn(n, n) / 10).astype(dtype)
	bnd.blas.linear(left, gpu(bnd, Wq), out=right)
	after = gres.get()
	within(after[:, 100:100 + n], rl @ Wq, productBound(rl, Wq.astype(np.float64), n), "side by side")
	assert np.array_equal(after[:, :100], now[:, :100])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_linear_nothing_to_do_and_values_that_are_not_numbers(bnd, dtype):
	W = np.eye(16, 24).astype(dtype)
	out = bnd.blas.linear(gpu(bnd, np.zeros((0, 16), dtype)), gpu(bnd, W))
	assert out.shape == (0, 24)
	wgrad, bgrad = gpu(bnd, np.ones((16, 24), np.float32)), gpu(bnd, np.ones(24, np.float32))
	dx, dw, db = bnd.blas.linearBackward(
		gpu(bnd, np.zeros((0, 24), dtype)), gpu(bnd, np.zeros((0, 16), dtype)), gpu(bnd, W), wgrad=wgrad, bgrad=bgrad, momentum=0.5
	)
	assert dx.shape == (0, 16) and np.all(dw.get() == 0.5) and np.all(db.get() == 0.5)
	# a NaN or an infinity stays in its row
	x = np.ones((5, 16), dtype)
	x[1, 3], x[3, 3] = np.nan, np.inf
	y = bnd.blas.linear(gpu(bnd, x), gpu(bnd, np.abs(W) + dtype(1)), act=bnd.FusedAct.relu).get()
	assert np.isnan(y[1]).all() and np.isposinf(y[3]).all() and np.isfinite(y[[0, 2, 4]]).all()
	# a dropped element is zero whatever it holds
	mask = bnd.DropoutMask(3, 4, 0.5)
	y = bnd.blas.linear(gpu(bnd, x), gpu(bnd, np.abs(W) + dtype(1)), dropout=mask).get()
	kept = keep(mask, (5, 24)) > 0
	assert np.all(y[~kept] == 0) and np.isnan(y[1][kept[1]]).all() and np.isposinf(y[3][kept[3]]).all()


def test_linear_twice_is_the_same_bits(bnd):
	for dtype in (np.float32, np.float16):
		c = Case(bnd, dtype, 150, 1032, 72, seed=2)
		args = gpu(bnd, c.x), gpu(bnd, c.W), gpu(bnd, c.b)
		first = bnd.blas.linear(*args).get()
		grads = [g.get() for g in bnd.blas.linearBackward(gpu(bnd, c.dy), *args[:2])]
		for _ in range(3):
			assert np.array_equal(bnd.blas.linear(*args).get(), first)
			assert all(np.array_equal(a, b.get()) for a, b in zip(grads, bnd.blas.linearBackward(gpu(bnd, c.dy), *args[:2])))


# ------------------------------------------------------------------------------------------------ dropout
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("count", [1, 3, 4, 7, 8, 63, 1000, 4097, 70001])
@pytest.mark.parametrize("p", [0.0, 0.1, 0.5, 0.97])
def test_counter_dropout(bnd, dtype, count, p):
	rng = np.random.RandomState(count)
	x, r = rng.randn(count).astype(dtype), rng.randn(count).astype(dtype)
	mask = bnd.DropoutMask((1 << 63) + 12345, (1 << 33) + 1, p)
	y, gx = bnd.GPUArray.empty((count, ), dtype=dtype), gpu(bnd, x)
	ker = bnd.counterDropoutKer(dtype)
	ker(y, gx, mask)
	want = x.astype(np.float64) * keep(mask, (count, ))
	# keep is a float32 number (u32), the quotient is rounded to float32 (u32), then to the type
	within(y.get(), want, 3 * U32 * np.abs(want), "y")
	assert np.array_equal(y.get() == 0, (want == 0)), "the mask"
	ker(y, gx, mask, residual=gpu(bnd, r))
	within(y.get(), want + r.astype(np.float64), 3 * U32 * np.abs(want) + U32 * np.abs(want + r), "y + residual")
	ker(gx, gx, mask)                                                               # in place
	within(gx.get(), want, 3 * U32 * np.abs(want), "in place")
	gr = gpu(bnd, r)
	ker(gr, gpu(bnd, x), mask, residual=gr)
	within(gr.get(), want + r.astype(np.float64), 3 * U32 * np.abs(want) + U32 * np.abs(want + r), "onto the residual")


def test_counter_dropout_is_the_stored_form(bnd):
	"""fillInteger + dropoutKer (Modules/Dropout.py:33-58) and a mask of the generator's same call give the same values"""
	n, p = 100003, 0.3
	x = gpu(bnd, np.random.RandomState(0).randn(n).astype(np.float32))
	stored, counted = bnd.RandomNumberGenerator(seed=77), bnd.RandomNumberGenerator(seed=77)
	for _ in range(3):
		bits = bnd.GPUArray.empty((n, ), dtype=np.uint32)
		stored.fillInteger(bits)
		a, b = bnd.GPUArray.empty((n, ), dtype=np.float32), bnd.GPUArray.empty((n, ), dtype=np.float32)
		keepProb = 1.0 - p
		bnd.dropoutKer(np.float32)(a, x, bits, int(keepProb * 0xffffffff), np.float32(keepProb))
		mask = counted.dropoutMask(p)
		bnd.counterDropoutKer(np.float32)(b, x, mask)
		assert np.array_equal(a.get(), b.get())
		share = float((b.get() != 0).mean())
		assert abs(share - keepProb) < 6 * np.sqrt(p * keepProb / n)                     # six standard deviations
	# unaligned views, another stream
	stream = bnd.Driver.Stream()
	big = gpu(bnd, np.random.RandomState(1).randn(1001).astype(np.float16))
	out = bnd.GPUArray.empty((1003, ), dtype=np.float16)
	bnd.counterDropoutKer(np.float16)(out[1:1001], big[1:], mask, stream=stream)
	want = big.get()[1:].astype(np.float64) * keep(mask, (1000, ))
	within(out.get()[1:1001], want, 3 * U32 * np.abs(want), "a view on a stream")
	# what is dropped is zero whatever it held
	bad = np.full(64, np.nan, np.float32)
	y = bnd.GPUArray.empty((64, ), dtype=np.float32)
	bnd.counterDropoutKer(np.float32)(y, gpu(bnd, bad), mask)
	kept = keep(mask, (64, )) > 0
	assert np.isnan(y.get()[kept]).all() and np.all(y.get()[~kept] == 0)


# ------------------------------------------------------------------------------------------------ group norm
def normOracle(x, scale, bias, groups, eps, name):
	n, c = x.shape[0], x.shape[-1]
	x64 = x.astype(np.float64).reshape(n, -1, groups, c // groups)
	mean = x64.mean(axis=(1, 3))
	var = ((x64 - mean[:, None, :, None]) ** 2).mean(axis=(1, 3))
	invvar = 1.0 / np.sqrt(var + eps)
	xhat = (x64 - mean[:, None, :, None]) * invvar[:, None, :, None]
	t = xhat * (1.0 if scale is None else scale.astype(np.float64).reshape(groups, -1)) + (0.0 if bias is None else bias.astype(np.float64).reshape(groups, -1))
	return mean, invvar, xhat, t


def normBounds(x, mean, invvar, groups):
	"""mean: m roundings of the running sum, of values up to max|x| of the group; 1/sqrt(var + eps): the centred squares carry 2 (d mean) /
	sigma relative and m roundings; xhat: both"""
	n, c = x.shape[0], x.shape[-1]
	x64 = np.abs(x.astype(np.float64)).reshape(n, -1, groups, c // groups)
	m = x64.shape[1] * x64.shape[3]
	steps = 8 + 2 * np.sqrt(m)                      # roundings that add up: partial sums are short (a thread's, a wave's, a block's)
	dmean = steps * U32 * x64.mean(axis=(1, 3)) + U32 * np.abs(mean)
	dinv = invvar * (steps * U32 + 4 * U32 + 0.5 * (dmean * invvar) ** 2 + 2.0 * U32 * x64.max(axis=(1, 3)) * invvar)
	return dmean, dinv


NORMS = [((2, 64, 64), 8), ((1, 1, 32), 2), ((3, 5, 7, 30), 3), ((2, 49, 320), 32), ((4, 16), 1), ((1, 300, 24), 24), ((2, 1000, 8), 2),
		 ((1, 17, 2048), 1), ((2, 2500, 64), 4), ((3, 1100, 40), 4), ((5, 33, 96), 3), ((1, 9000, 48), 3), ((2, 100, 1030), 103), ((70, 1, 128), 8)]


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", NORMS)
@pytest.mark.parametrize("name", ACTS)
def test_groupnorm(bnd, dtype, shape, groups, name):
	rng = np.random.RandomState(sum(shape))
	c = shape[-1]
	x = (rng.randn(*shape) * 1.5 + rng.randn(c)).astype(dtype)
	scale, bias = (1.0 + 0.1 * rng.randn(c)).astype(np.float32), (0.1 * rng.randn(c)).astype(np.float32)
	mean, invvar, xhat, t = normOracle(x, scale, bias, groups, 1e-5, name)
	dmean, dinv = normBounds(x, mean, invvar, groups)
	gx = gpu(bnd, x)
	out, gm, gv = bnd.dnn.groupNormNd(gx, gpu(bnd, scale), gpu(bnd, bias), groups, act=bnd.FusedAct[name])
	within(gm.get(), mean, dmean, "mean")
	within(gv.get(), invvar, dinv, "invvar")
	wide = lambda a: a[:, None, :, None]
	dt = np.abs(scale.reshape(groups, -1)) * (np.abs(xhat) * wide(dinv / invvar) + wide(dmean * invvar) + 4 * U32 * np.abs(xhat) + U32 * wide(np.abs(mean) * invvar)) + 2 * U32 * np.abs(t)
	y = act(t, name)
	within(out.get(), y.reshape(shape), (dt * LIPSCHITZ + actBound(t, name, np.dtype(dtype))).reshape(shape), "y")
	assert np.array_equal(gx.get(), x)
	test = bnd.dnn.groupNormNd(gx, gpu(bnd, scale), gpu(bnd, bias), groups, act=bnd.FusedAct[name], test=True)
	assert np.array_equal(test.get(), out.get())
	again, _, _ = bnd.dnn.groupNormNd(gx, gpu(bnd, scale), gpu(bnd, bias), groups, act=bnd.FusedAct[name], out=gx)      # in place
	assert again is gx and np.array_equal(gx.get(), out.get())


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
@pytest.mark.parametrize("shape,groups", NORMS)
@pytest.mark.parametrize("name", ["none", "relu", "silu"])
def test_groupnorm_backward(bnd, dtype, shape, groups, name):
	rng = np.random.RandomState(sum(shape) + 1)
	n, c = shape[0], shape[-1]
	x = (rng.randn(*shape) * 1.5 + rng.randn(c)).astype(dtype)
	dy = rng.randn(*shape).astype(dtype)
	scale, bias = (1.0 + 0.1 * rng.randn(c)).astype(np.float32), (0.1 * rng.randn(c)).astype(np.float32)
	mean, invvar, _, _ = normOracle(x, scale, bias, groups, 1e-5, name)
	mean, invvar = mean.astype(np.float32), invvar.astype(np.float32)         # what the backward pass is given

	x64 = x.astype(np.float64).reshape(n, -1, groups, c // groups)
	m = x64.shape[1] * x64.shape[3]
	wide = lambda a: a.astype(np.float64)[:, None, :, None]
	xhat = (x64 - wide(mean)) * wide(invvar)
	g = scale.astype(np.float64).reshape(groups, -1)
	t = xhat * g + bias.reshape(groups, -1)
	dt = 4 * U32 * (np.abs(xhat) + np.abs(t) + wide(np.abs(mean) * invvar))
	da = dy.astype(np.float64).reshape(x64.shape) * slope(t, name)
	if name == "relu":       # where t is nearer to zero than its own rounding the gate may fall either way: those elements say nothing
		assert (np.abs(t) <= dt).sum() <= 2 + 1e-4 * t.size
	unsure = np.abs(dy.astype(np.float64).reshape(x64.shape)) * (np.abs(t) <= dt) if name == "relu" else 0.0
	rough = np.abs(dy.astype(np.float64).reshape(x64.shape)) * (dt + (24 * U32 if dtype == np.float32 else 2.0 ** -13)) * (0.0 if name == "none" else 1.0) + unsure + U32 * np.abs(da)
	dbias, dscale = da.sum(axis=(0, 1)), (da * xhat).sum(axis=(0, 1))
	a, b = (da * g).sum(axis=(1, 3), keepdims=True) / m, (da * g * xhat).sum(axis=(1, 3), keepdims=True) / m
	dx = wide(invvar) * (da * g - a - xhat * b)

	steps = 8 + 2 * np.sqrt(m)
	prod = lambda v, w: (v * np.abs(w))
	da_x = rough * np.abs(xhat) + np.abs(da) * (2 * U32 * np.abs(xhat) + 2 * U32 * wide(np.abs(mean) * invvar))
	ab = (rough * g).mean(axis=(1, 3), keepdims=True) + steps * U32 * np.abs(da * g).mean(axis=(1, 3), keepdims=True)
	bb = (da_x * g).mean(axis=(1, 3), keepdims=True) + steps * U32 * np.abs(da * g * xhat).mean(axis=(1, 3), keepdims=True)
	dxb = wide(invvar) * (rough * g + ab + np.abs(xhat) * bb + np.abs(b) * 4 * U32 * (np.abs(xhat) + wide(np.abs(mean) * invvar)) + 4 * U32 * (np.abs(da * g) + np.abs(a) + np.abs(xhat * b)))
	count = n * x64.shape[1]
	many = 8 + 2 * np.sqrt(count)

	args = [gpu(bnd, v) for v in (dy, x, scale, bias, mean, invvar)]
	out, ds, db = bnd.dnn.groupNormNdBackward(*args, groups, act=bnd.FusedAct[name])
	within(out.get(), dx.reshape(shape), dxb.reshape(shape), "dx")
	within(ds.get(), dscale.reshape(-1), da_x.sum(axis=(0, 1)).reshape(-1) + many * U32 * np.abs(da * xhat).sum(axis=(0, 1)).reshape(-1), "dscale")
	within(db.get(), dbias.reshape(-1), rough.sum(axis=(0, 1)).reshape(-1) + many * U32 * np.abs(da).sum(axis=(0, 1)).reshape(-1), "dbias")
	alone = bnd.dnn.groupNormNdBackward(*args, groups, act=bnd.FusedAct[name], affine=False, out=args[0])                    # over the gradient
	assert alone is args[0] and np.array_equal(alone.get(), out.get())


def test_groupnorm_gradients_against_differences(bnd):
	rng = np.random.RandomState(0)
	shape, groups = (2, 6, 12), 3
	x, dy = rng.randn(*shape).astype(np.float32), rng.randn(*shape).astype(np.float32)
	scale, bias = (1 + 0.1 * rng.randn(12)).astype(np.float32), (0.1 * rng.randn(12)).astype(np.float32)

	def f(x, s, b):
		return float((bnd.dnn.groupNormNd(gpu(bnd, x), gpu(bnd, s), gpu(bnd, b), groups, act=bnd.FusedAct.silu, test=True).get().astype(np.float64) * dy).sum())

	_, mean, invvar = bnd.dnn.groupNormNd(gpu(bnd, x), gpu(bnd, scale), gpu(bnd, bias), groups, act=bnd.FusedAct.silu)
	grads = bnd.dnn.groupNormNdBackward(gpu(bnd, dy), gpu(bnd, x), gpu(bnd, scale), gpu(bnd, bias), mean, invvar, groups, act=bnd.FusedAct.silu)
	at = [x, scale, bias]
	for i in range(3):
		d = rng.randn(*at[i].shape).astype(np.float32)
		d /= np.linalg.norm(d)
		plus, minus = list(at), list(at)
		plus[i], minus[i] = at[i] + np.float32(2.0 ** -6) * d, at[i] - np.float32(2.0 ** -6) * d
		step = float(((plus[i].astype(np.float64) - minus[i]) * d).sum())
		exact = float((grads[i].get().astype(np.float64) * d).sum())
		assert abs((f(*plus) - f(*minus)) / step - exact) <= 2e-3 * (1.0 + abs(exact)), i


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_groupnorm_special_rows(bnd, dtype):
	"""constant groups, no affine pair, far means, one NaN, nothing at all"""
	F = bnd.FusedAct
	flat = np.full((2, 9, 16), 3.0, dtype)
	out, mean, inv = bnd.dnn.groupNormNd(gpu(bnd, flat), None, None, 4)
	assert np.all(out.get() == 0) and np.all(mean.get() == 3)
	assert np.allclose(inv.get(), 1e5 ** 0.5, rtol=1e-6)
	x = (np.random.RandomState(0).randn(1, 4000, 16) * 0.5 + 200.0).astype(dtype)              # far from zero: no squares are subtracted
	_, mean, inv = bnd.dnn.groupNormNd(gpu(bnd, x), None, None, 2)
	m64, i64, _, _ = normOracle(x, None, None, 2, 1e-5, "none")
	assert np.allclose(mean.get(), m64, rtol=1e-6) and np.allclose(inv.get(), i64, rtol=2e-5)
	x[0, 7, 3] = np.nan
	y = bnd.dnn.groupNormNd(gpu(bnd, x), None, None, 2, act=F.relu, test=True).get()
	assert np.isnan(y[..., :8]).all() and np.isfinite(y[..., 8:]).all()
	for shape in ((0, 4, 16), (2, 0, 16)):
		out, mean, inv = bnd.dnn.groupNormNd(gpu(bnd, np.zeros(shape, dtype)), None, None, 4)
		assert out.shape == shape and mean.shape == (shape[0], 4)
		dx, ds, db = bnd.dnn.groupNormNdBackward(out, out, None, None, mean, inv, 4)
		assert dx.shape == shape and np.all(ds.get() == 0) and np.all(db.get() == 0)


# ------------------------------------------------------------------------------------------------ together
@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_feed_forward_block(bnd, dtype):
	"""x + dropout(W2 gelu(W1 silu(norm x) + b1) + b2) over channels-last pixels, forward and backward, as one would chain it"""
	rng = np.random.RandomState(12)
	n, s, c, hidden, groups = 3, 50, 64, 160, 8
	F = bnd.FusedAct
	x = rng.randn(n, s, c).astype(dtype)
	scale, bias = (1 + 0.1 * rng.randn(c)).astype(np.float32), (0.1 * rng.randn(c)).astype(np.float32)
	W1, W2 = (rng.randn(c, hidden) / 8).astype(dtype), (rng.randn(hidden, c) / 12).astype(dtype)
	b1, b2 = (0.1 * rng.randn(hidden)).astype(np.float32), (0.1 * rng.randn(c)).astype(np.float32)
	dy = rng.randn(n, s, c).astype(dtype)
	mask = bnd.globalRng.dropoutMask(0.2)

	gx, gs, gb, g1, h1, g2, h2, gdy = [gpu(bnd, v) for v in (x, scale, bias, W1, b1, W2, b2, dy)]
	u, mean, inv = bnd.dnn.groupNormNd(gx, gs, gb, groups, act=F.silu)
	h, z1 = bnd.blas.linear(u, g1, h1, act=F.gelu, preact=True)
	y = bnd.blas.linear(h, g2, h2, dropout=mask, residual=gx)
	dh, dW2, db2 = bnd.blas.linearBackward(gdy, h, g2, dropout=mask)
	du, dW1, db1 = bnd.blas.linearBackward(dh, u, g1, act=F.gelu, preact=z1)
	dx, ds, db = bnd.dnn.groupNormNdBackward(du, gx, gs, gb, mean, inv, groups, act=F.silu)
	bnd.counterDropoutKer(dtype)                                      # (the same mask on its own)

	# 64 bits
	m64, i64, xhat, t = normOracle(x, scale, bias, groups, 1e-5, "silu")
	U64 = act(t, "silu").reshape(n * s, c)
	Z = U64 @ W1.astype(np.float64) + b1
	H = act(Z, "gelu")
	kp = keep(mask, (n, s, c)).reshape(n * s, c)
	Y = x.reshape(n * s, c) + (H @ W2.astype(np.float64) + b2) * kp
	DZ2 = dy.reshape(n * s, c).astype(np.float64) * kp
	DH = DZ2 @ W2.T.astype(np.float64)
	DZ1 = DH * slope(Z, "gelu")
	DU = (DZ1 @ W1.T.astype(np.float64)).reshape(t.shape) * slope(t, "silu")
	g64 = scale.astype(np.float64).reshape(groups, -1)
	mm = t.shape[1] * t.shape[3]
	a, b = (DU * g64).sum(axis=(1, 3), keepdims=True) / mm, (DU * g64 * xhat).sum(axis=(1, 3), keepdims=True) / mm
	DX = (i64[:, None, :, None] * (DU * g64 - a - xhat * b)).reshape(n, s, c)

	# relative to each tensor's size: the chain rounds five intermediate tensors (float16: 2^-11 each, float32: sums of 160 terms)
	tol = 5 * 2.0 ** -11 if dtype == np.float16 else 64 * U32
	for got, want, what in ((y, Y.reshape(n, s, c), "y"), (dW2, H.T @ DZ2, "dW2"), (db2, DZ2.sum(0), "db2"), (dW1, U64.T @ DZ1, "dW1"),
							(db1, DZ1.sum(0), "db1"), (dx, DX, "dx"), (ds, (DU * xhat).sum(axis=(0, 1)).reshape(-1), "dscale"),
							(db, DU.sum(axis=(0, 1)).reshape(-1), "dbias")):
		err = np.linalg.norm(got.get().astype(np.float64) - want) / np.linalg.norm(want)
		assert err <= tol, "%s: relative error %.3g" % (what, err)


# ------------------------------------------------------------------------------------------------ places beyond 32 bits
def put(buf, pitch, col, rows):
	"""rows -> columns col ... of a flat buffer whose rows stand `pitch` apart, one by one (strided copies take 4-byte types only)"""
	for i, row in enumerate(rows):
		buf[i * pitch + col:i * pitch + col + row.size].set(row)


def take(buf, pitch, col, m, n):
	return np.stack([buf[i * pitch + col:i * pitch + col + n].get() for i in range(m)])


@pytest.mark.parametrize("dtype", [np.float32, np.float16])
def test_linear_rows_beyond_32_bits(bnd, dtype):
	"""x, W, residual, out and pre-activation as columns of one buffer of more than 2^32 bytes (float16: more than 2^31 elements)"""
	m, k, n = 290, 290, 72
	pitch = (16 << 20) // np.dtype(dtype).itemsize
	rng = np.random.RandomState(21)
	x, W, r = rng.randn(m, k).astype(dtype), (rng.randn(k, n) / 16).astype(dtype), rng.randn(m, n).astype(dtype)
	buf = bnd.GPUArray.empty((m * pitch, ), dtype=dtype)
	grid = buf.reshape(m, pitch)
	cols = dict(x=0, W=1024, r=2048, out=4096, z=pitch - n)
	for name, ary in (("x", x), ("W", W), ("r", r)):
		put(buf, pitch, cols[name], ary)
	view = lambda name, width: grid[:, cols[name]:cols[name] + width]
	bnd.blas.linear(view("x", k), view("W", n), act=bnd.FusedAct.relu, residual=view("r", n), preact=view("z", n), out=view("out", n))
	x64, W64, r64 = (a.astype(np.float64) for a in (x, W, r))
	z = x64 @ W64
	bound = productBound(x64, W64, k)
	within(take(buf, pitch, cols["z"], m, n), z, bound, "preact")
	y = act(z, "relu") + r64
	within(take(buf, pitch, cols["out"], m, n), y, bound + U32 * np.abs(y), "out")
	for name, ary in (("x", x), ("W", W), ("r", r)):
		assert np.array_equal(take(buf, pitch, cols[name], *ary.shape), ary), name


def test_counter_dropout_beyond_32_bits(bnd):
	count = (1 << 32) + 1003
	mask = bnd.DropoutMask(77, 5, 0.25)
	rng = np.random.RandomState(22)
	buf = bnd.GPUArray.empty((count, ), dtype=np.float16)
	spots = [0, (1 << 30) - 500, (1 << 31) - 500, (1 << 32) - 500, count - 500]
	x = [rng.randn(500).astype(np.float16) for _ in spots]
	for at, v in zip(spots, x):
		buf[at:at + 500].set(v)
	bnd.counterDropoutKer(np.float16)(buf, buf, mask)
	for at, v in zip(spots, x):
		first = at // 4 * 4
		q = wordsFrom(mask.seed, mask.call, first // 4, 128)[at - first:at - first + 500]
		want = np.where(q < mask.key.threshold, v.astype(np.float64) / 0.75, 0.0)
		got = buf[at:at + 500].get()
		within(got, want, 3 * U32 * np.abs(want), "at %d" % at)
		assert np.array_equal(got == 0, want == 0), "the mask at %d" % at


def test_groupnorm_beyond_32_bits(bnd):
	"""3 x 3000001 x 256 float16 (2.3e9 elements) whose channels alternate between 2 and 1: mean 1.5, variance 1/4 in every group"""
	shape, groups, epsilon = (3, 3000001, 256), 2, 1e-5
	x = bnd.GPUArray.empty(shape, dtype=np.float16)
	x.gpudata.fillD32(0x3c004000)                                   # 2.0 in the low half
	scale, bias = gpu(bnd, np.full(256, 1.0, np.float32)), gpu(bnd, np.full(256, 0.25, np.float32))
	y, mean, inv = bnd.dnn.groupNormNd(x, scale, bias, groups, epsilon=epsilon)
	iv = 1.0 / np.sqrt(0.25 + epsilon)
	# a chunk's sums pass fewer than 64 additions one after the other, the chunks are joined in 64 bits
	within(mean.get(), np.full((3, groups), 1.5), 64 * U32 * 1.5, "mean")
	within(inv.get(), np.full((3, groups), iv), 64 * U32 * iv, "invvar")
	xhat = np.tile([0.5 * iv, -0.5 * iv], 128)
	spots = [0, (1 << 30) // 256 - 2, (1 << 31) // 256 - 2, 3 * 3000001 - 4]
	rows = lambda a: [a.reshape(-1, 256)[at:at + 4].get() for at in spots]
	for got in rows(y):
		within(got, np.tile(xhat + 0.25, (4, 1)), 200 * U32, "y")
	g = y
	g.gpudata.fillD32(0x38003c00)                                   # 1.0 in the low half, 0.5 in the high one
	dx, dscale, dbias = bnd.dnn.groupNormNdBackward(g, x, scale, bias, mean, inv, groups)
	d = np.tile([1.0, 0.5], 128)
	count = 3.0 * 3000001
	within(dbias.get(), count * d, 64 * U32 * count * d, "dbias")
	within(dscale.get(), count * d * xhat, 200 * U32 * count * d, "dscale")
	want = iv * (d - 0.75 - xhat * (d * xhat).mean())                # (nearly nothing: the terms cancel)
	for got in rows(dx):
		within(got, np.tile(want, (4, 1)), iv * 200 * U32 * 2.0, "dx")


def test_dropout_on_a_stream_then_a_product(bnd):
	"""a mask applied on a borrowed stream, a float16 product that reads it, the stream again: each waits for the other"""
	rng = np.random.RandomState(23)
	x, W = rng.randn(512, 256).astype(np.float16), (rng.randn(256, 512) / 16).astype(np.float16)
	gx, gW = gpu(bnd, x), gpu(bnd, W)
	ker = bnd.counterDropoutKer(np.float16)
	stream = bnd.Driver.Stream()
	for call in range(3):
		one, two = bnd.DropoutMask(9, 2 * call, 0.5), bnd.DropoutMask(9, 2 * call + 1, 0.5)
		h, out = bnd.GPUArray.empty(x.shape, dtype=np.float16), bnd.GPUArray.empty((512, 512), dtype=np.float16)
		ker(h, gx, one, stream=stream)
		y = bnd.blas.linear(h, gW)
		ker(out, y, two, stream=stream)
		dropped = x.astype(np.float64) * keep(one, x.shape)
		within(h.get(), dropped, 3 * U32 * np.abs(dropped), "h")
		within(y.get(), dropped @ W, productBound(dropped, W.astype(np.float64), 256), "y")
		assert np.array_equal(out.get(), (y.get() * keep(two, (512, 512))).astype(np.float16))
