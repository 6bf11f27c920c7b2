"""
Refusals and call sequences of blas.linear / linearBackward, counterDropoutKer and dnn.groupNormNd / groupNormNdBackward without a
device: run by tests/test_rowops_host.py in a child process in dry-run mode (C-ABI calls recorded, not executed; workspace sizes and
argument checks come from the real library). Usage: python tests/dryrun/rowops_checks.py <check name>
"""
import ctypes, os, sys

assert os.environ.get("PUZZLE_MI355_DRYRUN") == "1"
ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

import numpy as np

from puzzlelib_amd import backend, lib, lazy

bnd = backend.getBackend(0, initmode=2)
F = bnd.FusedAct
A = lambda *shape, dtype=np.float32: bnd.GPUArray.empty(shape, dtype=dtype)


def refused(call, *words, kind=ValueError):
	try:
		call()
	except kind as e:
		for word in words:
			assert word in str(e), "%r lacks %r" % (str(e), word)
		return
	raise AssertionError("accepted")


def linear_refusals():
	blas = bnd.blas
	x, W, b = A(6, 8), A(8, 10), A(10)
	refused(lambda: blas.linear(A(6, 8, dtype=np.int32), W), "float32 or float16")
	refused(lambda: blas.linear(x, A(8, 10, dtype=np.float16)), "W is")
	refused(lambda: blas.linear(x, A(9, 10)), "does not fit")
	refused(lambda: blas.linear(x, W, transpW=True), "does not fit")
	refused(lambda: blas.linear(A(8), W), "two axes")
	refused(lambda: blas.linear(x, A(2, 8, 10)), "matrix")
	refused(lambda: blas.linear(x, A(8, 0)), "does not fit")
	refused(lambda: blas.linear(x, W, A(9)), "bias")
	refused(lambda: blas.linear(x, W, A(10, dtype=np.float16)), "bias")
	refused(lambda: blas.linear(x, W, b, residual=A(6, 9)), "residual")
	refused(lambda: blas.linear(x, W, b, residual=A(6, 10, dtype=np.float16)), "residual")
	refused(lambda: blas.linear(x, W, b, out=A(5, 10)), "out")
	refused(lambda: blas.linear(x, W, b, preact=A(6, 11)), "preact")
	refused(lambda: blas.linear(x, W, b, dropout=0.5), "DropoutMask")
	refused(lambda: blas.linear(x, W, b, act="swish"), "swish")
	refused(lambda: blas.linear(A(12, 8)[::2].reshape(6, 8)[:, ::2], A(4, 10)), "last axis")
	cube = A(4, 6, 8)
	refused(lambda: blas.linear(cube[:, :5], W), "one pitch")
	# outputs over operands
	square = A(8, 8)
	refused(lambda: blas.linear(square, W[:, :8], out=square), "overlaps")
	refused(lambda: blas.linear(x, W, out=W[:6]), "overlaps")
	both = A(6, 20)
	refused(lambda: blas.linear(x, W, residual=both[:, :10], out=both[:, 5:15]), "overlaps")
	refused(lambda: blas.linear(x, W, residual=both[:, :10], out=both[:, 10:], preact=both[:, 8:18]), "overlaps")
	blas.linear(x, W, residual=both[:, :10], out=both[:, 10:])
	blas.linear(x, W, residual=both[:, :10], out=both[:, :10])
	# the way back
	g = A(6, 10)
	refused(lambda: blas.linearBackward(A(6, 9), x, W), "grad")
	refused(lambda: blas.linearBackward(g, x, W, act=F.gelu), "pre-activation")
	refused(lambda: blas.linearBackward(g, x, W, act=F.gelu, preact=A(6, 8)), "preact")
	refused(lambda: blas.linearBackward(g, x, W, wgrad=A(10, 8)), "wgrad")
	refused(lambda: blas.linearBackward(A(6, 10), x, W, wgrad=A(8, 10, dtype=np.float16)), "wgrad")
	refused(lambda: blas.linearBackward(g, x, W, bgrad=A(8)), "bgrad")
	refused(lambda: blas.linearBackward(g, x, W, wgrad=A(8, 10), momentum=1.0), "momentum")
	refused(lambda: blas.linearBackward(g, x, W, out=x), "overlaps")
	refused(lambda: blas.linearBackward(g, x, W, wgrad=W), "overlaps")
	for p in (-0.1, 1.0, 1.5, float("nan")):
		refused(lambda: bnd.DropoutMask(0, 0, p), "probability")
	refused(lambda: bnd.DropoutMask(-1, 0, 0.5), "64-bit")
	refused(lambda: bnd.DropoutMask(0, 1 << 64, 0.5), "64-bit")


def linear_c_entry_refusals():
	"""the library's own argument checks, reached without a device: nothing is launched"""
	real = lambda name: getattr(lib._lib, name)
	D = lambda **kw: lib.LinearDesc(*[{**dict(dtype=0, act=0, trans_w=0, m=4, n=8, k=8, ldx=8, ldw=8, ldy=8, ldr=8, ldp=8), **kw}[f] for f, _ in lib.LinearDesc._fields_])
	mask = lib.DropoutKey(1, 2, 3, 0.5)
	p = ctypes.c_void_p(4096)

	def fwd(desc, x=p, w=p, y=p, key=None, ws=None, nbytes=0):
		fn = real("pz_linear_fwd")
		fn.argtypes = lib._PROTOS["pz_linear_fwd"]
		return fn(ctypes.byref(desc), x, w, None, None, None if key is None else ctypes.byref(key), y, None, ws, nbytes, None)

	for bad in (D(dtype=2), D(act=4), D(act=-1), D(m=-1), D(n=0), D(k=0), D(ldx=7), D(ldw=7), D(ldy=7)):
		assert fwd(bad) == lib.PZ_ERR_INVALID, lib.lastError()
	assert fwd(D(), x=None) == fwd(D(), w=None) == fwd(D(), y=None) == lib.PZ_ERR_INVALID
	for keep in (0.0, -1.0, 1.5, float("nan")):
		assert fwd(D(), key=lib.DropoutKey(1, 2, 3, keep)) == lib.PZ_ERR_INVALID
	assert fwd(D(ldx=9, dtype=1)) == lib.PZ_ERR_INVALID and "workspace" in lib.lastError()          # a copy of x, no workspace for it
	assert fwd(D(m=0)) == lib.PZ_OK
	assert fwd(D(m=256, ldx=1 << 25)) == lib.PZ_ERR_INVALID and "too far apart" in lib.lastError()   # a tile's rows beyond 32-bit offsets
	assert fwd(D(ldw=1 << 28)) == lib.PZ_ERR_INVALID and "too far apart" in lib.lastError()
	for bad in (D(m=0x7fffffff), D(k=1 << 28, ldx=1 << 28), D(n=1 << 28, ldw=1 << 28, ldy=1 << 28)):
		assert fwd(bad) == lib.PZ_ERR_INVALID and "too large" in lib.lastError()

	bwd = real("pz_linear_bwd")
	bwd.argtypes = lib._PROTOS["pz_linear_bwd"]
	call = lambda d, dy=p, x=p, w=p, z=None, dx=p, dw=p, t=0, ws=None, n=0: bwd(ctypes.byref(d), dy, x, w, z, None, dx, dw, t, None, 1.0, 0.0, ws, n, None)
	assert call(D(act=2)) == lib.PZ_ERR_INVALID and "pre-activation" in lib.lastError()
	assert call(D(), t=1) == lib.PZ_ERR_INVALID and call(D(), dy=None) == lib.PZ_ERR_INVALID and call(D(ldr=7)) == lib.PZ_ERR_INVALID
	assert call(D(m=256, ldr=8, ldx=1 << 28)) == lib.PZ_ERR_INVALID and "too far apart" in lib.lastError()
	assert call(D(), x=None) == lib.PZ_ERR_INVALID and call(D(), w=None) == lib.PZ_ERR_INVALID
	assert call(D(act=1), z=p) == lib.PZ_ERR_INVALID and "workspace" in lib.lastError()

	drop = real("pz_dropout")
	drop.argtypes = lib._PROTOS["pz_dropout"]
	assert drop(2, p, None, p, 4, ctypes.byref(mask), None) == lib.PZ_ERR_INVALID
	assert drop(0, p, None, p, 4, None, None) == lib.PZ_ERR_INVALID
	assert drop(0, None, None, p, 4, ctypes.byref(mask), None) == lib.PZ_ERR_INVALID
	assert drop(0, p, None, p, 1 << 36, ctypes.byref(mask), None) == lib.PZ_ERR_INVALID and "too many" in lib.lastError()
	assert drop(0, None, None, None, 0, ctypes.byref(mask), None) == lib.PZ_OK

	G = lambda **kw: lib.GroupNormDesc(*[{**dict(dtype=0, act=0, n=2, pixels=3, c=8, groups=2, epsilon=1e-5), **kw}[f] for f, _ in lib.GroupNormDesc._fields_])
	size = ctypes.c_size_t(0)
	for bad in (G(dtype=3), G(act=9), G(n=-1), G(pixels=-1), G(c=0), G(groups=0), G(groups=3), G(epsilon=-1.0),
				G(n=1 << 30, c=64), G(c=1 << 26)):
		refused(lambda: lib.pz_groupnorm_workspace_bytes(ctypes.byref(bad), 0, ctypes.byref(size)))
	gf = real("pz_groupnorm_fwd")
	gf.argtypes = lib._PROTOS["pz_groupnorm_fwd"]
	assert gf(ctypes.byref(G()), None, None, None, p, None, None, None, 0, None) == lib.PZ_ERR_INVALID
	gb = real("pz_groupnorm_bwd")
	gb.argtypes = lib._PROTOS["pz_groupnorm_bwd"]
	assert gb(ctypes.byref(G()), p, p, None, None, p, p, p, p, p, None, 0, None) == lib.PZ_ERR_INVALID and "workspace" in lib.lastError()
	assert gb(ctypes.byref(G()), p, p, None, None, None, p, p, p, p, p, 1 << 20, None) == lib.PZ_ERR_INVALID


def workspace_sizes():
	"""every size the operators may be asked for has an answer: empty batches, single rows, the longest ones"""
	size = ctypes.c_size_t(0)
	for dtype in (lib.F32, lib.F16):
		for m in (0, 1, 2, 63, 64, 65, 1000, 8192, 1 << 20, (1 << 31) - 1 - (1 << 17)):
			for k, n in ((1, 1), (7, 5), (64, 64), (1000, 2048), (8192, 8192)):
				desc = lib.LinearDesc(dtype, 0, 0, m, n, k, k, n, n, n, n)
				lib.pz_linear_fwd_workspace_bytes(ctypes.byref(desc), 4096, 4096, ctypes.byref(size))
				desc.ldr = k
				for dropping in (0, 1):
					lib.pz_linear_bwd_workspace_bytes(ctypes.byref(desc), 4096, 4096, 4096, dropping, 1, 1, 1, ctypes.byref(size))
		for n in (0, 1, 3, 65535):
			for pixels in (0, 1, 7, 4096, 1 << 24):
				for c, groups in ((1, 1), (30, 3), (512, 32), (1030, 103), (16384, 1)):
					desc = lib.GroupNormDesc(dtype, 0, n, pixels, c, groups, 1e-5)
					for backward in (0, 1):
						lib.pz_groupnorm_workspace_bytes(ctypes.byref(desc), backward, ctypes.byref(size))


def dropout_refusals():
	ker = bnd.counterDropoutKer(np.float32)
	mask = bnd.DropoutMask(1, 2, 0.5)
	x, y = A(10), A(10)
	refused(lambda: bnd.counterDropoutKer(np.int32), kind=NotImplementedError)
	refused(lambda: ker(y, A(11), mask), "does not match")
	refused(lambda: ker(y, A(10, dtype=np.float16), mask), "does not match")
	refused(lambda: ker(y, x, mask, residual=A(9)), "does not match")
	refused(lambda: ker(y, x, 0.5), "DropoutMask")
	refused(lambda: ker(y, x, mask, slice=slice(0, 5)), "whole")
	refused(lambda: ker(y, A(20)[::2], mask), "contiguous")
	big = A(20)
	refused(lambda: ker(big[5:15], big[:10], mask), "overlaps")
	ker(big[:10], big[:10], mask)
	ker(big[10:], big[:10], mask)
	rng = bnd.RandomNumberGenerator(seed=5)
	one, two = rng.dropoutMask(0.5), rng.dropoutMask(0.5)
	assert (one.seed, one.call) != (two.seed, two.call)


def groupnorm_refusals():
	dnn = bnd.dnn
	x, s, b = A(2, 5, 12), A(12), A(12)
	refused(lambda: dnn.groupNormNd(A(2, 5, 12, dtype=np.int32), s, b, 3), "float32 or float16")
	refused(lambda: dnn.groupNormNd(x, s, b, 5), "groups")
	refused(lambda: dnn.groupNormNd(x, s, b, 0), "groups")
	refused(lambda: dnn.groupNormNd(x, s, b, 2.4), "groups")
	for epsilon in (-1e-5, float("nan")):
		refused(lambda: dnn.groupNormNd(x, s, b, 3, epsilon=epsilon), "epsilon")
	refused(lambda: dnn.groupNormNd(x, A(11), b, 3), "scale")
	refused(lambda: dnn.groupNormNd(x, s, A(12, dtype=np.float16), 3), "bias")
	refused(lambda: dnn.groupNormNd(x[:, :, :6], A(6), A(6), 3), "contiguous")
	refused(lambda: dnn.groupNormNd(A(12), s, b, 3), "batch")
	refused(lambda: dnn.groupNormNd(x, s, b, 3, out=A(2, 5, 11)), "out")
	refused(lambda: dnn.groupNormNd(x, s, b, 3, savemean=A(2, 4)), "savemean")
	refused(lambda: dnn.groupNormNd(x, s, b, 3, saveinvvar=A(2, 3, dtype=np.float16)), "saveinvvar")
	stat = A(2, 3)
	refused(lambda: dnn.groupNormNd(x, s, b, 3, savemean=stat, saveinvvar=stat), "overlaps")
	big = A(4, 5, 12)
	refused(lambda: dnn.groupNormNd(big[:2], s, b, 3, out=big[1:3]), "overlaps")
	out, mean, inv = dnn.groupNormNd(x, s, b, 3)
	assert mean.shape == inv.shape == (2, 3)
	dnn.groupNormNd(x, s, b, 3, out=x)
	refused(lambda: dnn.groupNormNdBackward(A(2, 5, 11), x, s, b, mean, inv, 3), "grad")
	refused(lambda: dnn.groupNormNdBackward(out, x, s, b, A(2, 4), inv, 3), "savemean")
	refused(lambda: dnn.groupNormNdBackward(out, x, s, b, mean, inv, 3, scalegrad=A(11)), "scalegrad")
	refused(lambda: dnn.groupNormNdBackward(out, x, s, b, mean, inv, 3, scalegrad=s), "overlaps")
	one = A(12)
	refused(lambda: dnn.groupNormNdBackward(out, x, s, b, mean, inv, 3, scalegrad=one, bgrad=one), "overlaps")


def matrix_kernels_keep_apart():
	"""a float16 product follows every foreign launch, and the next foreign launch follows it even when it brings an older mark"""
	def running(name, args):                                              # no event has passed yet
		if name == "pz_event_query":
			lib._store(args[1], 0)
		return name == "pz_event_query"

	lib.callHook = running
	stream = bnd.Driver.Stream()
	x, y = A(4096), A(4096)
	mark = lazy.newEvent()
	mark.record(None)
	bnd.counterDropoutKer(np.float32)(y, x, bnd.DropoutMask(1, 2, 0.5), stream=stream)
	lib.trace.clear()
	bnd.blas.linear(A(8, 16, dtype=np.float16), A(16, 8, dtype=np.float16))
	names = [n for n, _ in lib.trace]
	assert names.index("pz_stream_wait_event") < names.index("pz_linear_fwd"), names
	ready = lazy.foreignBegin(stream, mark)
	assert ready is not mark
	assert lazy.foreignBegin(stream, mark) is mark
	# ... on whichever stream: the older mark alone would let it run beside the product
	other = bnd.Driver.Stream()
	lib.trace.clear()
	assert lazy.foreignBegin(other, mark) is mark
	assert [n for n, _ in lib.trace].count("pz_stream_wait_event") == 2, lib.trace           # the product's event, then the mark
	lib.trace.clear()
	bnd.blas.linear(A(8, 16), A(16, 8))                                    # float32: no such order
	assert "pz_stream_wait_event" not in [n for n, _ in lib.trace]


if __name__ == "__main__":
	globals()[sys.argv[1]]()
	print("OK")
