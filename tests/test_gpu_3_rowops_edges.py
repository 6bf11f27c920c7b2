"""
The operators over rows of channels on the device, beyond tests/test_gpu_3_rowops.py (whose plain forms in 64 bits and bounds it uses):
values at the ends of the types' ranges, row pitches whose multiples pass 32 bits, the tiles and slabs of large problems, streams.
"""
import numpy as np
import pytest

from test_gpu_3_rowops import (
	ACTS, LIPSCHITZ, TINY, U, U32, Case, act, gpu, keep, normBounds, normOracle, productBound, put, slope, take, within
)

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
