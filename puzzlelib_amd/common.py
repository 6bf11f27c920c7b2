"""
Enumerations and small argument helpers shared by the context objects of the backend (puzzlelib_amd/blas.py, dnn.py,
modules.py, kernels.py, backend.py): the ids the reference's wrappers expose (Hip/Wrappers/MIOpen.py:23-88,
Cuda/Wrappers/CuBlas.py) and the checks every entry point makes on its operands.
"""
from enum import Enum

import numpy as np

from puzzlelib_amd import lib


class ConvFwdAlgo(Enum):              # Hip/Wrappers/MIOpen.py:24-31 (values are this library's algo ids)
	auto = -1
	gemm = 0
	direct = 1
	fft = 2
	winograd = 3
	implicitGemm = 5
	staticGemm = 4


class ConvBwdFilterAlgo(Enum):        # Hip/Wrappers/MIOpen.py:34-39
	auto = -1
	gemm = 0
	direct = 1
	winograd = 3
	implicitGemm = 5


class ConvBwdDataAlgo(Enum):          # Hip/Wrappers/MIOpen.py:42-49
	auto = -1
	gemm = 0
	direct = 1
	fft = 2
	winograd = 3
	transposeGemm = 4
	implicitGemm = 5


class PoolMode(Enum):                 # Hip/Wrappers/MIOpen.py:52-55
	max = 0
	avgWithPad = 1
	avgNoPad = 2


class SoftMaxMode(Enum):              # Hip/Wrappers/MIOpen.py:64-66
	perActivation = 0
	spatial = 1


class BatchNormMode(Enum):            # Hip/Wrappers/MIOpen.py:69-71
	perActivation = 0
	spatial = 1


class LRNMode(Enum):
	map = 0
	cross = 1


class RNNMode(Enum):
	relu = 0
	tanh = 1
	lstm = 2
	gru = 3


class DirectionMode(Enum):
	uni = 0
	bi = 1


class RNNAlgo(Enum):
	default = 0


class GroupFormat(Enum):              # Hip/Backend.py:39-41
	gbp = 0
	bgp = 1


class FusedAct(Enum):                  # the activation inside blas.linear / dnn.groupNormNd (enum PZ_ACT_*)
	none = 0
	relu = 1
	gelu = 2
	silu = 3


class DropoutMask:
	"""A dropout mask by its key. Element i of a tensor (row-major) is kept where word i of call `call` of the generator `seed` is
	below (1 - p) * (2^32 - 1), and kept elements are divided by 1 - p: the mask fillInteger + dropoutKer
	(Modules/Dropout.py:33-72) would apply, computed where it is needed instead of stored; at p = 0 every element is kept, also one
	whose word is 2^32 - 1. The same object gives the same mask forward and backward. RandomNumberGenerator.dropoutMask(p) hands out a mask nobody else gets."""
	__slots__ = ("seed", "call", "p", "key", "drops")

	def __init__(self, seed, call, p):
		if not 0.0 <= p < 1.0:
			raise ValueError("dropout probability %r is outside [0, 1)" % (p, ))
		self.seed, self.call, self.p = int(seed), int(call), float(p)
		if not (0 <= self.seed < 1 << 64 and 0 <= self.call < 1 << 64):
			raise ValueError("a dropout mask's seed and call are unsigned 64-bit numbers")
		keep = 1.0 - self.p
		self.key = lib.DropoutKey(self.seed, self.call, int(keep * np.iinfo(np.uint32).max), keep)
		self.drops = self.key.threshold != np.iinfo(np.uint32).max


class ConvPerf:                        # Hip/Wrappers/MIOpen.py:82-100
	def __init__(self, algo, time, memory):
		self.algo, self.time, self.memory = algo, time, memory

	def toString(self):
		return "%-40s %-25s %-28s" % (
			"Algo %s" % self.algo, "time %.6f secs" % self.time, "memory %.6f mbytes" % (self.memory / 1024**2)
		)

	__str__ = __repr__ = toString


def toAlgoId(algo):
	"""The reference's algo ids: `direct` is the one-thread-per-output kernel, `winograd` asks for F(2x2, 3x3) where it
	applies (3x3 stride-1 forward / backward-data), `implicitGemm` pins the MFMA implicit GEMM, every other id leaves the
	choice to the library."""
	algo = algo.value if isinstance(algo, Enum) else algo
	return {1: lib.CONV_ALGO_DIRECT, 3: lib.CONV_ALGO_WINOGRAD, 5: lib.CONV_ALGO_IMPLICIT_GEMM}.get(algo, lib.CONV_ALGO_AUTO)


def pair(v):
	return (int(v), int(v)) if isinstance(v, (int, np.integer)) else tuple(int(a) for a in v)


def requireF32(*arrays):
	for ary in arrays:
		if ary is None:
			continue
		if ary.dtype != np.float32:
			raise ValueError("float32 gpuarray expected, got %s" % ary.dtype)
		if not ary.contiguous:
			raise ValueError("gpuarray is not contiguous")


def rptrOf(ary):
	return None if ary is None else ary.rptr


# ---- operators over rows of channels (blas.linear, dnn.groupNormNd, counterDropoutKer): float32 and float16 tensors
ROW_DTYPES = {np.dtype(np.float32): lib.F32, np.dtype(np.float16): lib.F16}


def rowDtype(ary, what):
	dtype = ROW_DTYPES.get(ary.dtype, None)
	if dtype is None:
		raise ValueError("%s: float32 or float16 gpuarray expected, got %s" % (what, ary.dtype))
	return dtype


def rowPitch(ary, what):
	"""Elements from one row (the last axis) to the next: rows are dense, and all leading axes step by one pitch"""
	item = ary.dtype.itemsize
	if ary.contiguous:
		return ary.shape[-1]
	strides, shape = ary.strides, ary.shape
	pitch, expect = None, None
	if shape[-1] > 1 and strides[-1] != item:
		raise ValueError("%s: the last axis is not contiguous" % what)
	for axis in range(ary.ndim - 2, -1, -1):
		if shape[axis] == 1:
			continue
		if pitch is None:
			pitch = strides[axis]
		elif strides[axis] != expect:
			raise ValueError("%s: rows of one pitch expected, got strides %s of shape %s" % (what, strides, shape))
		expect = strides[axis] * shape[axis]
	pitch = shape[-1] * item if pitch is None else pitch
	if pitch % item or pitch < shape[-1] * item:
		raise ValueError("%s: rows overlap or do not start on whole elements (strides %s)" % (what, strides))
	return pitch // item


def requireVector(ary, size, what):
	if ary is not None and (ary.dtype != np.float32 or ary.size != size or not ary.contiguous):
		raise ValueError("%s: contiguous float32 vector of %d expected, got %s %s" % (what, size, ary.dtype, ary.shape))


def requireDisjoint(what, out, *others):
	"""`out` shares no element with any of `others` (side by side columns of one buffer are fine)"""
	if out is None:
		return
	a, asize = out.gpudata.ptr, out.gpudata.size
	for other in others:
		if other is None:
			continue
		b, bsize = other.gpudata.ptr, other.gpudata.size
		if a + asize <= b or b + bsize <= a:
			continue
		if out.ndim >= 2 and other.ndim >= 2 and not (out.contiguous and other.contiguous):
			pitch = rowPitch(out, what) * out.dtype.itemsize
			if pitch == rowPitch(other, what) * other.dtype.itemsize:
				off = (a - b) % pitch
				if off >= other.shape[-1] * other.dtype.itemsize and off + out.shape[-1] * out.dtype.itemsize <= pitch:
					continue
		raise ValueError("%s overlaps one of the operands" % what)
