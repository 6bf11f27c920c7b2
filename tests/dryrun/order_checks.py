"""
The order of launches on several streams, without a device: the calls of the library are recorded in dry-run mode and replayed on a
model of streams and events, which tells for any two launches whether one waits for the other. Run by tests/test_rowops_order.py in a
child process. Usage: python tests/dryrun/order_checks.py <check name>
"""
import os, sys

assert os.environ.get("PUZZLE_MI355_DRYRUN") == "1"
ROOT = os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
sys.path.insert(0, ROOT)

import numpy as np

from puzzlelib_amd import backend, lib, lazy, grid

bnd = backend.getBackend(0, initmode=2)
A = lambda *shape, dtype=np.float32: bnd.GPUArray.empty(shape, dtype=dtype)

NO_LAUNCH = ("pz_event_", "pz_stream_", "pz_pool_", "pz_malloc", "pz_free", "pz_host_", "pz_device_", "pz_comm_init", "pz_comm_info", "pz_comm_unique",
			 "pz_comm_destroy", "pz_comm_probe", "pz_comm_async", "pz_comm_wait", "pz_rng_create", "pz_rng_reserve", "pz_rng_destroy", "pz_module_")


class Order:
	"""before[i]: the launches that have ended when launch i starts, by what streams and events say. No event ever completes early."""

	def __init__(self):
		self.launches, self.before, self.ends, self.marks, self.host = [], [], {}, {}, frozenset()

	def hook(self, name, args):
		value = lambda x: getattr(x, "value", x)
		if name == "pz_event_record":
			self.marks[value(args[0])] = self.ended(value(args[1]))
		elif name == "pz_stream_wait_event":
			stream = value(args[0])
			self.ends[stream] = self.ended(stream) | self.marks.get(value(args[1]), frozenset())
		elif name == "pz_stream_sync":
			self.host |= self.ended(value(args[0]))
		elif name == "pz_event_sync":
			self.host |= self.marks.get(value(args[0]), frozenset())
		elif name == "pz_event_query":
			lib._store(args[1], 0)
			return True
		elif not name.startswith(NO_LAUNCH):
			stream, index = value(args[-1]), len(self.launches)
			self.launches.append((name, stream))
			self.before.append(self.ended(stream))
			self.ends[stream] = self.ended(stream) | {index}
		return False

	def ended(self, stream):
		return self.ends.get(stream, frozenset()) | self.host

	def only(self, *names, since=0):
		found = [i for i, (n, _) in enumerate(self.launches) if n in names and i >= since]
		assert len(found) == 1, (names, self.launches[since:])
		return found[0]

	def follows(self, later, earlier):
		assert earlier in self.before[later], "%s does not wait for %s" % (self.launches[later], self.launches[earlier])


def watched():
	order = Order()
	lib.callHook = order.hook
	return order


def oneRank():
	import socket
	with socket.socket() as sock:
		sock.bind(("127.0.0.1", 0))
		port = sock.getsockname()[1]
	return grid.connectNode(0, 1, 0, "127.0.0.1", port)


def products(which):
	"""a float16 product, forward or backward -> a function that launches it"""
	x, W, g = A(8, 16, dtype=np.float16), A(16, 8, dtype=np.float16), A(8, 8, dtype=np.float16)
	return (lambda: bnd.blas.linear(x, W)) if which == "pz_linear_fwd" else (lambda: bnd.blas.linearBackward(g, x, W))


def collectives():
	"""a float16 product waits for every collective in flight, and a collective for every product, also when its bucket was final before"""
	node = oneRank()
	node.ensureComm()
	arena = A(4096)
	for entry in ("pz_linear_fwd", "pz_linear_bwd"):
		product = products(entry)
		for name, exchange in (("pz_comm_allreduce_sum_f32", lambda ops, token: ops.allreduce(0, 4096, token)),
							   ("pz_comm_allreduce_sum_f32_ranges", lambda ops, token: ops.allreduceRanges([(0, 1024), (2048, 4096)], token))):
			order = watched()
			ops = node.reduceOps(arena)
			exchange(ops, ops.markReady())
			product()
			order.follows(order.only(entry), order.only(name))
			# a bucket that was final in front of the product leaves behind it
			since = len(order.launches)
			token = ops.markReady()
			product()
			exchange(ops, token)
			order.follows(order.only(name, since=since), order.only(entry, since=since))
			# ... and another product after that
			since = len(order.launches)
			product()
			order.follows(order.only(entry, since=since), [i for i, (n, _) in enumerate(order.launches) if n == name][-1])
	node.close()


def collective_out_of_a_barrier():
	"""taking the address of a gradient block may hand an earlier bucket to the transport (grid.ArenaWatcher): the product whose gradient that
	is still follows the collective"""
	node = oneRank()
	node.ensureComm()
	arena = A(1024)
	ops = node.reduceOps(arena)
	wgrad, bgrad = A(16, 8), A(8)
	sent = []

	def watch(lo, hi):
		if not sent:
			sent.append(True)
			ops.allreduce(0, 4096, ops.markReady())

	for array in (wgrad, bgrad):
		lazy.stateOf(array.gpudata.root).watch = watch
		del sent[:]
		order = watched()
		bnd.blas.linearBackward(A(8, 8, dtype=np.float16), A(8, 16, dtype=np.float16), A(16, 8, dtype=np.float16), wgrad=wgrad, bgrad=bgrad)
		order.follows(order.only("pz_linear_bwd"), order.only("pz_comm_allreduce_sum_f32"))
		lazy.stateOf(array.gpudata.root).watch = None
	out = A(8, 8, dtype=np.float16)
	lazy.stateOf(out.gpudata.root).watch = watch
	del sent[:]
	order = watched()
	bnd.blas.linear(A(8, 16, dtype=np.float16), A(16, 8, dtype=np.float16), out=out)
	order.follows(order.only("pz_linear_fwd"), order.only("pz_comm_allreduce_sum_f32"))
	node.close()


def float32_needs_no_order():
	"""float32 products run beside collectives as before"""
	node = oneRank()
	node.ensureComm()
	order = watched()
	arena = A(4096)
	ops = node.reduceOps(arena)
	ops.allreduce(0, 4096, ops.markReady())
	since = len(order.launches)
	bnd.blas.linear(A(8, 16), A(16, 8))
	assert order.only("pz_comm_allreduce_sum_f32") not in order.before[order.only("pz_linear_fwd", since=since)]
	node.close()


def entries():
	"""every entry that takes a stream: name, launch(stream), the array it reads, the array it writes, the library call"""
	f, h = np.float32, np.float16
	x, y, z, e = A(64), A(64), A(64), A(1)
	labels, few = A(64, dtype=np.int32), A(8, dtype=np.int32)
	half, other = A(64, dtype=h), A(64)
	host = np.zeros(64, f)
	grid2 = A(8, 16)
	mask = bnd.DropoutMask(1, 2, 0.5)
	scale = bnd.ElementwiseKernel([("float *", "out"), ("const float *", "data")], "out[i] = 2 * data[i]", "scaleKer")
	total = bnd.ReductionKernel(f, "0", "a + b", "data[i]", [("const float *", "data")], "totalKer")
	return [
		("eltwise", lambda s: bnd.toVectorAddVectorKer(f)(y, x, 1.0, stream=s), x, y, "pz_eltwise"),
		("addKer", lambda s: bnd.addKer(f)(y, x, 1.0, z, 1.0, stream=s), x, y, "pz_eltwise"),
		("counterDropoutKer", lambda s: bnd.counterDropoutKer(f)(y, x, mask, stream=s), x, y, "pz_dropout"),
		("castFP32toFP16", lambda s: bnd.castFP32toFP16(half, x, stream=s), x, half, "pz_cast_f32_f16"),
		("castFP16toFP32", lambda s: bnd.castFP16toFP32(x, half, stream=s), half, x, "pz_cast_f16_f32"),
		("bceKer", lambda s: bnd.bceKer(x, labels, e, y, 64, 1, stream=s), x, y, "pz_cost_pointwise"),
		("bceKer's error", lambda s: bnd.bceKer(x, labels, e, y, 64, 1, stream=s), labels, e, "pz_cost_pointwise"),
		("hingeKer", lambda s: bnd.hingeKer(x, labels, e, y, 8, 8, stream=s), x, y, "pz_cost_pointwise"),
		("smoothL1Ker", lambda s: bnd.smoothL1Ker(x, z, e, y, 1.0, 1.0, stream=s), z, y, "pz_cost_pointwise"),
		("l1HingeKer", lambda s: bnd.l1HingeKer(x, z, few, e, y, other, 8, 8, stream=s), few, other, "pz_cost_pointwise"),
		("set from an array", lambda s: y.set(x, stream=s), x, y, "pz_memcpy_d2d"),
		("strided set", lambda s: grid2[:, :8].set(x.reshape(8, 8), stream=s), x, grid2, "pz_strided_copy"),
		("set from the host", lambda s: y.set(host, stream=s), None, y, "pz_memcpy_h2d"),
		("get", lambda s: x.get(stream=s), x, None, "pz_memcpy_d2h"),
		("Buffer.fillD32", lambda s: y.gpudata.fillD32(1, stream=s), None, y, "pz_memset_d32"),
		("Buffer.copy", lambda s: x.gpudata.copy(y.gpudata, stream=s), x, y, "pz_memcpy_d2d"),
		("Buffer.set", lambda s: y.gpudata.set(host.ctypes.data, 256, stream=s), None, y, "pz_memcpy_h2d"),
		("Buffer.get", lambda s: x.gpudata.get(host.ctypes.data, 256, stream=s), x, None, "pz_memcpy_d2h"),
		("memcpy2D", lambda s: bnd.Driver.memcpy2D(16, 4, x.gpudata, 32, y.gpudata, 32, stream=s), x, y, "pz_memcpy_2d"),
		("ElementwiseKernel", lambda s: scale(y, x, stream=s), x, y, "pz_function_launch"),
		("ReductionKernel", lambda s: total(x, stream=s), x, None, "pz_function_launch"),
	]


def streams():
	"""each entry on a stream of the caller's: behind what the main stream was given, in front of what touches the same arrays there
	afterwards, and apart from float16 products on either side"""
	product = products("pz_linear_fwd")
	for name, launch, source, target, entry in entries():
		stream = bnd.Driver.Stream()
		order = watched()
		if source is not None:
			source.gpudata.fillD32(7)                            # its input is written on the main stream ...
		product()                                                # ... and a product runs there
		earlier = len(order.launches)
		launch(stream)
		foreign = [i for i, (n, s) in enumerate(order.launches) if n == entry and s == stream.handle]
		assert foreign and foreign[0] >= earlier, (name, order.launches)
		for i in foreign:
			for j in range(earlier):
				order.follows(i, j)
		product()
		order.follows(len(order.launches) - 1, foreign[-1])
		# afterwards on the main stream: reading what was written, overwriting what was read
		order = watched()
		launch(stream)
		foreign = [i for i, (n, s) in enumerate(order.launches) if n == entry and s == stream.handle]
		for array in (source, target):
			if array is not None:
				since = len(order.launches)
				(array.gpudata.copy if array is target else lambda: array.gpudata.fillD32(9))()
				order.follows(since, foreign[-1 if array is target else 0])         # (a reduction reads in its first launch)


def preact_is_a_choice():
	"""preact=False is what it says, as None is"""
	x, W = A(4, 16), A(16, 8)
	for preact in (None, False):
		lib.trace.clear()
		assert bnd.blas.linear(x, W, preact=preact).shape == (4, 8)
	out, z = bnd.blas.linear(x, W, preact=True)
	assert out.shape == z.shape == (4, 8)


def filter_gradient_behind_a_row_operator():
	"""A filter gradient may start at the mark in front of its layer's backward-data kernel, earlier than where it is called. Its workspace may
	be memory that an operator called in between has just given back, so it follows that operator."""
	f = np.float32
	dnn, conv = bnd.dnn, lambda: (A(8, 16, 12, 12), A(32, 16, 3, 3), A(8, 32, 10, 10))
	x, W, g = conv()
	wgrad, bgrad = A(32, 16, 3, 3), A(32)
	rows, V, norm, stat = A(6, 8), A(8, 10), A(2, 5, 12), A(2, 3)
	between = {
		"pz_linear_fwd": lambda: bnd.blas.linear(rows, V), "pz_linear_bwd": lambda: bnd.blas.linearBackward(A(6, 10), rows, V),
		"pz_groupnorm_fwd": lambda: dnn.groupNormNd(norm, None, None, 3),
		"pz_groupnorm_bwd": lambda: dnn.groupNormNdBackward(norm, norm, None, None, stat, stat, 3),
		"pz_dropout": lambda: bnd.counterDropoutKer(f)(A(6, 8), rows, bnd.DropoutMask(1, 2, 0.5)),
	}
	for entry in (None, ) + tuple(between):
		order = watched()
		taken = lazy.counters.get("wgrad_early_start", 0)
		ingrad = dnn.convNdBackwardData(g, W, data=x)
		if entry is not None:
			between[entry]()
		dnn.convNdBackwardParams(x, g, W, withbias=True, wgrad=wgrad, bgrad=bgrad, momentum=1.0)
		del ingrad
		filters = [i for i, (n, s) in enumerate(order.launches) if n.startswith("pz_conv2d_bwd_filter")][-1]
		assert order.launches[filters][1] is not None, "no second stream: nothing is tested"
		if entry is None:
			assert lazy.counters["wgrad_early_start"] == taken + 1, "no early start: nothing is tested"
		else:
			order.follows(filters, order.only(entry))


if __name__ == "__main__":
	globals()[sys.argv[1]]()
	print("OK")
