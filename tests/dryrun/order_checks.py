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


if __name__ == "__main__":
	globals()[sys.argv[1]]()
	print("OK")
