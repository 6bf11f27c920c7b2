"""
Timed cases of the operators of a feed-forward block over rows of channels (tokens, or pixels of a channels-last map):

  linear     y = residual + dropout(act(x W + b)), and its backward pass (dx, dW, db)      blas.linear / blas.linearBackward
  dropout    y = residual + x * keep / (1 - p), the mask drawn from a counter and never stored      counterDropoutKer
  groupnorm  y = act(gamma * (x - mean) / sqrt(var + eps) + beta) per sample and group of channels, channels last, and its
             backward pass                                                     dnn.groupNormNd / dnn.groupNormNdBackward

`own` false: the plain form, elementary torch operations in float32, rounded once at the end. `own` true: the calls a user of
this package makes. Both sides work on the same torch tensors (the package sees their memory as its own arrays).
"""
import math

import numpy as np
import torch

own = False

ACTS = ("none", "relu", "gelu", "silu")
DTYPES = {"f32": torch.float32, "f16": torch.float16}
NUMPY = {torch.float32: np.float32, torch.float16: np.float16}
EPSILON = 1e-5


# ------------------------------------------------------------------------------------------------ cases
def linear(way, dtype, m, k, n, act, p=0.0, residual=False, preact=False):
	return {"op": "linear", "way": way, "dtype": dtype, "m": m, "k": k, "n": n, "act": act, "p": p, "residual": residual,
			"preact": preact}


def dropout(dtype, rows, cols, p, residual):
	return {"op": "dropout", "dtype": dtype, "rows": rows, "cols": cols, "p": p, "residual": residual}


def groupnorm(way, dtype, batch, pixels, channels, groups, act):
	return {"op": "groupnorm", "way": way, "dtype": dtype, "batch": batch, "pixels": pixels, "channels": channels,
			"groups": groups, "act": act}


def listed():
	return [
		# the widening layer of a feed-forward block on a training batch of 8192 tokens: the pre-activation is kept for the way back
		dict(linear("fwd", "f16", 8192, 2048, 8192, "gelu", preact=True), name="linear_widen_f16"),
		# its narrowing layer: dropout and the residual sum behind the product
		dict(linear("fwd", "f16", 8192, 8192, 2048, "none", p=0.1, residual=True), name="linear_narrow_f16"),
		# the widening layer's backward pass: gate, bias gradient, data gradient and weight gradient
		dict(linear("bwd", "f16", 8192, 2048, 8192, "gelu"), name="linear_back_f16"),
		# one token of a serving step: the weights are read once
		dict(linear("fwd", "f16", 1, 4096, 16384, "silu"), name="linear_token_f16"),
		# a serving step of a few ragged requests, odd width
		dict(linear("fwd", "f16", 37, 1001, 4099, "gelu", residual=True), name="linear_odd_f16"),
		# the 4096 x 4096 x 4096 product of the package's GEMM benchmark, float32, with an epilogue
		dict(linear("fwd", "f32", 4096, 4096, 4096, "relu", residual=True), name="linear_f32"),
		# a classifier of 1000 classes over 2048 features at batch 256, float32, trained with dropout in front of its output
		dict(linear("bwd", "f32", 256, 2048, 1000, "gelu", p=0.5), name="linear_back_f32"),
		# dropout and the residual sum on the activations of a large training batch
		dict(dropout("f16", 8192, 8192, 0.1, True), name="dropout_large_f16"),
		# dropout on the hidden layer of a small classifier: launch latency
		dict(dropout("f32", 256, 1024, 0.5, False), name="dropout_small_f32"),
		# a 64 x 64 feature map of 512 channels at batch 32, in front of a 1 x 1 product
		dict(groupnorm("fwd", "f16", 32, 4096, 512, 32, "silu"), name="groupnorm_map_f16"),
		# the backward pass on 32 x 32 maps
		dict(groupnorm("bwd", "f16", 64, 1024, 512, 32, "silu"), name="groupnorm_back_f16"),
		# an odd map of an odd batch, float32, 10 channels to a group
		dict(groupnorm("bwd", "f32", 3, 37 * 53, 320, 32, "relu"), name="groupnorm_odd_f32"),
	]


def spread(rng, low, high):
	return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
	kind = rng.choice(("linear", "linear", "linear", "dropout", "groupnorm", "groupnorm"))
	dtype = rng.choice(("f16", "f16", "f32"))
	way = rng.choice(("fwd", "fwd", "bwd"))
	residual = rng.random() < 0.5
	p = rng.choice((0.0, 0.1, 0.25, 0.5))

	if kind == "linear":
		budget = (1 << 37) if dtype == "f16" else (1 << 35)             # products of one matrix product
		while True:
			m, k, n = spread(rng, 1, 16384), spread(rng, 64, 8192), spread(rng, 64, 16384)
			if rng.random() < 0.6:                                      # widths of networks are mostly multiples of 64
				k, n = -(-k // 64) * 64, -(-n // 64) * 64
			if m * k * n <= budget:
				break
		act = rng.choice(ACTS)
		return linear(way, dtype, m, k, n, act, p, residual and way == "fwd", way == "fwd" and act != "none" and rng.random() < 0.5)

	if kind == "dropout":
		cols = spread(rng, 16, 8192)
		rows = spread(rng, 1, (1 << 26) // cols)
		return dropout(dtype, rows, cols, rng.choice((0.1, 0.25, 0.5)), residual)

	width, groups = rng.choice((1, 2, 3, 4, 8, 10, 16, 20, 32, 64)), rng.choice((1, 2, 3, 8, 16, 32))
	channels = width * groups
	batch = spread(rng, 1, 128)
	pixels = spread(rng, 1, max(2, min(16384, (1 << 26) // (batch * channels))))
	pixels = max(pixels, -(-16 // width))                               # statistics of fewer than 16 values say nothing
	return groupnorm(way, dtype, batch, pixels, channels, groups, rng.choice(ACTS))


# ------------------------------------------------------------------------------------------------ inputs
def inputs(case, seed):
	gen = torch.Generator(device="cuda")
	gen.manual_seed(seed)
	dtype = DTYPES[case["dtype"]]

	def normal(*shape, std=1.0, mean=0.0, dtype=torch.float32):
		return (torch.randn(*shape, generator=gen, device="cuda") * std + mean).to(dtype)

	def empty(*shape, dtype=torch.float32):
		return torch.empty(*shape, dtype=dtype, device="cuda")

	# the key of the mask: what a generator hands out for one call
	state = {"case": case, "key": (0x9E3779B97F4A7C15 ^ (seed * 0x2545F4914F6CDD1D) & 0xffffffffffffffff, 7 + seed % 1000)}
	t = state["t"] = {}
	out = state["out"] = {}

	if case["op"] == "linear":
		m, k, n = case["m"], case["k"], case["n"]
		t["x"] = normal(m, k, dtype=dtype)
		t["W"] = normal(k, n, std=1.0 / math.sqrt(k), dtype=dtype)
		t["b"] = normal(n, std=0.1)
		if case["way"] == "fwd":
			if case["residual"]:
				t["residual"] = normal(m, n, dtype=dtype)
			out["y"] = empty(m, n, dtype=dtype)
			if case["preact"]:
				out["preact"] = empty(m, n, dtype=dtype)
		else:
			if case["act"] != "none":
				t["preact"] = (t["x"].float() @ t["W"].float() + t["b"]).to(dtype)
			t["dy"] = normal(m, n, dtype=dtype)
			out.update(dx=empty(m, k, dtype=dtype), dW=empty(k, n, dtype=dtype), db=empty(n))

	elif case["op"] == "dropout":
		shape = (case["rows"], case["cols"])
		t["x"] = normal(*shape, dtype=dtype)
		if case["residual"]:
			t["residual"] = normal(*shape, dtype=dtype)
		out["y"] = empty(*shape, dtype=dtype)

	else:
		b, s, c, g = case["batch"], case["pixels"], case["channels"], case["groups"]
		t["x"] = (normal(b, s, c, std=1.5) + normal(c)).to(dtype)          # channels have means of their own
		t["gamma"], t["beta"] = normal(c, std=0.1, mean=1.0), normal(c, std=0.1)
		if case["way"] == "fwd":
			out.update(y=empty(b, s, c, dtype=dtype), mean=empty(b, g), invvar=empty(b, g))
		else:
			grouped = t["x"].float().reshape(b, s, g, c // g)
			mean = grouped.mean(dim=(1, 3), keepdim=True)
			var = ((grouped - mean) ** 2).mean(dim=(1, 3))
			t["mean"], t["invvar"] = mean.reshape(b, g).contiguous(), 1.0 / torch.sqrt(var + EPSILON)
			t["dy"] = normal(b, s, c, dtype=dtype)
			out.update(dx=empty(b, s, c, dtype=dtype), dgamma=empty(c), dbeta=empty(c))

	return state


def prepare(case, seed):
	state = inputs(case, seed)
	if own:
		t, out = state["t"], state["out"]
		from puzzlelib_amd import backend, driver
		from puzzlelib_amd.gpuarray import GPUArray

		def view(tensor):
			span = driver.Buffer(tensor.data_ptr(), tensor.numel() * tensor.element_size())
			return GPUArray(tuple(tensor.shape), NUMPY[tensor.dtype], gpudata=span)

		bnd = state["bnd"] = backend.getBackend(0, initmode=2)
		state["a"] = {name: view(tensor) for name, tensor in list(t.items()) + [(name, out[name]) for name in out]}
		state["act"] = bnd.FusedAct[case.get("act", "none")]
		state["mask"] = bnd.DropoutMask(*state["key"], case["p"]) if case.get("p", 0.0) > 0.0 else None
	return state


# ------------------------------------------------------------------------------------------------ one pass
def run(state):
	return runOwn(state) if own else runPlain(state)


def runOwn(state):
	case, bnd, a, out = state["case"], state["bnd"], state["a"], state["out"]

	if case["op"] == "linear" and case["way"] == "fwd":
		bnd.blas.linear(
			a["x"], a["W"], a["b"], act=state["act"], residual=a.get("residual"), dropout=state["mask"], preact=a.get("preact"),
			out=a["y"], allocator=bnd.memoryPool
		)
	elif case["op"] == "linear":
		bnd.blas.linearBackward(
			a["dy"], a["x"], a["W"], act=state["act"], preact=a.get("preact"), dropout=state["mask"], wgrad=a["dW"], bgrad=a["db"],
			out=a["dx"], allocator=bnd.memoryPool
		)
	elif case["op"] == "dropout":
		bnd.counterDropoutKer(a["x"].dtype)(a["y"], a["x"], state["mask"], residual=a.get("residual"))
	elif case["way"] == "fwd":
		bnd.dnn.groupNormNd(
			a["x"], a["gamma"], a["beta"], case["groups"], EPSILON, act=state["act"], out=a["y"], savemean=a["mean"],
			saveinvvar=a["invvar"], allocator=bnd.memoryPool
		)
	else:
		bnd.dnn.groupNormNdBackward(
			a["dy"], a["x"], a["gamma"], a["beta"], a["mean"], a["invvar"], case["groups"], act=state["act"], out=a["dx"],
			scalegrad=a["dgamma"], bgrad=a["dbeta"], allocator=bnd.memoryPool
		)
	return out


LOW32 = 0xffffffff


def keepPlain(key, p, count):
	"""1 / (1 - p) where element i is kept and 0 elsewhere: word i % 4 of Philox4x32-10 at counter {i / 4, call} under the seed,
	kept where word < (1 - p) * (2^32 - 1). 32-bit words in int64 tensors: their products wrap to the right low 64 bits."""
	seed, call = key
	quads = torch.arange((count + 3) // 4, dtype=torch.int64, device="cuda")
	c0, c1 = quads & LOW32, quads >> 32
	c2, c3 = torch.full_like(quads, call & LOW32), torch.full_like(quads, call >> 32)
	k0, k1 = seed & LOW32, seed >> 32
	for _ in range(10):
		p0, p1 = c0 * 0xD2511F53, c2 * 0xCD9E8D57
		c0, c1, c2, c3 = (p1 >> 32 & LOW32) ^ c1 ^ k0, p1 & LOW32, (p0 >> 32 & LOW32) ^ c3 ^ k1, p0 & LOW32
		k0, k1 = (k0 + 0x9E3779B9) & LOW32, (k1 + 0xBB67AE85) & LOW32
	words = torch.stack((c0, c1, c2, c3), dim=1).reshape(-1)[:count]
	return (words < int((1.0 - p) * LOW32)).float() / (1.0 - p)


def actPlain(z, act):
	if act == "relu":
		return torch.clamp(z, min=0.0)
	if act == "gelu":
		return 0.5 * z * (1.0 + torch.erf(z * math.sqrt(0.5)))
	if act == "silu":
		return z / (1.0 + torch.exp(-z))
	return z


def actDerPlain(z, act):
	if act == "relu":
		return (z > 0.0).float()
	if act == "gelu":
		return 0.5 * (1.0 + torch.erf(z * math.sqrt(0.5))) + z * torch.exp(-0.5 * z * z) * (1.0 / math.sqrt(2.0 * math.pi))
	sig = 1.0 / (1.0 + torch.exp(-z))
	return sig * (1.0 + z * (1.0 - sig))


def runPlain(state):
	case, t = state["case"], state["t"]
	dtype = DTYPES[case["dtype"]]

	if case["op"] == "linear" and case["way"] == "fwd":
		z = t["x"].float() @ t["W"].float() + t["b"]
		y = actPlain(z, case["act"])
		if case["p"] > 0.0:
			y = y * keepPlain(state["key"], case["p"], y.numel()).reshape(y.shape)
		if case["residual"]:
			y = y + t["residual"].float()
		return {"y": y.to(dtype), "preact": z.to(dtype)} if case["preact"] else {"y": y.to(dtype)}

	if case["op"] == "linear":
		dz = t["dy"].float()
		if case["p"] > 0.0:
			dz = dz * keepPlain(state["key"], case["p"], dz.numel()).reshape(dz.shape)
		if case["act"] != "none":
			dz = dz * actDerPlain(t["preact"].float(), case["act"])
		dx, dW = dz @ t["W"].float().t(), t["x"].float().t() @ dz
		return {"dx": dx.to(dtype), "dW": dW.to(dtype), "db": dz.sum(dim=0)}

	if case["op"] == "dropout":
		y = t["x"].float() * keepPlain(state["key"], case["p"], t["x"].numel()).reshape(t["x"].shape)
		return {"y": (y + t["residual"].float() if case["residual"] else y).to(dtype)}

	b, s, c, g = case["batch"], case["pixels"], case["channels"], case["groups"]
	x = t["x"].float().reshape(b, s, g, c // g)
	gamma, beta = t["gamma"].reshape(g, c // g), t["beta"].reshape(g, c // g)
	if case["way"] == "fwd":
		mean = x.mean(dim=(1, 3), keepdim=True)
		var = ((x - mean) ** 2).mean(dim=(1, 3), keepdim=True)
		invvar = 1.0 / torch.sqrt(var + EPSILON)
		y = actPlain((x - mean) * invvar * gamma + beta, case["act"])
		return {"y": y.reshape(b, s, c).to(dtype), "mean": mean.reshape(b, g), "invvar": invvar.reshape(b, g)}

	invvar = t["invvar"].reshape(b, 1, g, 1)
	xhat = (x - t["mean"].reshape(b, 1, g, 1)) * invvar
	dy = t["dy"].float().reshape(b, s, g, c // g)
	if case["act"] != "none":
		dy = dy * actDerPlain(xhat * gamma + beta, case["act"])
	dgamma, dbeta = (dy * xhat).sum(dim=(0, 1)), dy.sum(dim=(0, 1))
	dxhat = dy * gamma
	dx = invvar * (dxhat - dxhat.mean(dim=(1, 3), keepdim=True) - xhat * (dxhat * xhat).mean(dim=(1, 3), keepdim=True))
	return {"dx": dx.reshape(b, s, c).to(dtype), "dgamma": dgamma.reshape(c), "dbeta": dbeta.reshape(c)}


# ------------------------------------------------------------------------------------------------ what a pass cannot do without
def work(case):
	size = 4 if case["dtype"] == "f32" else 2
	if case["op"] == "linear":
		m, k, n = case["m"], case["k"], case["n"]
		if case["way"] == "fwd":
			tensors = m * k + k * n + m * n * (1 + int(case["residual"]) + int(case["preact"]))
			return {"bytes": size * tensors + 4 * n, "flops": 2 * m * k * n}
		tensors = 2 * m * k + 2 * k * n + m * n * (1 + int(case["act"] != "none"))
		return {"bytes": size * tensors + 4 * n, "flops": 4 * m * k * n}
	if case["op"] == "dropout":
		count = case["rows"] * case["cols"]
		return {"bytes": size * count * (2 + int(case["residual"])), "flops": 2 * count}
	count, stats = case["batch"] * case["pixels"] * case["channels"], 8 * case["batch"] * case["groups"]
	if case["way"] == "fwd":
		return {"bytes": 2 * size * count + stats + 8 * case["channels"], "flops": 8 * count}
	return {"bytes": 3 * size * count + stats + 16 * case["channels"], "flops": 16 * count}


# ------------------------------------------------------------------------------------------------ in 64 bits, from the definitions
def keepExact(key, p, count):
	"""The mask in numpy, word by word from the definition of Philox4x32-10 (J. Salmon et al., "Parallel random numbers: as easy
	as 1, 2, 3")."""
	mask = np.uint64(LOW32)
	shift = np.uint64(32)
	index = np.arange((count + 3) // 4, dtype=np.uint64)
	words = [index & mask, index >> shift, np.full_like(index, key[1] & LOW32), np.full_like(index, key[1] >> 32)]
	keys = [key[0] & LOW32, key[0] >> 32]
	for _ in range(10):
		first, third = words[0] * np.uint64(0xD2511F53), words[2] * np.uint64(0xCD9E8D57)
		words = [
			(third >> shift) ^ words[1] ^ np.uint64(keys[0]), third & mask, (first >> shift) ^ words[3] ^ np.uint64(keys[1]), first & mask
		]
		keys = [(keys[0] + 0x9E3779B9) % (1 << 32), (keys[1] + 0xBB67AE85) % (1 << 32)]
	flat = np.empty((index.size, 4), dtype=bool)
	for lane in range(4):
		flat[:, lane] = words[lane] < np.uint64(int((1.0 - p) * LOW32))
	return torch.from_numpy(flat.reshape(-1)[:count].copy()).cuda().double() / (1.0 - p)


def actExact(z, act):
	return {
		"none": lambda: z, "relu": lambda: torch.where(z > 0, z, torch.zeros_like(z)), "gelu": lambda: z * torch.special.ndtr(z),
		"silu": lambda: z * torch.sigmoid(z)
	}[act]()


def exact(case, seed):
	state = inputs(case, seed)
	t = {name: tensor.double() for name, tensor in state["t"].items()}
	torch.cuda.synchronize()

	if case["op"] == "dropout" or case["op"] == "linear":
		shape = (case["rows"], case["cols"]) if case["op"] == "dropout" else (case["m"], case["n"])
		keep = keepExact(state["key"], case["p"], shape[0] * shape[1]).reshape(shape) if case["p"] > 0.0 else 1.0

	if case["op"] == "dropout":
		return {"y": torch.where(keep > 0, t["x"] * keep, 0.0) + t.get("residual", 0.0)}

	if case["op"] == "linear" and case["way"] == "fwd":
		z = torch.addmm(t["b"], t["x"], t["W"])
		y = actExact(z, case["act"]) * keep + t.get("residual", 0.0)
		return {"y": y, "preact": z} if case["preact"] else {"y": y}

	if case["op"] == "linear":
		z = t["preact"].requires_grad_() if case["act"] != "none" else torch.zeros_like(t["dy"]).requires_grad_()
		dz, = torch.autograd.grad(actExact(z, case["act"]) * keep, z, t["dy"])
		return {"dx": torch.mm(dz, t["W"].T.contiguous()), "dW": torch.mm(t["x"].T.contiguous(), dz), "db": dz.sum(0)}

	b, s, c, g = case["batch"], case["pixels"], case["channels"], case["groups"]

	def forward(x, gamma, beta, mean, invvar):
		spread = lambda v: v.repeat_interleave(c // g, dim=1).unsqueeze(1)              # (b, g) -> (b, 1, c)
		return actExact(gamma * (x - spread(mean)) * spread(invvar) + beta, case["act"])

	def moments(x):
		rows = x.reshape(b, s, g, c // g).transpose(1, 2).reshape(b, g, -1)
		return rows.mean(-1), (rows.var(-1, unbiased=False) + EPSILON) ** -0.5

	if case["way"] == "fwd":
		mean, invvar = moments(t["x"])
		return {"y": forward(t["x"], t["gamma"], t["beta"], mean, invvar), "mean": mean, "invvar": invvar}

	leaves = [t[name].requires_grad_() for name in ("x", "gamma", "beta")]
	# the saved statistics are what the backward pass is given; how they move with x comes from their definition
	y = forward(*leaves, *moments(leaves[0]))
	return dict(zip(("dx", "dgamma", "dbeta"), torch.autograd.grad(y, leaves, t["dy"])))
