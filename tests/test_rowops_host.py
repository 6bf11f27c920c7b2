"""
CPU tests of the operators over rows of channels (blas.linear, counterDropoutKer, dnn.groupNormNd and their backward passes): what they
refuse, the workspace sizes they ask for, how float16 products are kept apart from other streams' kernels. Each runs in a child process
in dry-run mode (tests/dryrun/rowops_checks.py).
"""
import ctypes, os, subprocess, sys

import pytest

from conftest import ROOT

SCRIPT = os.path.join(ROOT, "tests", "dryrun", "rowops_checks.py")


@pytest.mark.parametrize("check", ["linear_refusals", "linear_c_entry_refusals", "workspace_sizes", "dropout_refusals", "groupnorm_refusals",
								   "matrix_kernels_keep_apart"])
def test_rowops(check):
	env = dict(os.environ, PUZZLE_MI355_DRYRUN="1", PUZZLE_MI355_LAZY="1")
	env.pop("PUZZLE_MI355_DEBUG_ALLOC", None)
	res = subprocess.run([sys.executable, SCRIPT, check], env=env, capture_output=True, text=True, timeout=300)
	assert res.returncode == 0 and "OK" in res.stdout, "%s failed:\n%s\n%s" % (check, res.stdout[-3000:], res.stderr[-6000:])


def test_struct_layouts():
	from puzzlelib_amd import lib
	assert ctypes.sizeof(lib.DropoutKey) == 24 and ctypes.sizeof(lib.LinearDesc) == 6 * 4 + 5 * 8 and ctypes.sizeof(lib.GroupNormDesc) == 28
