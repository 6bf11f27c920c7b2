"""
CPU tests of how launches on other streams — the gradient exchange's collectives, the package's entries that take a stream — are ordered
against float16 products and against the main stream. Each runs in a child process in dry-run mode (tests/dryrun/order_checks.py).
"""
import os, subprocess, sys

import pytest

from conftest import ROOT

SCRIPT = os.path.join(ROOT, "tests", "dryrun", "order_checks.py")


@pytest.mark.parametrize("check", ["collectives", "collective_out_of_a_barrier", "float32_needs_no_order", "streams", "preact_is_a_choice", "filter_gradient_behind_a_row_operator"])
def test_order(check):
	env = dict(os.environ, PUZZLE_MI355_DRYRUN="1", PUZZLE_MI355_LAZY="1")
	env.pop("PUZZLE_MI355_DEBUG_ALLOC", None)
	res = subprocess.run([sys.executable, SCRIPT, check], env=env, capture_output=True, text=True, timeout=300)
	assert res.returncode == 0 and "OK" in res.stdout, "%s failed:\n%s\n%s" % (check, res.stdout[-3000:], res.stderr[-6000:])
