"""The debug build of the four-bit cache's kernels (tests/test_range_check_gpu.py says what it is): indices beyond the declared
bounds are reported, and the ordinary tests of attention and of the products run green in it. Child processes, because the build
is chosen when the libraries are loaded."""
import os
import sys

import pytest

from test_range_check_gpu import HERE, run

pytestmark = pytest.mark.gpu


def test_an_index_beyond_the_declared_bounds_is_reported_and_the_access_left_out():
    proc = run([os.path.join(HERE, "range_check_four_bits.py")])
    assert proc.returncode == 0 and "four-bit range check cases ok" in proc.stdout, (proc.stdout + proc.stderr)[-3000:]


def test_the_edges_run_green_in_the_debug_build():
    proc = run(["-m", "pytest", os.path.join(HERE, "test_four_bits_edges_gpu.py"), "-q", "-x", "-m", "gpu", "-k", "chunks_of_any or behind or gigabytes"])
    assert proc.returncode == 0 and " passed" in proc.stdout, (proc.stdout + proc.stderr)[-3000:]
