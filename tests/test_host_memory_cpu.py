"""C entries that run out of host memory return a status; no C++ exception leaves them."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

PACKAGE = Path(__file__).resolve().parent.parent / "llm-serving_b200"
CHECK = """
import ctypes, resource, sys
import numpy
sys.path.insert(0, {package!r})
from model import _native
layers, at = 30_000_000, 1 << 20
array = numpy.full(layers, at, dtype=numpy.int64)
pools = ctypes.cast(array.ctypes.data, ctypes.POINTER(ctypes.c_void_p))
s3 = (ctypes.c_int64 * 3)(2048, 128, 64)
here = ctypes.c_void_p(at)
used = int(open("/proc/self/statm").read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (64 << 20),) * 2)
status = _native.lib.pd_evict(pools, pools, layers, 8, 16, 2, 64, _native.PD_BF16, s3, s3, here, 4, 4, None, 0, 0, here, here,
                              here, s3, here, s3, 64, 1, 8, 2, 1, here, 1 << 20, None)
print("status", status, _native.lib.pd_last_error_string().decode())
"""


def test_eviction_of_more_layers_than_memory():
    done = subprocess.run([sys.executable, "-c", CHECK.format(package=str(PACKAGE))], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0, done.stderr
    assert done.stdout.strip() == "status 1 no host memory for that many layers"
