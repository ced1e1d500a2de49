"""A pool that host memory does not suffice for is refused: no exception leaves the C entry point."""
import os
import subprocess
import sys

import pytest

RUN = """
import ctypes, resource, sys
sys.path.insert(0, sys.argv[1])
import gkv
L, h = gkv.lib(), ctypes.c_void_p()
with open("/proc/self/statm") as f:
    used = int(f.read().split()[0]) * resource.getpagesize()
resource.setrlimit(resource.RLIMIT_AS, (used + (1 << 30), used + (1 << 30)))
cfg = gkv.PoolConfig(2**31 - 1, 1, 64, int(sys.argv[2]), 2, 100, 8, 0, 0, 0)  # (a list of 8 GB over the layers)
st = L.gkv_pool_create_kept(ctypes.byref(cfg), 16, ctypes.byref(h)) if cfg.window else L.gkv_pool_create(
    ctypes.byref(cfg), ctypes.byref(h))
print("status", st, h.value)
"""


@pytest.mark.parametrize("window", [0, 32])
def test_no_exception_leaves_the_pool(gkv, window):
    p = subprocess.run([sys.executable, "-c", RUN, os.path.dirname(gkv.__file__), str(window)], capture_output=True,
                       text=True, timeout=300)
    assert p.returncode == 0 and p.stdout.split()[-3:] == ["status", str(gkv.GKV_ERR_CAPACITY), "None"], p.stderr[-500:]
