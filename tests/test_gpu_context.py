"""The library in a thread whose current context is not the device's primary one."""
from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

ROOT = Path(__file__).resolve().parents[1]

# No kernel is launched and no memory touched: only the context that the call leaves is looked at.
CHILD = """
import ctypes, sys
sys.path.insert(0, sys.argv[1])
from arc._lib import OP_LINEAR, kernel_name
cuda = ctypes.CDLL("libcuda.so.1")
dev, mine, now = ctypes.c_int(), ctypes.c_void_p(), ctypes.c_void_p()
assert cuda.cuInit(0) == 0 and cuda.cuDeviceGet(ctypes.byref(dev), 0) == 0
assert cuda.cuCtxCreate_v2(ctypes.byref(mine), 0, dev) == 0
assert kernel_name(OP_LINEAR, 16, 14336, 4096).startswith("gemm_linear")
assert cuda.cuCtxGetCurrent(ctypes.byref(now)) == 0
assert now.value == mine.value, "the caller's context was replaced"
assert cuda.cuCtxDestroy_v2(mine) == 0
print("kept")
"""


def test_the_callers_context_stays(cuda_device):
    res = subprocess.run([sys.executable, "-c", CHILD, str(ROOT / "arc-gemm_b200")], capture_output=True, text=True,
                         timeout=120)
    assert res.returncode == 0 and "kept" in res.stdout, res.stdout + res.stderr
