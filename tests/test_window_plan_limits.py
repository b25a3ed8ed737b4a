"""CPU tests of the window planner at the ends of host memory and of its arguments."""
import subprocess
import sys
from pathlib import Path

import pytest

from inferno_amd import _lib
from inferno_amd.kv import KVRunTable, WindowPlan

ROOT = Path(__file__).resolve().parent.parent

NO_MEMORY = """
import ctypes as C, resource
import numpy as np
from inferno_amd import _lib

lib, n = _lib.lib(), 1 << 20
runs = np.zeros((n, 4), dtype=np.int32)
runs[:, 0] = np.arange(n)
runs[:, 3] = 1
rows = np.zeros(1, dtype=np.int32)
img = np.ones(lib.ifr_plan_window_bytes(n, 1, n, 0) // 4, dtype=np.int32)
info = (C.c_int64 * _lib.WINDOW_INFO_LEN)()

def plan():
    return lib.ifr_plan_window(img.ctypes.data, img.nbytes, runs.ctypes.data_as(_lib.P_I32), n, rows.ctypes.data_as(_lib.P_I32), 1,
                               n, 0, 0, 64, 64, 8, 8, 128, 0, info)

size = int(next(l for l in open("/proc/self/status") if l.startswith("VmSize")).split()[1]) << 10
kept = resource.getrlimit(resource.RLIMIT_AS)
resource.setrlimit(resource.RLIMIT_AS, (size + (8 << 20), kept[1]))
short = plan()
resource.setrlimit(resource.RLIMIT_AS, kept)
print("status", short, _lib.last_error())
print("status", plan())
"""


def test_a_plan_that_finds_no_host_memory_is_an_error():
    """A million sequences in an address space with 8 MiB left; then with what it was."""
    got = subprocess.run([sys.executable, "-c", NO_MEMORY], cwd=ROOT, capture_output=True, text=True, timeout=300)
    assert got.returncode == 0, got.stderr[-500:]
    lines = [l for l in got.stdout.splitlines() if l.startswith("status")]
    assert lines[0].startswith("status -5") and "host memory" in lines[0] and lines[1] == "status 0", got.stdout


@pytest.mark.parametrize("args", [((1 << 24) + 1, 1, 1 << 24, 0), (1, 1 << 29, 1, 0), (1, 1, (1 << 24) + 1, 0), (1, 1, 1 << 60, 0),
                                  (1 << 62, 1, 1, 16), (1, 1 << 62, 1, 0)])
def test_bytes_of_plans_that_there_are_not(args):
    assert _lib.lib().ifr_plan_window_bytes(*args) == -1


def test_bytes_of_the_largest_plans():
    assert _lib.lib().ifr_plan_window_bytes(1 << 24, (1 << 29) - 1, 1 << 24, 16) > 4 << 29


@pytest.mark.parametrize("tokens", [1 << 40, (1 << 62) + 1])
def test_the_plan_refuses_a_step_of_too_many_tokens_by_name(tokens):
    table = KVRunTable()
    table.begin_run(0, 0)
    table.add_base_row(0)
    with pytest.raises(_lib.InfernoHipError, match="seq_len"):
        WindowPlan(table, tokens, page_len=64, cache_rows=64, num_q=8, num_kv=8, head_dim=128, device="cpu")
