"""First calls of several host threads at once, of different sizes, in a process of their own."""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

import pytest

pytestmark = pytest.mark.gpu

PACKAGE = Path(__file__).resolve().parent.parent / "llm-serving_b200"

PROGRAM = """
import sys, threading
sys.path.insert(0, sys.argv[1])
import torch
from model import _native
from model.paged_fp4 import fp4_pages, fp4_workspace

torch.cuda.init()
calls = []
for d in (64, 128, 256):
    pages = fp4_pages(4, 16, 1, d)
    for rows, heads in ((1, 1), (896, 8), (33, 4), (896, 1), (300, 8), (1, 8)):
        q = torch.zeros(rows, heads, d, dtype=torch.bfloat16, device="cuda")
        calls.append((pages, q, torch.full_like(q, 7), torch.zeros(rows, 1, dtype=torch.int32, device="cuda"),
                      torch.ones(rows, dtype=torch.int32, device="cuda"), fp4_workspace(pages)))
torch.cuda.synchronize()
barrier = threading.Barrier(len(calls))
status = [None] * len(calls)

def run(i):
    pages, q, out, table, lens, ws = calls[i]
    rows, heads, d = q.shape
    barrier.wait()
    # ctypes gives the interpreter's lock up for the call
    status[i] = _native.lib.pd_fp4_decode(q.data_ptr(), heads * d, d, pages.data_ptr(), 4, 16, None, table.data_ptr(), 1, 1,
                                          lens.data_ptr(), out.data_ptr(), heads * d, d, rows, heads, 1, d,
                                          _native.PD_BF16, 1.0, ws.data_ptr(), ws.numel(), None)

for _ in range(2):
    threads = [threading.Thread(target=run, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    assert status == [0] * len(calls), status
    assert all(not out.any() for _, _, out, _, _, _ in calls)
    for _, _, out, _, _, _ in calls:
        out.fill_(7)
assert _native.device_error() == 0
"""


def test_threads_whose_first_calls_need_different_amounts_of_shared_memory(cuda_device):
    for _ in range(3):
        done = subprocess.run([sys.executable, "-c", PROGRAM, str(PACKAGE)], capture_output=True, text=True, timeout=120)
        assert done.returncode == 0, done.stderr[-2000:]
