"""The drop-in: the modules that replace the reference's, copied by themselves beside the library, are enough."""

from __future__ import annotations

import os
import shutil
import subprocess
import sys
from pathlib import Path

import pytest

PACKAGE = Path(__file__).resolve().parent.parent / "llm-serving_b200"
HOST = """
import torch
from model.paged import PagedKV, PagedPool
from model.triton_decode import paged_decode, paged_decode_plan
pool = PagedPool(1, 4, 16, 2, 64, dtype=torch.float32, device="cpu", n_head=4)
print("fine", pool.keys[0].shape[0])
"""
DEVICE = HOST + """
pool = PagedPool(1, 4, 16, 2, 64, dtype=torch.float32, device="cuda", n_head=4)
for more in ({}, {"window": 5, "sinks": 1}):
    kv = PagedKV(pool, [[0, 1]], [0], rope_len=20, n_head=4, **more)
    kv.build_mask(next_token=True)
    k = v = torch.ones(1, 2, 1, 64, device="cuda")
    kv.write(0, k, v)
    assert bool((kv.attend(0, torch.ones(1, 4, 1, 64, device="cuda")) == 1).all())
    kv.advance()
"""


def _run(tmp_path, code):
    (tmp_path / "model").mkdir()
    for name in ("_native.py", "triton_decode.py", "paged.py"):
        shutil.copy(PACKAGE / "model" / name, tmp_path / "model" / name)
    (tmp_path / "model" / "__init__.py").write_text("")
    shutil.copy(PACKAGE / "libpaged_decode.so", tmp_path)
    done = subprocess.run([sys.executable, "-c", code], cwd=tmp_path, env={**os.environ, "PYTHONPATH": str(tmp_path)},
                          capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and done.stdout.strip() == "fine 4", done.stderr


def test_three_files_are_enough(tmp_path):
    _run(tmp_path, HOST)


@pytest.mark.gpu
def test_three_files_step(tmp_path):
    _run(tmp_path, DEVICE)
