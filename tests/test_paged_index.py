"""The paged kernels' index arithmetic, walked on the CPU (tests/paged_index_main.cpp), and the
refusals that need no device."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import pytest

from fpga_qwen_b200 import qattn

ROOT = Path(__file__).resolve().parents[1]


def test_split_places_and_eviction_order(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("g++ not available")
    exe = tmp_path / "paged_index_main"
    subprocess.run(["g++", "-std=c++17", "-O2", "-Wall", "-Werror", "-fsanitize=undefined", "-fno-sanitize-recover",
                    str(ROOT / "tests" / "paged_index_main.cpp"), "-o", str(exe)], check=True, capture_output=True, text=True)
    res = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and res.stdout == "ok\n", res.stdout + res.stderr


def test_calls_without_a_context_are_refused():
    lib, pages = qattn.lib(), qattn.Pages(16, 16, 1, 16)
    size = ctypes.c_size_t()
    assert lib.qa_rope_positions(None, 8) == qattn.QA_ERR_INVALID
    assert lib.qa_paged_workspace(None, 1, 1, 1, 0, ctypes.byref(size)) == qattn.QA_ERR_INVALID
    assert lib.qa_paged_append(None, pages, 16, 1, 1, None, 16, 16, 1, 0, 1, 16, 16, 16, 16) == qattn.QA_ERR_INVALID
    assert lib.qa_paged_attn(None, pages, 16, 1, 16, 1, 0, 1, 16, 16, 0, 16, 1 << 30) == qattn.QA_ERR_INVALID
    assert lib.qa_paged_evict(None, pages, 16, 1, 16, 1, 16, 16, 1, 1, 0, 16) == qattn.QA_ERR_INVALID
