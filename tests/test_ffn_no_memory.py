"""The feed-forward C entry points let no exception out: tests/cpp/ffn_no_memory.cpp
calls each while every host allocation fails."""
from __future__ import annotations

import os
import shutil
import subprocess

import pytest

from brovisionml_amd.build import INCLUDE, LIB_FFN, ROOT


def test_entry_points_return_when_host_memory_ends(tmp_path):
    if shutil.which("g++") is None:
        pytest.skip("needs g++")
    exe = str(tmp_path / "ffn_no_memory")
    subprocess.run(["g++", "-std=c++17", "-O1", "-rdynamic", "-I", INCLUDE,
                    os.path.join(ROOT, "tests", "cpp", "ffn_no_memory.cpp"), "-o", exe, "-ldl"],
                   check=True)
    run = subprocess.run([exe, LIB_FFN], stdout=subprocess.PIPE, stderr=subprocess.STDOUT, text=True,
                         timeout=60)
    assert run.returncode == 0, run.stdout
    assert all(int(s) != 0 for s in run.stdout.split()) and len(run.stdout.split()) == 7
