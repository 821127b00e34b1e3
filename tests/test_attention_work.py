"""The cut of paged attention into pieces (plain arithmetic shared by host and device)."""
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_every_token_tile_lies_in_one_range(tmp_path):
    exe = tmp_path / "attention_work_test"
    subprocess.run(["g++", "-std=c++17", "-O1", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "gewell_b200" / "csrc"),
                    str(ROOT / "tests" / "cpp" / "attention_work_test.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout + done.stderr
    assert "PASS" in done.stdout


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs g++")
def test_work_that_31_bits_cannot_count_is_seen(tmp_path):
    exe = tmp_path / "attention_bound_test"
    subprocess.run(["g++", "-std=c++17", "-O2", "-fsanitize=undefined", "-fno-sanitize-recover=all", "-I", str(ROOT / "gewell_b200" / "csrc"),
                    str(ROOT / "tests" / "cpp" / "attention_bound_test.cpp"), "-o", str(exe)], check=True)
    done = subprocess.run([str(exe)], capture_output=True, text=True)
    assert done.returncode == 0 and "PASS" in done.stdout, done.stdout + done.stderr
