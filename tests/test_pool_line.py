"""The arithmetic that cuts attention and selections over the fp16 page pool into items, parts and workspace
(csrc/pool_line.h), on the CPU: tests/native/pool_line.cpp."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")
def test_line_of_work(tmp_path):
    obj, exe = str(tmp_path / "pool_line.o"), str(tmp_path / "pool_line")
    subprocess.run(["hipcc", "-x", "hip", "--offload-arch=gfx950", "--cuda-host-only", "-std=c++17", "-O1", "-w", "-c",
                    os.path.join(HERE, "native", "pool_line.cpp"), "-o", obj], check=True, capture_output=True, timeout=300)
    subprocess.run(["g++", "-no-pie", obj, "-Wl,--unresolved-symbols=ignore-all", "-o", exe], check=True, capture_output=True, timeout=120)
    r = subprocess.run([exe], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0 and r.stdout.startswith("ok"), (r.returncode, r.stdout, r.stderr)
