"""What the experts' operators' kernels take for granted, checked without a GPU."""
from __future__ import annotations

import os
import subprocess


def test_instructions_have_shapes_that_the_tensor_cores_take(tmp_path):
    here = os.path.dirname(os.path.abspath(__file__))
    exe = str(tmp_path / "product_columns")
    subprocess.run(["g++", "-std=c++17", "-I", os.path.join(os.path.dirname(here), "turbinator_c_b200", "csrc"),
                    os.path.join(here, "product_columns.cpp"), "-o", exe], check=True, timeout=120)
    run = subprocess.run([exe], capture_output=True, text=True, timeout=60)
    assert run.returncode == 0, run.stdout
