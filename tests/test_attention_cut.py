"""The cut of the attention's work, compiled for the host from the header that its kernels use."""
import os
import shutil
import subprocess

import pytest

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_cut_of_the_attention(tmp_path):
    nvcc = shutil.which(os.environ.get("NVCC", "nvcc"))
    if not nvcc:
        pytest.skip("no nvcc")
    exe = tmp_path / "attention_cut"
    subprocess.run([nvcc, "-gencode", "arch=compute_100a,code=sm_100a", "-std=c++17", "-O1", "-diag-suppress", "177",
                    "-I", os.path.join(HERE, "..", "vitni-tensor_b200", "csrc"), os.path.join(HERE, "attention_cut.cu"),
                    "-o", str(exe)], check=True)
    got = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert got.returncode == 0, got.stdout
