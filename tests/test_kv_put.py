"""The launches of a reservation in the paged K/V cache, without a GPU."""
import os
import subprocess

from brewference_b200 import build as B

HERE = os.path.dirname(os.path.abspath(__file__))


def test_the_length_is_published_with_the_last_page(tmp_path):
    exe = str(tmp_path / "kv_put_check")
    cuda = os.path.dirname(os.path.dirname(B.nvcc()))
    subprocess.check_call(["g++", "-std=c++17", "-O1", "-I", os.path.join(cuda, "include"), "-I", B.CSRC,
                           os.path.join(HERE, "kv_put_check.cpp"), "-o", exe])
    out = subprocess.run([exe], capture_output=True, text=True)
    assert out.returncode == 0 and out.stdout.strip() == "ok", out.stdout
