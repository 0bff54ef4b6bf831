"""The size of a decode work item is one constant of all decode kernels and of the workspace; a size that an item's pages or a
stage do not fit does not compile."""
import os
import re
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "oxide_infer_b200", "csrc")


def _compiles(tmp_path, chunk):
    src = tmp_path / "chunk.cu"
    src.write_text('#include "kernels.h"\nstatic_assert(oxi::DECODE_CHUNK == %d, "one constant");\n' % chunk)
    flags = [f"-DOXI_DEC_CHUNK={chunk}"] if chunk != 256 else []
    r = subprocess.run([os.environ.get("NVCC", "nvcc"), "-std=c++17", "-gencode", "arch=compute_100a,code=sm_100a", "-I", CSRC, *flags,
                        "-c", str(src), "-o", str(tmp_path / "chunk.o")], capture_output=True, text=True)
    return r.returncode == 0, r.stderr


@pytest.mark.parametrize("chunk,good", [(256, True), (128, True), (512, False), (96, False)])
def test_sizes_of_a_work_item(tmp_path, chunk, good):
    ok, err = _compiles(tmp_path, chunk)
    assert ok == good, err
    assert good or "work item" in err


def test_no_decode_kernel_has_a_size_of_its_own():
    for name in ("decode_attn.cu", "decode_attn_q8.cu"):
        with open(os.path.join(CSRC, name)) as f:
            assert re.findall(r"^constexpr int CHUNK = (\w+);", f.read(), re.M) == ["DECODE_CHUNK"], name
