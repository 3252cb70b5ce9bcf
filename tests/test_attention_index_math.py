"""The index arithmetic that the flash-mode attention passes share, compiled from
their own header and run on the host: division by a launch's constants, packing
of query rows into tiles, key ranges."""
import subprocess
from pathlib import Path

from emx_onnx_cgen_b200.build import ARCH, NVCC_FLAGS, nvcc


def test_index_arithmetic_of_the_kernels_header(tmp_path):
    exe = tmp_path / "check"
    src = Path(__file__).with_name("attention_index_check.cu")
    r = subprocess.run([nvcc(), *ARCH, *NVCC_FLAGS, str(src), "-o", str(exe)], capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=120)
    assert (r.returncode, r.stdout) == (0, "ok\n"), r.stdout + r.stderr
