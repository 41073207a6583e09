"""What the kernels' compiler flags refuse."""
import importlib.util
import os
import shutil
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.skipif(shutil.which("hipcc") is None, reason="no hipcc")
def test_a_loop_request_without_effect_is_an_error(tmp_path):
    """The loop's trip count is not known and a barrier must not be copied past its end: it is not unrolled, whatever the pragma asks for."""
    spec = importlib.util.spec_from_file_location("_ogl_build_flags", os.path.join(ROOT, "online-gnn-learning_amd", "build.py"))
    b = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(b)
    src = tmp_path / "loop.hip"
    for pragma, ok in (("", True), ("#pragma unroll 4", False)):
        src.write_text("#include <hip/hip_runtime.h>\n__global__ void k(float* x, int n) {\n%s\n  for (int i = threadIdx.x; i < n; i += 7) {\n"
                       "    x[i] += 1.f;\n    __syncthreads();\n  }\n}\n" % pragma)
        got = subprocess.run(["hipcc", *b.FLAGS, "--cuda-device-only", "-c", str(src), "-o", str(tmp_path / "loop.o")], capture_output=True, text=True)
        assert (got.returncode == 0) == ok, got.stderr
        assert ok or "loop not unrolled" in got.stderr
