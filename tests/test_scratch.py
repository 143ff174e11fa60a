"""A context's scratch where it cannot grow (tests/cpp/test_scratch.cpp), on the host."""
import os
import shutil

import pytest

from test_serving_args import LIB, ROCM, build_and_run


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(ROCM), reason="g++ or ROCm not available")
def test_scratch_that_cannot_grow(tmp_path):
    build_and_run(tmp_path, "test_scratch", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include", f"-L{LIB}", "-lmimir_hip",
                  f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{LIB}", f"-Wl,-rpath,{ROCM}/lib")
