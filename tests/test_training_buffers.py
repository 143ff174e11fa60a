"""Outputs of the training operators in place of their inputs
(tests/cpp/test_training_buffers.cpp), on the host."""
import os
import shutil

import pytest

from test_serving_args import LIB, ROCM, build_and_run


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(ROCM), reason="g++ or ROCm not available")
def test_buffers_in_place_of_others(tmp_path):
    build_and_run(tmp_path, "test_training_buffers", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include", f"-L{LIB}", "-lmimir_hip",
                  f"-L{ROCM}/lib", "-lamdhip64", f"-Wl,-rpath,{LIB}", f"-Wl,-rpath,{ROCM}/lib")
