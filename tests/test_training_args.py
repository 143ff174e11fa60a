"""The training operators on the host: refusals of every entry point
(tests/cpp/test_training_args.cpp, with a context of a device that is not there),
and the Python forms' own checks."""
import os
import shutil

import pytest

import mimir_hip as M
from test_serving_args import LIB, ROCM, build_and_run


@pytest.mark.skipif(shutil.which("g++") is None or not os.path.isdir(ROCM), reason="g++ or ROCm not available")
def test_refusals(tmp_path):
    build_and_run(tmp_path, "test_training_args", "-D__HIP_PLATFORM_AMD__", f"-I{ROCM}/include",
                  f"-I{os.path.join(M._lib.REPO_ROOT, 'include')}", f"-L{LIB}", "-lmimir_hip", f"-L{ROCM}/lib", "-lamdhip64",
                  f"-Wl,-rpath,{LIB}", f"-Wl,-rpath,{ROCM}/lib")


def test_null_context_is_einval():
    lib = M.load()
    assert lib.mimir_linear_cross_entropy_fwd(None, 0, None, 4, None, 4, None, 0, 4, 4, None, None, None) == M.EINVAL
    assert lib.mimir_linear_cross_entropy_bwd(None, 0, None, 4, None, 4, None, 0, 4, 4, None, None, None, 1.0, None, 4, 0, None,
                                              4, 0) == M.EINVAL
    assert lib.mimir_gated_linear_fwd(None, 0, 0, None, 4, None, None, 4, 0, 4, 4, None, 4, None) == M.EINVAL
    assert lib.mimir_gated_linear_bwd(None, 0, 0, None, 4, None, None, 4, 0, 4, 4, None, None, 4, None, 4, 0, None, None, 4,
                                      0) == M.EINVAL
    assert lib.mimir_grad_norm(None, None, 0, None) == M.EINVAL
    assert lib.mimir_grad_clip(None, None, 0, 1.0, None) == M.EINVAL


def test_names_are_checked():
    with pytest.raises(ValueError):
        M.TensorList([(16, 3, "f16")])
    t = M.TensorList([(16, 3, "f32"), (32, 4, "bf16", 48)])
    assert len(t) == 2 and t.c[0].out == 16 and t.c[1].out == 48 and t.c[1].type == 1
    assert len(M.TensorList([])) == 0
