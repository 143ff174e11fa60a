"""Room for the slices of split contractions, on the host (tests/cpp/test_matdeal.cpp)."""
import shutil

import pytest

from test_serving_args import build_and_run


@pytest.mark.skipif(shutil.which("g++") is None, reason="g++ not available")
def test_slices_fit(tmp_path):
    build_and_run(tmp_path, "test_matdeal", "-Werror")
