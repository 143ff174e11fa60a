"""two_terms on the host: for bf16 gradients alone."""
import pytest

import mimir_hip as M
from mimir_hip.device import _num_bwd


def test_types():
    assert _num_bwd("f32", False) == 0 and _num_bwd("bf16", False) == 1
    assert _num_bwd("bf16", True) == 1 | M._lib.NUM_TWO_TERMS
    with pytest.raises(ValueError):
        _num_bwd("f32", True)
    with open(M._lib.HEADER_PATH) as f:
        assert f"#define MIMIR_NUM_TWO_TERMS 0x{M._lib.NUM_TWO_TERMS:x}\n" in f.read()
