"""Training operators whose work is cut into pieces and whose contractions are split
at once, with a short last piece, against float64."""
import numpy as np
import pytest

import mimir_hip as M
from test_gpu_gated_linear import hold, make, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("tokens,dim,hidden,piece", [(1024, 256, 5400, 5120), (1100, 136, 3350, 3328), (2100, 64, 1034, 1024)])
def test_gated_products_last_piece(monkeypatch, tokens, dim, hidden, piece, dtype):
    """Weights' gradients: the last piece has fewer tiles and so more splits than the others."""
    monkeypatch.setenv("MIMIR_TUNE", f"matpiece={piece}")
    with M.Context(0) as c:
        a = make(tokens, tokens, dim, hidden, dtype)
        hold(run(c, *a, "silu", dtype), *a, "silu", dtype)
        start = [np.random.default_rng(i).standard_normal(v.shape) for i, v in enumerate(a[:3])]
        hold(run(c, *a, "silu", dtype, start=start), *a, "silu", dtype, start=start)
