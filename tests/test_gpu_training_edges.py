"""Calls of the training operators at the edges of what their documentation allows."""
import numpy as np
import pytest

import mimir_hip as M
from _training import Mat

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad,offset", [(0, 0), (3, 1), (8, 8)])
@pytest.mark.parametrize("dtype,dim", [("f32", 3), ("f32", 8), ("bf16", 8), ("bf16", 9)])
def test_no_tokens_no_inputs(ctx, dtype, dim, pad, offset):
    """Without tokens no input is there to be read: weights' gradients are zeros, or what they were."""
    v = 300
    kw = dict(dtype=dtype, ld_x=dim + pad, ld_w=dim + pad)
    mean = ctx.to_device(np.full(2, 5, np.float32))
    ctx.linear_cross_entropy(None, None, None, 0, dim, v, None, None, mean, **kw)
    assert (mean.numpy() == 0).all()
    ctx.linear_cross_entropy(None, None, None, 0, dim, v, None, None, None, **kw)
    for accumulate in (True, False):
        DW, DX = Mat(ctx, np.full((v, dim), 3.0), dtype, pad, offset), Mat(ctx, np.full((2, dim), 3.0), dtype, pad, offset)
        ctx.linear_cross_entropy_bwd(None, None, None, None, None, mean, DX.ptr, DW.ptr, 0, dim, v, ld_dx=DX.ld, ld_dw=DW.ld,
                                     accumulate_w=accumulate, **kw)
        assert (DW.get() == (3 if accumulate else 0)).all() and (DX.get() == 3).all()
        ctx.linear_cross_entropy_bwd(None, None, None, None, None, None, DX.ptr, None, 0, dim, v, ld_dx=DX.ld, **kw)
        assert (DX.get() == 3).all()
        A, B = (Mat(ctx, np.full((v, dim), 3.0), dtype, pad, offset) for _ in range(2))
        ctx.gated_linear_bwd(None, None, None, None, None, DX.ptr, A.ptr, B.ptr, 0, v, dim, dtype=dtype, ld_x=v, ld_w=dim + pad,
                             ld_dx=v, ld_dw=A.ld, accumulate_w=accumulate)
        assert (A.get() == (3 if accumulate else 0)).all() and (B.get() == A.get()).all() and (DX.get() == 3).all()
