"""Forms of xgboost.nn's operators that the grids of test_nn_gpu.py leave out,
against the same 64-bit forms and bounds."""
import pytest
import torch

import nn_reference as R
from xgboost import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(g, *shape, dtype=F32):
    return torch.randn(*shape, generator=g).to(dtype).to(DEV)


# One cluster, parts of warps, of a block, of the stream; rows that registers do not hold.
@pytest.mark.parametrize("rows,dim,a,p", [(40, 64, F32, F32), (9000, 200, BF16, F32), (30, 1000, F16, F16),
                                          (2400, 2048, BF16, BF16), (3, 40000, F32, F32), (0, 300, F32, F32)])
def test_bias_without_a_weight(rows, dim, a, p):
    g = torch.Generator().manual_seed(rows + dim)
    x, grad, b = _randn(g, rows, dim, dtype=a), _randn(g, rows, dim, dtype=a), _randn(g, dim, dtype=p)
    y, mean, rstd = nn.layer_norm(x, None, b)
    R.close(y, R.norm(x, None, b)[0], "y")
    db = torch.full((dim,), 7.0, dtype=p, device=DEV)
    dx, dw, got = nn.layer_norm_backward(grad, x, mean, rstd, dbias=db)
    want = R.norm_grad(grad, x, mean, rstd, None, p)
    assert dw is None and got is db
    R.close(dx, want[0], "dx")
    R.close(db, want[2], "dbias")
    assert nn.layer_norm_backward(grad, x, mean, rstd)[1:] == (None, None)
