"""xgboost.nn without a GPU: the 64-bit forms that the GPU tests hold the
kernels to, against differences; and what the library and the Python layer
refuse before any device is touched."""
import ctypes
import os
import struct
import subprocess

import numpy as np
import pytest
import torch

import nn_reference as R
import xgboost as xgb
from xgboost import nn
from xgboost.core import _LIB


def _difference(f, x, direction, step):
    return (f(x + step * direction) - f(x - step * direction)) / (2 * step)


def test_bag_gradients_are_the_derivatives():
    g = torch.Generator().manual_seed(1)
    tokens = torch.randint(-1, 11, (9, 5), generator=g)
    table, scales = torch.randn(11, 3, generator=g).double(), torch.rand(9, 5, generator=g).double()
    grad = torch.randn(9, 3, generator=g).double()
    d, ds = torch.randn(11, 3, generator=g).double(), torch.randn(9, 5, generator=g).double()
    by_table = _difference(lambda w: (R.bag(tokens, w, 0.7, scales)[0] * grad).sum(), table, d, 1.0)
    by_scale = _difference(lambda s: (R.bag(tokens, table, 0.7, s)[0] * grad).sum(), scales, ds, 1.0)
    # Both are linear: the differences are exact up to rounding.
    assert abs(float(by_table - (R.bag_grad(grad, tokens, 11, 0.7, scales)[0] * d).sum())) < 1e-12
    assert abs(float(by_scale - (R.scale_grad(grad, tokens, table, 0.7)[0] * ds).sum())) < 1e-12


@pytest.mark.parametrize("rows,dim", [(1, 2), (5, 7), (3, 64)])
def test_norm_gradients_are_the_derivatives(rows, dim):
    g = torch.Generator().manual_seed(rows * 100 + dim)
    x, grad, dx = (torch.randn(rows, dim, generator=g).double() for _ in range(3))
    w, b, dw, db = (torch.randn(dim, generator=g).double() for _ in range(4))
    eps = 0.5  # bends the row so gently that the third-order term of the difference is small

    def forward(x, w, b):
        mean = x.mean(1, keepdim=True)
        rstd = 1 / torch.sqrt((x - mean).square().mean(1, keepdim=True) + eps)
        return ((x - mean) * rstd * w + b), mean[:, 0], rstd[:, 0]

    _, mean, rstd = forward(x, w, b)
    got = R.norm_grad(grad, x, mean, rstd, w)
    h = 1e-4  # truncation of order h^2 = 1e-8 of values of order 10
    for at, (wanted, direction) in enumerate(((dx, 0), (dw, 1), (db, 2))):
        args = [x, w, b]

        def loss(v):
            a = list(args)
            a[direction] = v
            return (forward(*a)[0] * grad).sum()

        assert abs(float(_difference(loss, args[direction], wanted, h) - (got[at][0] * wanted).sum())) < 1e-5


class _Fake:
    """A device array by its interface alone; nothing reads its memory."""

    def __init__(self, shape, typestr="<f4", strides=None, ptr=4096):
        self.__cuda_array_interface__ = {"data": (ptr, False), "shape": tuple(shape), "typestr": typestr,
                                         "strides": strides, "version": 3}


F, K = _Fake, lambda *s: _Fake(s, "<i4")  # noqa: E731

REFUSED = [
    (lambda: nn.embedding(np.zeros(3, np.int32), F((4, 2)), out=F((3, 2))), "device array"),
    (lambda: nn.embedding(torch.zeros(3, dtype=torch.int32), F((4, 2)), out=F((3, 2))), "device memory"),
    (lambda: nn.embedding(F((3,)), F((4, 2)), out=F((3, 2))), "int32 or int64"),
    (lambda: nn.embedding(K(3), F((4, 2))), "out must be given"),
    (lambda: nn.embedding(K(3), F((4, 2)), out=F((3, 3))), "out must have the shape"),
    (lambda: nn.embedding(K(3), F((8,)), out=F((3, 2))), "two dimensions"),
    (lambda: nn.embedding(K(3), F((4, 2), strides=(4, 16)), out=F((3, 2))), "contiguous values"),
    (lambda: nn.embedding(K(3), F((4, 2), "<f8"), out=F((3, 2))), "float32, float16 or bfloat16"),
    (lambda: nn.embedding(K(3), F((4, 2)), out=F((3, 2)), token_scale=F((2,))), "token_scale"),
    (lambda: nn.embedding(K(3), F((4, 2)), out=F((3, 2)), token_scale=F((3,), "<f2")), "token_scale"),
    (lambda: nn.embedding(K(3), F((4, 2)), out=F((3, 2)), scale=float("nan")), "scale must be finite"),
    (lambda: nn.embedding(K(3), F((0, 2)), out=F((3, 2))), "vocab"),
    (lambda: nn.embedding(K(3), F((4, 0)), out=F((3, 0))), "dim"),
    (lambda: nn.embedding(K(3), F((4, 2), ptr=4098), out=F((3, 2))), "aligned"),
    (lambda: nn.embedding(K(3), F((4, 2), ptr=0), out=F((3, 2))), "null"),
    (lambda: nn.embedding(K(3), F((4, 2)), out=F((3, 2), strides=(0, 4))), "overlap"),
    (lambda: nn.embedding(K(3, 2, 2), F((4, 2)), out=F((3, 2, 2, 2)), token_scale=F((3, 2, 2), strides=(4, 24, 8))),
     "one stride"),
    (lambda: nn.embedding_backward(F((3, 2)), K(3), 4, out=F((5, 2))), "out must have the shape"),
    (lambda: nn.embedding_backward(F((4, 2)), K(3), 4, out=F((4, 2))), "shape of the lookup"),
    (lambda: nn.embedding_backward(F((3, 2)), K(3), 4, accumulate=True), "accumulate needs out"),
    (lambda: nn.embedding_backward(F((1 << 17, 2)), K(1 << 17), 4, out=F((4, 2), ptr=8192)), "workspace must be given"),
    (lambda: nn.embedding_backward(F((1 << 17, 2)), K(1 << 17), 4, out=F((4, 2), ptr=8192), workspace=F((8,))),
     "workspace must be"),
    (lambda: nn.embedding_backward(F((3, 2)), K(3), 1 << 31, out=F((1 << 31, 2))), "vocab"),
    (lambda: nn.embedding_backward(F((1 << 16, 2)), K(1 << 16, 1 << 16), 4, bag=True, out=F((4, 2))), "tokens"),
    (lambda: nn.embedding_scale_backward(F((3, 2)), K(3), F((4, 3)), out=F((3,))), "shape of the lookup"),
    (lambda: nn.layer_norm(F((3, 4))), "out must be given"),
    (lambda: nn.layer_norm(F((3, 4)), out=F((3, 4)), mean=F((3,)), rstd=F((3,))), "y must not be x"),
    (lambda: nn.layer_norm(F((3, 4)), F((3,)), out=F((3, 4)), mean=F((3,)), rstd=F((3,))), "weight must be 4"),
    (lambda: nn.layer_norm(F((3, 4)), F((4,), "<f2"), out=F((3, 4)), mean=F((3,)), rstd=F((3,))), "x's type"),
    (lambda: nn.layer_norm(F((3, 4)), F((4,)), out=F((3, 4), ptr=8192), mean=F((2,)), rstd=F((3,))), "mean"),
    (lambda: nn.layer_norm(F((3, 4)), eps=-1.0, out=F((3, 4), ptr=8192), mean=F((3,)), rstd=F((3,))), "eps"),
    (lambda: nn.layer_norm(F((3, 0)), out=F((3, 0), ptr=8192), mean=F((3,)), rstd=F((3,))), "dim"),
    (lambda: nn.layer_norm_backward(F((3, 4)), F((3, 5)), F((3,)), F((3,))), "x's shape"),
    (lambda: nn.layer_norm_backward(F((3, 4)), F((3, 4)), F((3,)), F((3,)), out=F((3, 4))), "neither"),
    (lambda: nn.layer_norm_backward(F((3, 4)), F((3, 4)), F((3,)), F((3,)), out=F((3, 4), ptr=8192),
                                    dweight=F((4,))), "need weight"),
    (lambda: nn.layer_norm_backward(F((3, 400)), F((3, 400)), F((3,)), F((3,)), F((400,)), out=F((3, 400), ptr=8192),
                                    dweight=F((400,)), dbias=F((400,))), "workspace must be given"),
]


@pytest.mark.parametrize("at", range(len(REFUSED)))
def test_wrong_arguments_are_refused(at):
    call, needle = REFUSED[at]
    with pytest.raises(xgb.XGBoostError, match=needle):
        call()


def test_library_refuses_before_it_touches_a_device():
    # Types that do not pair up, an index type that is none, a workspace that is missing, not aligned or too small.
    rows = 1 << 17
    need = nn.embedding_backward_workspace(rows, 1, 4, 2)

    def backward(**kw):
        a = dict(grad_type=1, token_type=7, out_type=1, workspace=4096, size=need)
        a.update(kw)
        ret = _LIB.XGBBEmbeddingBackward(nn._pack_embedding_backward(
            8192, 0, rows, 1, 1, 0, 0, 0, a["token_type"], 1.0, 4096, 16384, a["workspace"], 0, a["size"], 4, 2, 2, 2,
            a["grad_type"], a["out_type"], 0, -1))
        return ret, _LIB.XGBGetLastError().decode()

    for kw, needle in ((dict(grad_type=3, out_type=4), "grad's type"), (dict(token_type=1), "int32"),
                       (dict(grad_type=2), "float32"), (dict(workspace=0), "null"),
                       (dict(workspace=4097), "aligned"), (dict(size=need - 1), "smaller")):
        ret, message = backward(**kw)
        assert ret == -1 and needle in message, (kw, message)
    for name in ("Embedding", "EmbeddingBackward", "EmbeddingScaleBackward", "LayerNorm", "LayerNormBackward"):
        assert getattr(_LIB, "XGBB" + name)(None) == -1


def test_argument_structures_are_packed_as_the_header_lays_them_out(tmp_path):
    """The sizes and a few offsets of the packed arguments, against the C compiler's."""
    source = tmp_path / "sizes.c"
    source.write_text('''#include <stdio.h>
#include "xgb_b200.h"
int main(void) {
  printf("%zu %zu %zu %zu %zu %zu", sizeof(XGBBTokens), sizeof(XGBBEmbeddingArgs), sizeof(XGBBEmbeddingBackwardArgs),
         sizeof(XGBBEmbeddingScaleBackwardArgs), sizeof(XGBBLayerNormArgs), sizeof(XGBBLayerNormBackwardArgs));
  return 0;
}''')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    program = str(tmp_path / "sizes")
    subprocess.run(["gcc", "-I", include, str(source), "-o", program], check=True)
    got = [int(v) for v in subprocess.run([program], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [struct.calcsize("@" + nn._TOKENS), struct.calcsize("@" + nn._TOKENS + "PPPQQqqiii4x"),
                   len(nn._pack_embedding_backward(*[0] * 9, 1.0, *[0] * 13)),
                   len(nn._pack_embedding_scale_backward(*[0] * 9, 1.0, *[0] * 11)),
                   len(nn._pack_layer_norm(*[0] * 14, 1.0)), len(nn._pack_layer_norm_backward(*[0] * 19))]


def test_workspace_sizes_are_refused_like_the_calls():
    with pytest.raises(xgb.XGBoostError, match="tokens"):
        nn.embedding_backward_workspace(1 << 20, 1 << 20, 4, 2)
    with pytest.raises(xgb.XGBoostError, match="dim"):
        nn.layer_norm_backward_workspace(3, 0)
    assert _LIB.XGBBLayerNormBackwardWorkspace(3, 4, None) == -1
    size = ctypes.c_size_t()
    assert _LIB.XGBBEmbeddingBackwardWorkspace(1 << 17, 2, 5, 4, ctypes.byref(size)) == 0 and size.value > 0
