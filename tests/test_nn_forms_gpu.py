"""Forms of xgboost.nn's operators that the grids of test_nn_gpu.py leave out,
against the same 64-bit forms and bounds."""
import numpy as np
import pytest
import torch

import nn_reference as R
import xgboost as xgb
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


@pytest.mark.parametrize("a,b", [(F32, F32), (BF16, F32), (F16, F16)])
@pytest.mark.parametrize("scales", [None, (30, 12), (12,), (30, 1)])
def test_autograd_of_bags(a, b, scales):
    g = torch.Generator().manual_seed(5)
    tokens = torch.randint(-1, 90, (30, 12), generator=g).to(DEV)
    table, grad = _randn(g, 90, 20, dtype=a).requires_grad_(), _randn(g, 20, 30, dtype=b).t()  # no contiguous rows
    s = None if scales is None else _randn(g, *scales).requires_grad_()
    y = nn.embedding(tokens, table, scale=0.7, token_scale=s, bag=True, out_dtype=b)
    R.close(y.detach(), R.bag(tokens, table.detach(), 0.7, None if s is None else s.detach(), b))
    y.backward(grad)
    R.close(table.grad, R.bag_grad(grad, tokens, 90, 0.7, None if s is None else s.detach(), a), "dtable")
    if s is not None:
        value, bound = R.scale_grad(grad, tokens, table.detach(), 0.7)
        # A broadcast scale's gradient is torch's float32 sum of at most 30 of these.
        for i in (0, 1):
            if s.numel() < 360 and (2 - i > s.dim() or s.shape[i - 2] == 1):
                error = 30 * R.U * (value.abs() + bound).sum(i, keepdim=True)
                value, bound = value.sum(i, keepdim=True), bound.sum(i, keepdim=True) + error
        R.close(s.grad, (value.reshape(s.shape), bound.reshape(s.shape)), "dscale")


@pytest.mark.parametrize("which", ["x", "w", "b", "xwb", "xw", "xb"])
@pytest.mark.parametrize("a,p", [(F32, F32), (BF16, F32), (F16, F16)])
def test_autograd_of_the_norm(which, a, p):
    g = torch.Generator().manual_seed(6)
    x, w, b = _randn(g, 30, 70, dtype=a), _randn(g, 70, dtype=p), _randn(g, 70, dtype=p)
    grad = _randn(g, 70, 30, dtype=a).t()
    if which == "xb":
        w = None
    for name, t in (("x", x), ("w", w), ("b", b)):
        if name in which:
            t.requires_grad_()
    y, mean, rstd = nn.layer_norm(x, w, b)
    assert y.requires_grad and not mean.requires_grad and not rstd.requires_grad
    y.backward(grad)
    wants = R.norm_grad(grad, x.detach(), mean, rstd, None if w is None else w.detach(), p)
    for name, t, want in zip("xwb", (x, w, b), wants):
        if name in which:
            R.close(t.grad, want, name)
        else:
            assert t is None or t.grad is None


def test_autograd_on_another_stream_and_its_refusals():
    g = torch.Generator().manual_seed(7)
    tokens, table = torch.randint(0, 40, (200, 5), generator=g).to(DEV), _randn(g, 40, 16).requires_grad_()
    w, grad = _randn(g, 16).requires_grad_(), _randn(g, 200, 16)

    def run(stream=None):
        table.grad = w.grad = None
        y = nn.layer_norm(nn.embedding(tokens, table, bag=True, stream=stream), w, stream=stream)[0]
        if stream is not None:
            torch.cuda.current_stream().wait_stream(stream)
        y.backward(grad)
        return y.detach(), table.grad, w.grad

    want, stream = run(), torch.cuda.Stream(DEV)
    torch.cuda.synchronize()
    got = run(stream)
    torch.cuda.synchronize()
    assert all(torch.equal(v, u) for v, u in zip(got, want))
    with torch.no_grad():  # nothing is recorded, and results may be given
        out = torch.empty(200, 16, device=DEV)
        assert nn.embedding(tokens, table, bag=True, out=out) is out
        y = nn.layer_norm(out, w)[0]
        assert torch.equal(y, want[0]) and not y.requires_grad
    with pytest.raises(xgb.XGBoostError, match="automatic differentiation"):
        nn.embedding(tokens, table, bag=True, out=out)
    with pytest.raises(xgb.XGBoostError, match="automatic differentiation"):
        nn.layer_norm(out, w, mean=torch.empty(200, device=DEV))
    x = torch.ones(3, 4, device=DEV, requires_grad=True)
    dx, = torch.autograd.grad(nn.layer_norm(x)[0].sum(), x, create_graph=True)
    with pytest.raises(RuntimeError):  # not differentiated again
        dx.sum().backward()


def test_the_modules_first_example_runs():
    rng = np.random.default_rng(8)
    X = rng.normal(size=(300, 4)).astype(np.float32)
    d = xgb.DMatrix(X, label=X[:, 0])
    g = torch.Generator().manual_seed(8)
    names = {"xgboost": xgb, "torch": torch, "dmatrix": d, "table": _randn(g, 5 * 8, 16), "weight": _randn(g, 16),
             "bias": _randn(g, 16),
             "booster": xgb.train({"tree_method": "hist", "device": "cuda", "max_depth": 3}, d, 5)}
    lines = [line.strip() for line in nn.__doc__.splitlines() if line.startswith("    ")]
    assert len(lines) >= 3
    exec("\n".join(lines), names)
    assert names["vocab"] <= 5 * 8
    R.close(names["h"], R.bag(names["tokens"], names["table"]))
    R.close(names["y"], R.norm(names["h"], names["weight"], names["bias"])[0])


@pytest.mark.parametrize("scales", [(4, 5), (5,), (6, 1, 5), (6, 4, 1), (1,), (4, 1)])
@pytest.mark.parametrize("bag", [False, True])
def test_scales_that_broadcast_over_leading_dimensions(scales, bag):
    g = torch.Generator().manual_seed(9)
    tokens, table = torch.randint(-1, 30, (6, 4, 5), generator=g).to(DEV), _randn(g, 30, 8)
    s, per_row = _randn(g, *scales), 5 if bag else 1
    rows = 120 // per_row
    k, f = tokens.reshape(rows, per_row), s.expand(6, 4, 5).reshape(rows, per_row)
    y = nn.embedding(tokens, table, bag=bag, token_scale=s)
    R.close(y.reshape(rows, 8), R.bag(k, table, 1.0, f))
    grad = _randn(g, *y.shape)
    R.close(nn.embedding_backward(grad, tokens, 30, bag=bag, token_scale=s),
            R.bag_grad(grad.reshape(rows, 8), k, 30, 1.0, f))
    leaf = s.clone().requires_grad_()
    assert torch.equal(nn.embedding(tokens, table, bag=bag, token_scale=leaf).detach(), y)


def _norm_case(g, rows, dim, a, p, has, pad):
    x, grad = (_randn(g, rows, dim + pad, dtype=a)[:, :dim] for _ in range(2))
    w, b = _randn(g, dim, dtype=p) if "w" in has else None, _randn(g, dim, dtype=p) if "b" in has else None
    y = torch.full((rows, dim + pad), 7.0, dtype=a, device=DEV)
    dx = y.clone()
    got, mean, rstd = nn.layer_norm(x, w, b, out=y[:, :dim])
    for value, want, what in zip((got, mean, rstd), R.norm(x, w, b), ("y", "mean", "rstd")):
        R.close(value, want, what)
    db = torch.full((dim,), 7.0, dtype=p, device=DEV) if b is not None else None
    got, dw, db = nn.layer_norm_backward(grad, x, mean, rstd, w, out=dx[:, :dim], dbias=db, bias_grad=b is not None)
    want = R.norm_grad(grad, x, mean, rstd, w, p)
    R.close(got, want[0], "dx")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if w is not None:
        R.close(dw, want[1], "dweight")
    if b is not None:
        R.close(db, want[2], "dbias")
    assert (y[:, dim:] == 7).all() and (dx[:, dim:] == 7).all()  # what lies between the rows stays


# The forms of many rows: a warp's lanes, a warp; streams of a block, of whole and of partly filled ones, of 32 threads
# and of 1024; clusters of two, four and eight; parts of a block where there are few.
@pytest.mark.parametrize("has", ["wb", "w", "b", ""])
@pytest.mark.parametrize("rows,dim,a,p,pad", [
    (2401, 64, BF16, F32, 8), (2403, 512, F32, F32, 4), (2402, 1024, F16, F16, 8), (9473, 1000, BF16, BF16, 8),
    (2369, 4096, BF16, F32, 8), (2371, 3080, F32, F32, 4), (1190, 8192, BF16, F32, 8), (600, 16000, F16, F32, 16),
    (260, 32768, BF16, BF16, 8), (2400, 777, BF16, F32, 3), (40, 1024, BF16, F32, 8)])
def test_many_padded_rows_with_and_without_weight_and_bias(rows, dim, a, p, pad, has):
    _norm_case(torch.Generator().manual_seed(rows + dim), rows, dim, a, p, has, pad)


@pytest.mark.parametrize("has", ["b", ""])
@pytest.mark.parametrize("rows,dim,a", [(5, 64, F32), (3, 1001, F16), (2, 16385, BF16), (1, 40001, F32)])
def test_few_rows_without_a_weight(rows, dim, a, has):
    _norm_case(torch.Generator().manual_seed(rows + dim), rows, dim, a, a, has, 0)


# One block sorts and the others zero absent rows: 12 or 24 entries a thread, rows of plain stores of 4 and 2 bytes and
# of whole copies, tokens of both types, with and without scales.
@pytest.mark.parametrize("n,per_row,vocab,dim,a,b,index,scaled", [
    (9000, 1, 1100003, 33, F32, F32, torch.int32, False), (20000, 4, 1920001, 35, BF16, BF16, torch.int64, True),
    (12288, 3, 33001, 1028, F16, F32, torch.int64, True), (12289, 1, 140003, 256, F32, F32, torch.int64, False)])
def test_gradient_sorted_beside_the_zeros(n, per_row, vocab, dim, a, b, index, scaled):
    assert vocab * dim * b.itemsize >= 128 << 20
    g = torch.Generator().manual_seed(n)
    rows = n // per_row
    tokens = torch.randint(-vocab // 8, vocab, (rows, per_row), generator=g)
    tokens[: rows // 3] %= 5
    tokens, grad = tokens.to(index).to(DEV), _randn(g, rows, dim, dtype=a)
    s = _randn(g, rows, per_row) if scaled else None
    out = torch.full((vocab, dim), 7.0, dtype=b, device=DEV)
    nn.embedding_backward(grad, tokens, vocab, bag=True, scale=0.3, token_scale=s, out=out)
    # The rows that have tokens, by their order, and all others zero.
    present, k = torch.unique(tokens[tokens >= 0].cpu(), return_inverse=True)
    dense = torch.full((rows, per_row), -1, dtype=torch.int64)
    dense[tokens.cpu() >= 0] = k
    R.close(out[present.to(DEV)], R.bag_grad(grad, dense, len(present), 0.3, s, b))
    out[present.to(DEV)] = 0
    assert not out.any()


@pytest.mark.parametrize("n,vocab,dim", [(300, 50, 40), (9000, 70000, 40), (30000, 300, 40), (9000, 1100003, 33),
                                         (9000, 40000, 1024)])
def test_gradient_of_tokens_of_which_none_is_there(n, vocab, dim):
    grad = torch.full((n, dim), float("nan"), device=DEV)
    for nothing in (-1, vocab):
        tokens = torch.full((n,), nothing, dtype=torch.int32, device=DEV)
        out = torch.full((vocab, dim), 7.0, device=DEV)
        assert not nn.embedding_backward(grad, tokens, vocab, out=out).any()
        out.fill_(3.0)
        nn.embedding_backward(grad, tokens, vocab, out=out, accumulate=True)
        assert (out == 3).all()
