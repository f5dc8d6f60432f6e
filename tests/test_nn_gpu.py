"""xgboost.nn on the GPU against plain 64-bit forms, each value within the
bound that float32 sums and one rounding give it (nn_reference.py)."""
import json

import numpy as np
import pytest
import torch

import nn_reference as R
import xgboost as xgb
from xgboost import nn

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
PAIRS = [(F32, F32), (F32, BF16), (F16, F16), (F16, F32), (BF16, BF16), (BF16, F32)]


def _gen(*key):
    g = torch.Generator()
    g.manual_seed(sum(int(v) * 7919 ** i for i, v in enumerate(key)) % (1 << 60))
    return g


def _tokens(g, rows, per_row, vocab, index=torch.int32, missing=0.1, hot=0.3):
    k = torch.randint(0, vocab, (rows, per_row), generator=g)
    k = torch.where(torch.rand(rows, per_row, generator=g) < hot, k % min(3, vocab), k)
    return torch.where(torch.rand(rows, per_row, generator=g) < missing, -1 - k, k).to(index).to(DEV)


def _matrix(g, rows, dim, dtype, pad=0, scale=1.0):
    """Rows of `dim` values, `pad` values apart."""
    return (scale * torch.randn(rows, dim + pad, generator=g)).to(dtype).to(DEV)[:, :dim]


# -- embedding -------------------------------------------------------------------

# rows, per_row, vocab, dim, pad
BAGS = [(1, 1, 1, 1, 0), (1, 2, 3, 1, 0), (5, 3, 7, 2, 0), (3, 8, 9, 4, 0), (33, 9, 40, 8, 0), (17, 31, 100, 16, 0),
        (2, 2000, 500, 33, 0), (1, 4097, 300, 64, 0), (700, 100, 2560, 64, 0), (65, 7, 50, 100, 3), (9, 5, 20, 264, 8),
        (3, 2, 6, 1030, 2), (2, 1, 5, 2048, 0), (4001, 1, 700, 24, 0), (11, 1, 31, 77, 0), (0, 5, 4, 8, 0),
        (4, 0, 4, 8, 0)]


@pytest.mark.parametrize("types", range(len(PAIRS)))
@pytest.mark.parametrize("shape", range(len(BAGS)))
def test_bag(shape, types):
    (rows, per_row, vocab, dim, pad), (a, b) = BAGS[shape], PAIRS[types]
    g = _gen(1, shape, types)
    table = _matrix(g, vocab, dim, a, pad)
    tokens = _tokens(g, rows, per_row, vocab, torch.int64 if types % 2 else torch.int32)
    scales = torch.randn(rows, per_row, generator=g).to(DEV) if shape % 2 else None
    y = nn.embedding(tokens, table, scale=0.7, token_scale=scales, bag=True, out_dtype=b)
    assert y.dtype == b
    R.close(y, R.bag(tokens, table, 0.7, scales, b), "y")


@pytest.mark.parametrize("types", range(len(PAIRS)))
@pytest.mark.parametrize("shape", range(len(BAGS)))
def test_bag_gradients(shape, types):
    (rows, per_row, vocab, dim, pad), (a, b) = BAGS[shape], PAIRS[types]
    g = _gen(2, shape, types)
    grad = _matrix(g, rows, dim, a, pad)
    tokens = _tokens(g, rows, per_row, vocab, torch.int32 if types % 2 else torch.int64)
    tokens.view(-1)[:1] = vocab + 3  # past the table: no gradient
    scales = torch.randn(rows, per_row, generator=g).to(DEV) if shape % 2 == 0 else None
    out = torch.full((vocab, dim + pad), 7.0, dtype=b, device=DEV)[:, :dim]
    got = nn.embedding_backward(grad, tokens, vocab, scale=-1.3, token_scale=scales, bag=True, out=out)
    assert got is out
    R.close(got, R.bag_grad(grad, tokens, vocab, -1.3, scales, b), "dtable")
    onto = out.clone()
    nn.embedding_backward(grad, tokens, vocab, scale=0.4, token_scale=scales, bag=True, out=out, accumulate=True)
    R.close(out, R.bag_grad(grad, tokens, vocab, 0.4, scales, b, onto), "accumulated")
    if pad:  # what lies between the rows stays
        assert torch.equal(torch.as_strided(out, (vocab, pad), (dim + pad, 1), dim).float(),
                           torch.full((vocab, pad), 7.0, device=DEV))
    table = _matrix(g, vocab, dim, b, pad)
    R.close(nn.embedding_scale_backward(grad, tokens, table, scale=0.9, bag=True),
            R.scale_grad(grad, tokens, table, 0.9), "dscale")


# Sorted lists of every size around the sort's tile and the shares, all one token, few tokens, or more table rows than
# two digits of the sort reach.
@pytest.mark.parametrize("rows,vocab,dim", [(8192, 3000, 64), (8192, 70001, 8), (5000, 1 << 21, 2), (255, 1, 8), (256, 2, 8), (257, 1, 3), (4095, 255, 8), (4096, 256, 8),
                                            (4097, 257, 8), (20000, 1, 40), (20011, 2, 33), (50000, 65535, 4),
                                            (50000, 65536, 4), (3000, 70000, 2), (600001, 300, 8), (4200, 70000, 160),
                                            (13000, 17, 300), (24576, 1 << 20, 4), (24577, 900, 24),
                                            (100000, 1 << 17, 12), (250000, 3, 520)])
def test_sorted_gradient(rows, vocab, dim):
    g = _gen(3, rows, vocab, dim)
    grad = _matrix(g, rows, dim, F32)
    tokens = _tokens(g, rows, 1, vocab).reshape(rows)
    R.close(nn.embedding_backward(grad, tokens, vocab), R.bag_grad(grad, tokens[:, None], vocab), "dtable")
    low = _tokens(g, rows, 1, min(vocab, 7)).reshape(rows)  # tokens that lie together
    R.close(nn.embedding_backward(grad, low, vocab), R.bag_grad(grad, low[:, None], vocab), "low tokens")
    one = torch.full((rows,), vocab - 1, dtype=torch.int64, device=DEV)
    R.close(nn.embedding_backward(grad, one, vocab), R.bag_grad(grad, one[:, None], vocab), "one token")


def test_lookup_shapes_and_strides():
    g = _gen(4)
    table = _matrix(g, 50, 24, BF16)
    k3 = _tokens(g, 30, 4, 50).reshape(5, 6, 4)
    y = nn.embedding(k3, table, scale=3.0)
    assert y.shape == (5, 6, 4, 24)
    R.close(y.reshape(-1, 24), R.bag(k3.reshape(-1, 1), table, 3.0, None, BF16))
    y = nn.embedding(k3, table, bag=True)
    assert y.shape == (5, 6, 24)
    R.close(y.reshape(-1, 24), R.bag(k3.reshape(-1, 4), table, 1.0, None, BF16))
    columns = k3.reshape(30, 4).t().contiguous().t()  # tokens of a bag lie apart
    R.close(nn.embedding(columns, table, bag=True), R.bag(columns, table, 1.0, None, BF16))
    every = k3.reshape(-1)[::3]
    R.close(nn.embedding(every, table), R.bag(every[:, None], table, 1.0, None, BF16))
    R.close(nn.embedding(columns[0], table, bag=True)[None], R.bag(columns[:1], table, 1.0, None, BF16))
    # Scales for each tree, and for each row.
    for s in (torch.rand(4, generator=g).to(DEV), torch.rand(30, 1, generator=g).to(DEV)):
        R.close(nn.embedding(columns, table, bag=True, token_scale=s), R.bag(columns, table, 1.0, s, BF16))
        grad = _matrix(g, 30, 24, F32, 8)
        R.close(nn.embedding_backward(grad, columns, 50, bag=True, token_scale=s),
                R.bag_grad(grad, columns, 50, 1.0, s))
    # One row's gradient for all rows (a broadcast), tokens apart.
    grad = _matrix(g, 1, 24, F32).expand(30, 24)
    R.close(nn.embedding_backward(grad, columns, 50, bag=True), R.bag_grad(grad, columns, 50))
    R.close(nn.embedding_scale_backward(grad, columns, table, bag=True), R.scale_grad(grad, columns, table))
    # Rows at odd addresses.
    odd = torch.randn(50 * 24 + 1, generator=g).to(F16).to(DEV)[1:].reshape(50, 24)
    R.close(nn.embedding(columns, odd, bag=True), R.bag(columns, odd, 1.0, None, F16))


def test_missing_tokens_and_tokens_past_the_table():
    table = torch.full((4, 8), float("inf"), device=DEV)
    table[2] = 1.5
    tokens = torch.tensor([[2, -1, 2], [-1, -5, -(1 << 40)], [2, 4, -1], [1 << 40, 2, 2], [2, 2, 2]], device=DEV)
    scales = torch.full((5, 3), float("nan"), device=DEV)
    scales[tokens >= 0] = 2.0
    y = nn.embedding(tokens, table, bag=True, token_scale=scales)
    want = torch.tensor([6.0, 0.0, float("nan"), float("nan"), 9.0], device=DEV)[:, None].expand(5, 8)
    assert torch.equal(torch.isnan(y), torch.isnan(want)) and torch.equal(y.nan_to_num(-1), want.nan_to_num(-1))
    flat = nn.embedding(tokens.reshape(-1), table, token_scale=scales.reshape(-1)).reshape(5, 3, 8)
    assert torch.equal(flat[0, :, 0], torch.tensor([3.0, 0.0, 3.0], device=DEV))
    assert torch.isnan(flat[2, 1]).all() and torch.isnan(flat[3, 0]).all() and not flat[1].any()
    # NaN gradients of rows with no token, and scales of missing tokens, reach nothing.
    grad = torch.ones(5, 8, device=DEV)
    grad[1] = float("nan")
    dt = nn.embedding_backward(grad, tokens, 4, bag=True, token_scale=scales)
    assert torch.equal(dt[2], torch.full((8,), 2.0 * 8, device=DEV)) and not dt[[0, 1, 3]].any()
    ds = nn.embedding_scale_backward(torch.ones(5, 8, device=DEV), tokens, table, bag=True)
    assert torch.equal(ds.nan_to_num(-1), torch.tensor(
        [[12.0, 0, 12], [0, 0, 0], [12, -1, 0], [-1, 12, 12], [12, 12, 12]], device=DEV))


def test_gradients_against_differences():
    """Sums are linear in the table and in the scales: the loss's difference over a whole step is the gradient's
    product with the step, up to rounding."""
    g = _gen(5)
    tokens, table = _tokens(g, 40, 12, 90), _matrix(g, 90, 20, F32)
    scales, grad = torch.rand(40, 12, generator=g).to(DEV), _matrix(g, 40, 20, F32)
    step, by = _matrix(g, 90, 20, F32), torch.randn(40, 12, generator=g).to(DEV)

    def loss(w, s):
        y = nn.embedding(tokens, w, bag=True, token_scale=s)
        bound = R.bag(tokens, w, 1.0, s)[1]
        return (y.double() * grad.double()).sum().item(), (bound * grad.double().cpu().abs()).sum().item()

    dt, ds = nn.embedding_backward(grad, tokens, 90, bag=True, token_scale=scales), nn.embedding_scale_backward(
        grad, tokens, table, bag=True)
    # Adding the step rounds each value of the table or the scales once more: 2 u of the sums' magnitude.
    size = 4 * R.U * (R.bag(tokens, table.abs() + step.abs(), 1.0, scales + by.abs())[0] *
                      grad.double().cpu().abs()).sum().item()
    for (lo, hi), d, way, want in (((loss(table, scales), loss(table + step, scales)), dt, step,
                                    R.bag_grad(grad, tokens, 90, 1.0, scales)),
                                   ((loss(table, scales), loss(table, scales + by)), ds, by,
                                    R.scale_grad(grad, tokens, table))):
        bound = lo[1] + hi[1] + size + (want[1] * way.double().cpu().abs()).sum().item()
        assert abs(hi[0] - lo[0] - (d.double() * way.double()).sum().item()) <= bound


# -- layer norm ------------------------------------------------------------------

NORMS = [(1, 1, 0), (3, 2, 0), (5, 7, 0), (300, 8, 0), (77, 33, 0), (509, 64, 0), (64, 96, 32), (40, 100, 0),
         (33, 256, 0), (19, 257, 3), (130, 784, 0), (9, 1000, 8), (7, 1024, 0), (5, 2048, 0), (9, 3000, 0),
         (3, 4096, 0), (2, 5001, 0), (3, 8192, 0), (2, 8200, 0), (3, 16384, 0), (2, 16385, 0), (1, 40000, 0),
         (2, 70001, 0), (2000, 24, 0), (0, 16, 0)]


@pytest.mark.parametrize("types", range(4))
@pytest.mark.parametrize("shape", range(len(NORMS)))
def test_layer_norm_and_its_gradient(shape, types):
    rows, dim, pad = NORMS[shape]
    a, p = [(F32, F32), (F16, F16), (BF16, BF16), (BF16, F32)][types]
    g = _gen(6, shape, types)
    x = (torch.randn(rows, dim + pad, generator=g) * 2 + 1).to(a).to(DEV)[:, :dim]
    w, b = (1 + 0.2 * torch.randn(dim, generator=g)).to(p).to(DEV), torch.randn(dim, generator=g).to(p).to(DEV)
    which = shape % 3  # with weight and bias, weight alone, neither
    if which == 1:
        b = None
    elif which == 2:
        w = b = None
    y, mean, rstd = nn.layer_norm(x, w, b, eps=1e-5)
    for got, want, what in zip((y, mean, rstd), R.norm(x, w, b, 1e-5), ("y", "mean", "rstd")):
        R.close(got, want, what)
    grad = _matrix(g, rows, dim, a, pad)
    out = torch.full((rows, dim + pad), 7.0, dtype=a, device=DEV)[:, :dim]
    dx, dw, db = nn.layer_norm_backward(grad, x, mean, rstd, w, bias_grad=b is not None, out=out)
    wants = R.norm_grad(grad, x, mean, rstd, w, p)
    R.close(dx, wants[0], "dx")
    assert (dw is None) == (w is None) and (db is None) == (b is None)
    if dw is not None:
        R.close(dw, wants[1], "dweight")
    if db is not None:
        R.close(db, wants[2], "dbias")
    if pad:
        assert torch.equal(torch.as_strided(out, (rows, pad), (dim + pad, 1), dim).float(),
                           torch.full((rows, pad), 7.0, device=DEV))


# Rows enough that blocks take many each, of 64 lanes' values or fewer, of whole and of partly filled blocks.
@pytest.mark.parametrize("rows,dim,a,p", [
    (5000, 64, F32, F32), (3001, 200, F32, F32), (300, 64, BF16, F32), (2000, 40, F32, F32), (16000, 8, F16, F16), (1203, 1024, F32, F32), (2500, 3, F32, F32), (700, 2048, F32, F32),
    (601, 777, F32, F32), (9001, 512, BF16, F32), (5003, 1000, F16, F16), (2501, 2048, BF16, BF16),
    (2500, 1996, F32, F32), (2401, 4096, F32, F32), (2400, 3080, F16, F32), (2399, 4096, BF16, F32),
    (2403, 8192, BF16, F32), (2402, 8000, F32, F32), (2370, 16384, BF16, BF16), (2369, 16000, F16, F32),
    (300, 9001, F32, F32), (300, 20000, BF16, F32), (260, 32768, F32, F32), (2000, 1001, BF16, BF16),
    (500, 5001, F16, F32), (3000, 33, BF16, F32)])
def test_many_rows(rows, dim, a, p):
    g = _gen(7, rows, dim)
    x = (torch.randn(rows, dim, generator=g) * 2 + 30 * torch.randn(rows, 1, generator=g)).to(a).to(DEV)
    grad, w, b = _matrix(g, rows, dim, a), _matrix(g, 1, dim, p)[0], _matrix(g, 1, dim, p)[0]
    y, mean, rstd = nn.layer_norm(x, w, b)
    for got, want, what in zip((y, mean, rstd), R.norm(x, w, b), ("y", "mean", "rstd")):
        R.close(got, want, what)
    dx, dw, db = nn.layer_norm_backward(grad, x, mean, rstd, w)
    wants = R.norm_grad(grad, x, mean, rstd, w, p)
    for got, want, what in zip((dx, dw, db), wants, ("dx", "dweight", "dbias")):
        R.close(got, want, what)


def test_norm_strides_and_odd_addresses():
    g = _gen(8)
    x = torch.randn(3, 5, 48, generator=g).to(DEV)
    y, mean, rstd = nn.layer_norm(x)
    assert y.shape == x.shape and mean.shape == rstd.shape == (3, 5)
    R.close(y.reshape(15, 48), R.norm(x.reshape(15, 48))[0])
    flat = torch.randn(20 * 48 + 1, generator=g).to(BF16).to(DEV)[1:].reshape(20, 48)
    y, mean, rstd = nn.layer_norm(flat)
    R.close(y, R.norm(flat)[0])
    R.close(nn.layer_norm_backward(flat, flat, mean, rstd)[0], R.norm_grad(flat, flat, mean, rstd)[0])
    # The three matrices and the weight aligned differently.
    w = torch.randn(49, generator=g).to(DEV)[1:]
    even = torch.randn(20, 48, generator=g).to(BF16).to(DEV)
    R.close(nn.layer_norm(even, w)[0], R.norm(even, w)[0])
    out = torch.empty(20 * 48 + 1, dtype=BF16, device=DEV)[1:].reshape(20, 48)
    dx, dw, db = nn.layer_norm_backward(flat, even, mean, rstd, w, out=out)
    for got, want in zip((dx, dw, db), R.norm_grad(flat, even, mean, rstd, w)):
        R.close(got, want)
    one = torch.randn(48, generator=g).to(DEV)
    y, mean, rstd = nn.layer_norm(one)
    assert y.shape == (48,) and mean.shape == ()
    R.close(y[None], R.norm(one[None])[0])
    same = torch.randn(1, 48, generator=g).to(DEV).expand(6, 48)  # one row for all
    R.close(nn.layer_norm(same)[0], R.norm(same)[0])


def test_norm_of_constant_far_off_and_broken_rows():
    x = torch.zeros(6, 96, device=DEV)
    x[0] = 5.0
    x[1] = 1e4 + torch.randn(96, generator=_gen(9)).to(DEV)
    x[2, 3] = float("nan")
    x[3, 4] = float("inf")
    x[4] = 1e-30 * torch.arange(96, device=DEV)
    y, mean, rstd = nn.layer_norm(x, eps=1e-5)
    assert not y[0].any() and not y[5].any()
    assert torch.isnan(y[2]).all() and torch.isnan(y[3]).all()
    good = [0, 1, 4, 5]
    for got, want, what in zip((y, mean, rstd), R.norm(x[good]), ("y", "mean", "rstd")):
        R.close(got[good], want, what)
    # A broken row's gradient stays its own; the weight's gradient over all rows is NaN.
    w = torch.ones(96, device=DEV)
    dx, dw, _ = nn.layer_norm_backward(torch.ones_like(x), x, mean, rstd, w)
    assert torch.isnan(dx[2]).all() and torch.isfinite(dx[good]).all() and torch.isnan(dw).all()


def test_norm_gradient_against_differences():
    g = _gen(10)
    x, way, grad = _matrix(g, 30, 70, F32), _matrix(g, 30, 70, F32), _matrix(g, 30, 70, F32)
    w, b = _matrix(g, 1, 70, F32)[0], _matrix(g, 1, 70, F32)[0]
    h = 2.0 ** -6
    lo, hi = x - h * way, x + h * way
    c = grad.double().cpu()

    def loss(v):
        y = nn.layer_norm(v, w, b)[0]
        value, bound = R.norm(v, w, b)[0]
        return (y.double().cpu() * c).sum().item(), (value * c).sum().item(), (bound * c.abs()).sum().item()

    a, z = loss(lo), loss(hi)
    _, mean, rstd = nn.layer_norm(x, w, b)
    dx = nn.layer_norm_backward(grad, x, mean, rstd, w)[0]
    value, bound = R.norm_grad(grad, x, mean, rstd, w)[0]
    d = way.double().cpu()
    truncation = abs((z[1] - a[1]) / (2 * h) - (value * d).sum().item())  # of the 64-bit form's difference
    allowed = truncation + (a[2] + z[2]) / (2 * h) + (bound * d.abs()).sum().item()
    assert abs((z[0] - a[0]) / (2 * h) - (dx.double().cpu() * d).sum().item()) <= allowed


# -- streams, repeats, other arrays, capture ----------------------------------------------


def _everything(g, stream=None, **given):
    rows, per_row, vocab, dim = 3000, 20, 640, 40
    if not given:
        given.update(tokens=_tokens(g, rows, per_row, vocab), table=_matrix(g, vocab, dim, BF16),
                     scales=torch.rand(rows, per_row, generator=g).to(DEV), grad=_matrix(g, rows, dim, F32),
                     w=_matrix(g, 1, dim, F32)[0], b=_matrix(g, 1, dim, F32)[0])
    v = given
    h = nn.embedding(v["tokens"], v["table"], bag=True, token_scale=v["scales"], out_dtype=F32, stream=stream)
    y, mean, rstd = nn.layer_norm(h, v["w"], v["b"], stream=stream)
    dh, dw, db = nn.layer_norm_backward(v["grad"], h, mean, rstd, v["w"], stream=stream)
    dt = nn.embedding_backward(dh, v["tokens"], vocab, bag=True, token_scale=v["scales"], stream=stream)
    ds = nn.embedding_scale_backward(dh, v["tokens"], v["table"], bag=True, stream=stream)
    return given, (h, y, mean, rstd, dh, dw, db, dt, ds)


def test_equal_inputs_give_equal_bits_on_any_stream():
    given, first = _everything(_gen(11))
    torch.cuda.synchronize()
    other = torch.cuda.Stream(DEV)
    other.wait_stream(torch.cuda.current_stream())
    for stream in (None, other, other.cuda_stream, 0):
        _, again = _everything(None, stream, **given)
        torch.cuda.synchronize()
        for a, b in zip(first, again):
            assert torch.equal(a, b)
    with torch.cuda.stream(other):
        _, again = _everything(None, **given)
    other.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_capture_and_replay():
    given, first = _everything(_gen(12))
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        _, held = _everything(None, **given)
    for t in held:
        t.zero_()
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(first, held))


class _Plain:
    """A device array by its interface alone."""

    def __init__(self, t):
        self.keep = t
        self.__cuda_array_interface__ = {
            "data": (t.data_ptr(), False), "shape": tuple(t.shape), "version": 3,
            "typestr": {F32: "<f4", F16: "<f2", torch.int32: "<i4", torch.uint8: "|u1"}[t.dtype],
            "strides": tuple(s * t.element_size() for s in t.stride())}


def test_arrays_by_their_interface():
    g = _gen(13)
    tokens, table = _tokens(g, 50, 6, 30), _matrix(g, 30, 12, F32, 4)
    out, dt = torch.empty(50, 12, device=DEV), torch.empty(30, 12, device=DEV)
    y, mean, rstd = torch.empty(50, 12, device=DEV), torch.empty(50, device=DEV), torch.empty(50, device=DEV)
    torch.cuda.synchronize()
    P = _Plain
    nn.embedding(P(tokens), P(table), bag=True, out=P(out))
    nn.layer_norm(P(out), out=P(y), mean=P(mean), rstd=P(rstd), stream=0)
    space = torch.empty(nn.embedding_backward_workspace(50, 6, 30, 12), dtype=torch.uint8, device=DEV)
    nn.embedding_backward(P(out), P(tokens), 30, bag=True, out=P(dt), workspace=P(space))
    torch.cuda.synchronize()
    R.close(out, R.bag(tokens, table))
    R.close(y, R.norm(out)[0])
    R.close(dt, R.bag_grad(out, tokens, 30))


def test_offsets_past_32_bits():
    """A table, tokens' outputs and rows whose last value lies past 2^32 values."""
    dim, vocab = 4096, (1 << 20) + 3
    table = torch.zeros(vocab, dim, dtype=F16, device=DEV)
    table[-1] = 1.0
    table[0] = 2.0
    rows = (1 << 20) + 2
    tokens = torch.full((rows,), -1, dtype=torch.int32, device=DEV)
    tokens[0], tokens[-1] = vocab - 1, 0
    y = nn.embedding(tokens, table, scale=3.0)
    assert (y[0] == 3).all() and (y[-1] == 6).all() and not y[1:-1].any()
    bags = nn.embedding(tokens[-2:, None].expand(2, 3), table, bag=True)
    assert (bags[1] == 6).all() and not bags[0].any()
    y[-1] = torch.arange(dim, device=DEV).to(F16) / 64
    del table
    _, mean, rstd = nn.layer_norm(y)
    R.close(mean[-1:], R.norm(y[-1:])[1])
    dx, dw, db = nn.layer_norm_backward(y, y, mean, rstd, torch.ones(dim, device=DEV))
    R.close(dx[-1:], R.norm_grad(y[-1:], y[-1:], mean[-1:], rstd[-1:])[0])
    del dx
    dt = nn.embedding_backward(y, tokens, vocab)
    assert torch.equal(dt[0], y[-1]) and torch.equal(dt[-1], y[0]) and not dt[1:-1].any()


def test_refusals_of_tensors():
    k, w = torch.zeros(3, dtype=torch.int32, device=DEV), torch.zeros(4, 8, device=DEV)
    for call, needle in ((lambda: nn.embedding(k, w.double()), "float32"),
                         (lambda: nn.embedding(k, w.half(), out_dtype=BF16), "table's type"),
                         (lambda: nn.embedding(k, w.t()), "contiguous"),
                         (lambda: nn.embedding(k, w[0]), "two dimensions"),
                         (lambda: nn.embedding(k.float(), w), "int32 or int64"),
                         (lambda: nn.embedding(k[0], w, bag=True), "at least one dimension"),
                         (lambda: nn.embedding_backward(w, k, 9), "shape of the lookup"),
                         (lambda: nn.embedding_backward(w[:3], k, 1 << 31), "vocab"),
                         (lambda: nn.embedding_backward(w[:3].half(), k, 9, out_dtype=BF16), "grad's type"),
                         (lambda: nn.embedding_scale_backward(w[:3], k, w[:, :4]), "shape of the lookup"),
                         (lambda: nn.layer_norm_backward(w, w.half(), k, k, w[0]), "x's shape and type"),
                         (lambda: nn.layer_norm_backward(w, w, w[0], w[0], w[0]), "one value a row"),
                         (lambda: nn.layer_norm(w, w[0].half()), "x's type"),
                         (lambda: nn.embedding(k.cpu(), w), "device memory"),
                         (lambda: nn.embedding(k, w, token_scale=torch.zeros(2, device=DEV)), "broadcast"),
                         (lambda: nn.embedding(k, w, out=w[:3]), "out must not be"),
                         (lambda: nn.layer_norm(w, out=w), "must not be"),
                         (lambda: nn.layer_norm(w, torch.zeros(8, device=DEV), torch.zeros(7, device=DEV)), "bias")):
        with pytest.raises(xgb.XGBoostError, match=needle):
            call()


def test_leaf_tokens_number_the_leaves():
    rng = np.random.default_rng(5)
    X = rng.normal(size=(800, 6)).astype(np.float32)
    y = rng.integers(0, 3, 800).astype(np.float32)
    d = xgb.DMatrix(X, label=y)
    b = xgb.train({"objective": "multi:softprob", "num_class": 3, "max_depth": 3, "tree_method": "hist",
                   "device": "cuda"}, d, 4)
    tokens, vocab = nn.leaf_tokens(b, d)
    nodes = b.predict(d, pred_leaf=True)
    assert tokens.shape == nodes.shape == (800, 12) and tokens.dtype == np.int32
    assert 0 <= tokens.min() and tokens.max() < vocab
    for t in range(12):  # one number for each leaf, the trees' numbers apart
        pairs = {(int(a), int(c)) for a, c in zip(nodes[:, t], tokens[:, t])}
        assert len(pairs) == len({a for a, _ in pairs}) == len({c for _, c in pairs})
        if t:
            assert tokens[:, t].min() > tokens[:, t - 1].max()
    part, few = nn.leaf_tokens(b, d, iteration_range=(1, 3))
    assert part.shape == (800, 6) and few < vocab
    np.testing.assert_array_equal(part - part.min(0), (tokens - tokens.min(0))[:, 3:9])
    # The margins are the bags of the leaves' values, a column for each class.
    trees = json.loads(bytes(b.save_raw("json")).decode())["learner"]["gradient_booster"]["model"]["trees"]
    table = np.zeros((vocab, 3), np.float32)
    at = 0
    for t, tree in enumerate(trees):
        leaf = np.flatnonzero(np.asarray(tree["left_children"]) < 0)
        table[at:at + len(leaf), t % 3] = np.asarray(tree["split_conditions"], np.float32)[leaf]
        at += len(leaf)
    table, k = torch.from_numpy(table).to(DEV), torch.from_numpy(tokens).to(DEV)
    sums = nn.embedding(k, table, bag=True)
    rest = b.predict(d, output_margin=True).astype(np.float64) - sums.double().cpu().numpy()
    # The intercept is left: both sums of 12 values and an intercept of size 1 at most are within 16 u of their size.
    size = R.bag(k, table.abs())[0].max().item() + 1.0
    assert np.abs(rest - rest[0]).max() <= 4 * 16 * R.U * size


def test_a_head_on_leaves_learns():
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "leaf_embedding.py")
    spec = importlib.util.spec_from_file_location("leaf_embedding", path)
    example = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(example)
    _, first, last = example.main(rows=6000, cols=8, trees=10, depth=4, dim=16, steps=40)
    assert abs(first - np.log(2)) < 1e-3  # a head of zeros
    assert last < first - 0.05
    # Its gradients are those that torch derives for the same formula in 64 bits.
    g = _gen(14)
    head = example.Head(90, 12, 24, torch.device(DEV))
    tokens, labels = _tokens(g, 300, 12, 90), (torch.rand(300, generator=g) < 0.5).float().to(DEV)
    head.v = _matrix(g, 1, 24, F32)[0]
    margin, saved = head.forward(tokens)
    d_margin = torch.sigmoid(margin) - labels
    grads = head.backward(d_margin, saved)
    leaves = [t.double().requires_grad_() for t in (head.table, head.weight, head.bias, head.v, head.c)]
    table, weight, bias, v, c = leaves
    h = (table[tokens.clamp(min=0).long()] * (tokens >= 0)[..., None]).sum(1) * head.scale
    y = torch.nn.functional.layer_norm(h, (24,), weight, bias)
    ((y @ v + c) * d_margin.double()).sum().backward()
    for got, leaf in zip(grads, leaves):
        want = leaf.grad
        # Sums of up to 300 x 24 float32 terms: 2^-24 of their size for each, and their size is at most that
        # many times the largest; held here to 1e-4 of the largest, a thousand roundings.
        assert float((got.double() - want).abs().max()) <= 1e-4 * float(want.abs().max())


@pytest.mark.parametrize("rows,per_row,vocab,dim", [(9000, 1, 300, 40), (30000, 1, 70000, 8), (700, 100, 2560, 64),
                                                    (16000, 1, 40000, 1024)])
def test_what_a_workspace_held_does_not_matter(rows, per_row, vocab, dim):
    """Back to back and replayed, on workspaces full of what never was an index."""
    g = _gen(15, rows, vocab)
    grad, tokens = _matrix(g, rows, dim, F32), _tokens(g, rows, per_row, vocab)
    want = nn.embedding_backward(grad, tokens, vocab, bag=True)
    R.close(want, R.bag_grad(grad, tokens, vocab))
    space = torch.empty(nn.embedding_backward_workspace(rows, per_row, vocab, dim), dtype=torch.uint8, device=DEV)
    out = torch.empty_like(want)
    x, w = _matrix(g, 3000, 600, F32), torch.ones(600, device=DEV)
    _, mean, rstd = nn.layer_norm(x, w)
    first = nn.layer_norm_backward(x, x * 2, mean, rstd, w)
    twice = x * 2
    parts = torch.empty(nn.layer_norm_backward_workspace(3000, 600), dtype=torch.uint8, device=DEV)

    def both():
        space.fill_(0xff)
        parts.fill_(0xff)
        nn.embedding_backward(grad, tokens, vocab, bag=True, out=out, workspace=space)
        return nn.layer_norm_backward(x, twice, mean, rstd, w, workspace=parts)

    for _ in range(3):
        again = both()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(again, first))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        again = both()
    for _ in range(3):
        out.fill_(7.0)
        for a in again:
            a.fill_(7.0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and all(torch.equal(a, b) for a, b in zip(again, first))
