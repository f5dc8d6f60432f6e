"""Plain 64-bit forms of xgboost.nn's operators on the CPU, each with the
largest error that float32 sums and one final rounding can have.

A float32 sum of n products, in any order, is within (n + 1) u of the sum of
the products' magnitudes, u = 2^-24; a value rounded to p significant bits is
within 2^-p of itself. The bounds below add these up step by step."""
import numpy as np
import torch

U = 2.0 ** -24
ROUND = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8,
         torch.float64: 2.0 ** -53}
# Half the smallest step of a type (subnormals).
STEP = {torch.float32: 2.0 ** -150, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134,
        torch.float64: 0.0}


def rounded(value, error, dtype):
    """The bound of a result that is within `error` of `value` before it is rounded to dtype."""
    return error + ROUND[dtype] * (value.abs() + error) + STEP[dtype]


def bag(tokens, table, scale=1.0, token_scale=None, dtype=torch.float32):
    """(y, bound) of tokens [rows, per_row]; below 0 missing, past the table NaN."""
    w, vocab = table.double().cpu(), table.shape[0]
    k = tokens.long().cpu()
    f = torch.ones(k.shape, dtype=torch.float64) if token_scale is None else token_scale.double().cpu().expand(k.shape)
    here = (k >= 0) & (k < vocab)
    f = torch.where(here, f, torch.zeros_like(f))
    rows = w[torch.where(here, k, torch.zeros_like(k))]
    rows = torch.where(here[..., None], rows, torch.zeros_like(rows))
    y = (rows * f[..., None]).sum(1) * scale
    size = (rows * f[..., None]).abs().sum(1) * abs(scale)
    y[(k >= vocab).any(1)] = float("nan")
    return y, rounded(y, (k.shape[1] + 4) * U * size, dtype)


def bag_grad(grad, tokens, vocab, scale=1.0, token_scale=None, dtype=torch.float32, onto=None):
    """(dtable, bound), added to `onto` where given."""
    g, k = grad.double().cpu(), tokens.long().cpu()
    f = torch.ones(k.shape, dtype=torch.float64) if token_scale is None else token_scale.double().cpu().expand(k.shape)
    r, t = ((k >= 0) & (k < vocab)).nonzero(as_tuple=True)
    terms = g[r] * f[r, t][:, None] * scale
    zero = torch.zeros(vocab, g.shape[1], dtype=torch.float64)
    y = zero.clone().index_add_(0, k[r, t], terms)
    size = zero.clone().index_add_(0, k[r, t], terms.abs())
    count = torch.zeros(vocab, dtype=torch.float64).index_add_(0, k[r, t], torch.ones(len(r), dtype=torch.float64))
    error = (count[:, None] + 4) * U * size
    if onto is not None:
        old = onto.double().cpu()
        error = error + U * (old.abs() + y.abs())
        y = y + old
    return y, rounded(y, error, dtype)


def scale_grad(grad, tokens, table, scale=1.0):
    g, w, k = grad.double().cpu(), table.double().cpu(), tokens.long().cpu()
    here = (k >= 0) & (k < len(w))
    rows = w[torch.where(here, k, torch.zeros_like(k))]
    y = torch.where(here, torch.einsum("rd,rtd->rt", g, rows), torch.zeros(k.shape, dtype=torch.float64)) * scale
    size = torch.einsum("rd,rtd->rt", g.abs(), rows.abs()) * abs(scale)
    y[k >= len(w)] = float("nan")
    return y, rounded(y, (w.shape[1] + 4) * U * size, torch.float32)


def terms(n):
    """Terms that one float32 chain of a row's sum can have: rows of over 64 values are summed by 16 lanes or more."""
    return n if n <= 64 else n / 16 + 32


def norm(x, weight=None, bias=None, eps=1e-5):
    """((y, bound), (mean, bound), (rstd, bound))."""
    v, n, c = x.double().cpu(), x.shape[1], terms(x.shape[1])
    mean = v.mean(1, keepdim=True)
    rstd = 1.0 / torch.sqrt((v - mean).square().mean(1, keepdim=True) + eps)
    h = (v - mean) * rstd
    e_mean = (c + 3) * U * v.abs().mean(1, keepdim=True)
    # The mean square about a mean that is off by e: var + e^2, and each square 3 roundings.
    e_rstd = rstd * (0.5 * ((c + 8) * U + (e_mean * rstd).square()) + 4 * U)
    w = torch.ones(n, dtype=torch.float64) if weight is None else weight.double().cpu()
    b = torch.zeros(n, dtype=torch.float64) if bias is None else bias.double().cpu()
    y = h * w + b
    e_h = rstd * (e_mean + U * (v - mean).abs()) + h.abs() * (e_rstd / rstd + U)
    e_y = 1.01 * (w.abs() * e_h + 3 * U * ((h * w).abs() + b.abs()))
    return ((y, rounded(y, e_y, x.dtype)), (mean[:, 0], e_mean[:, 0] + 1e-44), (rstd[:, 0], 1.01 * e_rstd[:, 0]))


def norm_grad(grad, x, mean, rstd, weight=None, param=torch.float32):
    """((dx, bound), (dweight, bound), (dbias, bound)) at the given mean and rstd."""
    g0, v, c = grad.double().cpu(), x.double().cpu(), terms(x.shape[1])
    q = rstd.double().cpu()[:, None]
    h = (v - mean.double().cpu()[:, None]) * q
    w = torch.ones(v.shape[1], dtype=torch.float64) if weight is None else weight.double().cpu()
    g = g0 * w
    a, b = g.mean(1, keepdim=True), (g * h).mean(1, keepdim=True)
    dx = q * (g - a - h * b)
    size_a, size_b = g.abs().mean(1, keepdim=True), (g * h).abs().mean(1, keepdim=True)
    e_dx = 1.01 * q * U * ((c + 12) * (size_a + h.abs() * size_b) + 6 * g.abs())
    rows = len(v)
    dw, db = (g0 * h).sum(0), g0.sum(0)
    e_dw, e_db = 1.01 * (rows + 8) * U * (g0 * h).abs().sum(0), 1.01 * (rows + 4) * U * g0.abs().sum(0)
    return (dx, rounded(dx, e_dx, x.dtype)), (dw, rounded(dw, e_dw, param)), (db, rounded(db, e_db, param))


def close(got, want, what=""):
    """Every value of `got` within its bound; NaN exactly where expected."""
    value, bound = want
    assert tuple(got.shape) == tuple(value.shape), (what, got.shape, value.shape)
    v = got.double().cpu()
    nan = torch.isnan(value)
    assert torch.equal(torch.isnan(v), nan), "%s: NaN in other places" % what
    off = torch.where(nan, torch.zeros_like(v), (v - value).abs() - bound)
    assert not off.numel() or float(off.max()) <= 0, "%s: over its bound by %g (at %s)" % (
        what, float(off.max()), np.unravel_index(int(off.argmax()), off.shape))
