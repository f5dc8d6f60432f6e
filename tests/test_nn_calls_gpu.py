"""How xgboost.nn's calls go with one another and with the arrays' producers, on
the GPU: host threads, streams; and the widest rows."""
import threading

import pytest
import torch

import nn_reference as R
from xgboost import nn
from xgboost.core import _LIB

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16 = torch.float32, torch.bfloat16


def _refused(calls, times):
    """How many of each call's repetitions the library refused, every call on a host thread of its own."""
    refused, start = [0] * len(calls), threading.Barrier(len(calls))

    def work(i):
        function, args = calls[i]
        start.wait()
        refused[i] = sum(function(args) != 0 for _ in range(times))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return refused


# The library's calls back to back, which leave no time between one thread's and another's: with the shared memory's
# limit set to each launch's own, 72 to 610 of 20000 gradients of the longer list were refused in each of 4 threads.


def test_threads_with_short_and_long_lists():
    g = torch.Generator().manual_seed(1)
    held, calls = [], []
    for n, vocab in ((600, 40), (8192, 3000)) * 2:
        grad, k = torch.randn(n, 16, generator=g).to(DEV), torch.randint(0, vocab, (n,), generator=g).to(DEV)
        out, stream = torch.zeros(vocab, 16, device=DEV), torch.cuda.Stream(DEV)
        held.append((grad, k, out, stream))
        calls.append((_LIB.XGBBEmbeddingBackward, nn._pack_embedding_backward(
            k.data_ptr(), 0, n, 1, 1, 1, 0, 0, 8, 1.0, grad.data_ptr(), out.data_ptr(), 0, stream.cuda_stream, 0, vocab,
            16, 16, 16, 1, 1, 0, 0)))
    torch.cuda.synchronize()
    assert _refused(calls, 20000) == [0] * 4
    for grad, k, out, _ in held:
        R.close(out, R.bag_grad(grad, k[:, None], len(out)))


def test_threads_with_rows_of_different_lengths():
    g = torch.Generator().manual_seed(2)
    held, forward, backward = [], [], []
    for dim in (3080, 4096):
        x, w, stream = torch.randn(2400, dim, generator=g).to(BF16).to(DEV), torch.ones(dim, device=DEV), \
            torch.cuda.Stream(DEV)
        y, dx = torch.zeros_like(x), torch.zeros_like(x)
        _, mean, rstd = nn.layer_norm(x)
        dw, db = torch.zeros(dim, device=DEV), torch.zeros(dim, device=DEV)
        size = nn.layer_norm_backward_workspace(2400, dim)
        space = torch.empty(size, dtype=torch.uint8, device=DEV)
        held.append((x, w, stream, y, dx, mean, rstd, dw, db, space))
        forward.append((_LIB.XGBBLayerNorm, nn._pack_layer_norm(
            x.data_ptr(), w.data_ptr(), 0, y.data_ptr(), 0, 0, stream.cuda_stream, 2400, dim, dim, dim, 4, 1, 0, 1e-5)))
        backward.append((_LIB.XGBBLayerNormBackward, nn._pack_layer_norm_backward(
            x.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), w.data_ptr(), dx.data_ptr(), dw.data_ptr(),
            db.data_ptr(), space.data_ptr(), stream.cuda_stream, size, 2400, dim, dim, dim, dim, 4, 1, 0)))
    torch.cuda.synchronize()
    assert _refused(forward, 800) == [0] * 2 and _refused(backward, 800) == [0] * 2
    for x, w, _, y, dx, mean, rstd, dw, db, _ in held:
        R.close(y, R.norm(x, w)[0])
        for got, want in zip((dx, dw, db), R.norm_grad(x, x, mean, rstd, w)):
            R.close(got, want)


# More tiles of 8 and of 16 lanes than a grid has in y, 65535.
@pytest.mark.parametrize("dim", [524290, 1048561])
def test_rows_of_more_tiles_than_a_grid_has(dim):
    table = torch.arange(3 * dim, device=DEV, dtype=F32).reshape(3, dim) % 1024  # sums below are whole numbers
    tokens = torch.tensor([[0, 2], [1, -1], [2, 2]], device=DEV)
    want = torch.stack((table[0] + table[2], table[1], 2 * table[2]))
    assert torch.equal(nn.embedding(tokens, table, bag=True), want)
    assert torch.equal(nn.embedding_scale_backward(torch.ones(3, 1, device=DEV).expand(3, dim).contiguous(), tokens,
                                                   torch.ones_like(table), bag=True),
                       torch.tensor([[dim, dim], [dim, 0], [dim, dim]], device=DEV, dtype=F32))
    for n in (5, 8200):  # one row's gradient for all tokens
        k = torch.arange(n, device=DEV) % 2
        got = nn.embedding_backward(table[:1].expand(n, dim), k, 3)
        assert torch.equal(got, table[:1] * torch.tensor([[n - n // 2], [n // 2], [0]], device=DEV))


class _Filled:
    """A tensor by its interface alone, as one that is filled on a stream."""

    def __init__(self, t, stream=None):
        self.keep = t
        self.__cuda_array_interface__ = {"data": (t.data_ptr(), False), "shape": tuple(t.shape), "version": 3,
                                         "typestr": "<f4", "strides": None, "stream": stream}


def test_arrays_that_are_filled_on_another_stream():
    x, y, mean, rstd = (torch.zeros(s, device=DEV) for s in ((64, 96), (64, 96), 64, 64))
    filled = torch.randn(64, 96, generator=torch.Generator().manual_seed(3)).to(DEV)
    producer, consumer = torch.cuda.Stream(DEV), torch.cuda.Stream(DEV)

    def call(stream):
        out = [_Filled(t) for t in (y, mean, rstd)]
        nn.layer_norm(_Filled(x, producer.cuda_stream), out=out[0], mean=out[1], rstd=out[2], stream=stream)

    for stream in (0, consumer.cuda_stream, producer.cuda_stream):
        x.zero_()
        y.zero_()
        torch.cuda.synchronize()
        with torch.cuda.stream(producer):
            torch.cuda._sleep(50_000_000)  # 25 to 50 ms
            x.copy_(filled)
        call(stream)
        torch.cuda.synchronize()
        R.close(y, R.norm(filled)[0])
    # In a capture: of a stream that is none of it, nothing is recorded; of one that is, the order.
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=consumer):
        call(consumer.cuda_stream)
    y.zero_()
    graph.replay()
    torch.cuda.synchronize()
    R.close(y, R.norm(filled)[0])
    other = torch.cuda.CUDAGraph()
    with torch.cuda.graph(other, stream=consumer):
        producer.wait_stream(consumer)
        with torch.cuda.stream(producer):
            torch.cuda._sleep(50_000_000)
            x.copy_(filled)
        call(consumer.cuda_stream)
        consumer.wait_stream(producer)
    for _ in range(2):
        x.zero_()
        y.zero_()
        torch.cuda.synchronize()
        other.replay()
        torch.cuda.synchronize()
        R.close(y, R.norm(filled)[0])


def test_a_refused_call_leaves_nothing_to_the_next():
    x, y = torch.randn(3, 8, device=DEV), torch.empty(3, 8, device=DEV)

    def call(device):
        return _LIB.XGBBLayerNorm(nn._pack_layer_norm(x.data_ptr(), 0, 0, y.data_ptr(), 0, 0, 0, 3, 8, 8, 8, 1, 1, device,
                                                      1e-5))

    torch.cuda.synchronize()
    for _ in range(2):
        assert call(99) == -1 and "device" in _LIB.XGBGetLastError().decode()
        assert call(0) == 0, _LIB.XGBGetLastError().decode()
    torch.cuda.synchronize()
    R.close(y, R.norm(x)[0])
