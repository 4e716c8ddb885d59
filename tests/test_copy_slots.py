"""Slots of pools and rows of windows copied to other slots: values, odd sizes and strides, what is refused."""

import ctypes

import pytest
import torch

from bmx_b200 import _lib


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


def _arrays(n, sizes, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.randint(0, 256, (n, s), generator=g, dtype=torch.uint8).to(dev) for s in sizes]


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 700, 3000, 3001])
@pytest.mark.parametrize("sizes", [[16], [16384], [16400, 48], [104448, 65536], [16, 32, 48, 64, 80, 96, 112, 128]])
def test_copies_between_pools_and_inside_one(n, sizes):
    from bmx_b200 import kernels as K

    dev = _dev()
    if n * sum(sizes) > 600e6:
        n = 1500
    src, dst = _arrays(n + 5, sizes, dev), _arrays(2 * n + 3, sizes, dev, 1)
    g = torch.Generator().manual_seed(n)
    a, b = torch.randint(0, n + 5, (n,), generator=g), torch.randperm(2 * n + 3, generator=g)[:n]
    want = [d.clone() for d in dst]
    for s, w in zip(src, want):
        w[b.to(dev)] = s[a.to(dev)]
    K.copy_slots(src, dst, a.tolist(), b.tolist())                       # the same source slot may be named often
    assert all(torch.equal(d, w) for d, w in zip(dst, want))
    half = torch.randperm(2 * n + 2, generator=g)
    a, b = half[:n], half[n:2 * n]
    for w in want:
        w[b.to(dev)] = w[a.to(dev)]
    K.copy_slots(dst, dst, a, b.to(torch.int32))
    assert all(torch.equal(d, w) for d, w in zip(dst, want))


@pytest.mark.gpu
@pytest.mark.parametrize("tail", [1, 7, 128, 200, 256])
def test_parts_of_window_rows_leave_the_rest_alone(tail):
    from bmx_b200 import kernels as K

    dev = _dev()
    g = torch.Generator().manual_seed(tail)
    wins = [torch.randn(5, 3, 256, 128, generator=g).half().to(dev) for _ in range(3)]
    want = [w.clone() for w in wins]
    for w in want:
        w[4, :, :tail] = w[1, :, :tail]
        w[0, :, :tail] = w[1, :, :tail]
    views = [w.flatten(0, 1)[:, :tail] for w in wins]
    K.copy_slots(views, views, [3, 4, 5, 3, 4, 5], [12, 13, 14, 0, 1, 2])
    assert all(torch.equal(a, b) for a, b in zip(wins, want))
    shared = [views[0], views[1], views[0]]                              # one window that serves as two arrays (RTN caches)
    K.copy_slots(shared, shared, [0], [9])
    assert torch.equal(wins[0][3, 0, :tail], wins[0][0, 0, :tail]) and torch.equal(wins[2][3], want[2][3])


@pytest.mark.gpu
def test_another_stream_a_graph_and_lists_that_are_gone():
    from bmx_b200 import kernels as K

    dev = _dev()
    src, dst = _arrays(300, [4096], dev), _arrays(300, [4096], dev, 1)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        K.copy_slots(src, dst, list(range(299)), list(range(1, 300)))
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(dst[0][1:], src[0][:299])
    graph = torch.cuda.CUDAGraph()
    a, b = torch.arange(100, dtype=torch.int32), torch.arange(100, 200, dtype=torch.int32)
    with torch.cuda.graph(graph):
        K.copy_slots(src, dst, a, b)
    a.zero_(), b.zero_()                                                 # the launch holds its own copy
    src[0].random_(0, 256)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(dst[0][100:200], src[0][:100])
    K.copy_slots(src, dst, [], [])


def _call(n_arrays=1, src=(4096,), dst=(1 << 20,), ss=(256,), ds=(256,), nb=(256,), a=(0, 1), b=(2, 3), n=None, n_src=8, n_dst=8):
    k = max(len(src), 1)
    return _lib.lib().bmxk_copy_slots(n_arrays, (ctypes.c_void_p * k)(*src), (ctypes.c_void_p * k)(*dst), (ctypes.c_int64 * k)(*ss), (ctypes.c_int64 * k)(*ds),
                                      (ctypes.c_int64 * k)(*nb), (ctypes.c_int32 * max(1, len(a)))(*a), (ctypes.c_int32 * max(1, len(b)))(*b),
                                      len(a) if n is None else n, n_src, n_dst, None)


@pytest.mark.parametrize("kw,word", [
    (dict(n_arrays=0), b"n_arrays"), (dict(n_arrays=9), b"n_arrays"), (dict(n=-1), b"n=-1"),
    (dict(a=(0, 8)), b"source slot out of range"), (dict(a=(-1, 0)), b"source slot out of range"),
    (dict(b=(2, 8)), b"destination slot out of range"), (dict(b=(-2, 3)), b"destination slot out of range"),
    (dict(b=(3, 3)), b"named twice"), (dict(src=(0,)), b"null"), (dict(src=(4100,)), b"multiples of 16"), (dict(nb=(250,)), b"multiples of 16"),
    (dict(nb=(0,)), b"bytes"), (dict(nb=(512,)), b"bytes"), (dict(ss=(0,)), b"bytes"),
    (dict(dst=(4096,), a=(0, 2), b=(2, 3)), b"both read and written"),            # a copy inside one pool
    (dict(dst=(4096,), a=(1, 1), b=(1, 3)), b"both read and written"),
    (dict(dst=(4096 + 256,)), b"overlaps"), (dict(dst=(4096,), ds=(512,)), b"overlaps"),
    (dict(n_arrays=2, src=(4096, 1 << 22), dst=(1 << 20, 1 << 20), ss=(256,) * 2, ds=(256,) * 2, nb=(256,) * 2), b"destinations 0 and 1 overlap"),
    (dict(n_dst=1 << 31), b"out of range"),
])
def test_refusals_before_any_launch(kw, word):
    assert _call(**kw) == _lib.BMXK_ERR_INVALID
    assert word in _lib.lib().bmxk_last_error(), _lib.lib().bmxk_last_error()


def test_nothing_to_copy_is_no_error_and_the_wrapper_checks_its_lists():
    assert _call(a=(), b=()) == _lib.BMXK_OK
    from bmx_b200 import kernels as K

    x, y = torch.zeros(4, 32, dtype=torch.uint8), torch.zeros(4, 32, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA tensors"):
        K.copy_slots([x], [y], [0], [1])
    for srcs, dsts, a, b in (([x], [y, y], [0], [1]), ([x], [y[:, :16]], [0], [1]), ([x], [y.view(torch.int8)], [0], [1]), ([x], [y], [0, 1], [1]),
                             ([x, x[:2]], [y, y], [0], [1]), ([x], [y], [1 << 40], [0])):
        with pytest.raises(ValueError):
            K.copy_slots(srcs, dsts, a, b)
    with pytest.raises(ValueError, match="one piece"):
        K.copy_slots([torch.zeros(4, 8, 8)[:, :, :4]], [torch.zeros(4, 8, 8)[:, :, :4]], [0], [1])
    for bad in ([0.5], torch.zeros(1, 1, dtype=torch.int64), torch.zeros(1)):
        with pytest.raises(TypeError):
            K.copy_slots([x], [y], bad, [1])
