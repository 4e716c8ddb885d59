"""Calls at the edges of the paged layer and of the steps under it: many sequences, long windows, several streams, wrong operands.

Two kernels' results for the same step are compared (`agree`).  Each is within P.REL of the exact result in the 2-norm and within 5 P.REL of
a row's largest in an entry: the bounds that tests/k2b_plain.py derives for |K| <= 8.  The keys here are normal, |K| = sqrt(128) = 11.3, so that a score moves by
1.41 u instead of u and the output by sqrt(2 + 2/3) u = 1.63 u = 8.0e-4, still below P.REL = 1.5e-3.  Their difference is at most the sum,
relative to the exact result, which is itself within P.REL of the reference: 2 P.REL / (1 - P.REL), and 10 P.REL / (1 - 5 P.REL) in an entry."""

import ctypes
import math

import pytest
import torch

from bmx_b200 import _lib
from tests import k2b_plain as P
from tests.test_paging_serving import Bench

D = 128


def test_a_shared_step_that_cannot_run_is_refused_before_its_first_launch():
    lib = _lib.lib()
    a = 4096

    def call(g, batch, tail_cap):
        return lib.bmxk_k2b_decode_shared(ctypes.byref(g), a, a, a, a, a, 3, a, batch, 3, 2, a, a, a, 1, 2, 1, a, a, a, 4, a, a, a, tail_cap,
                                          (ctypes.c_uint32 * 4)(), a, 0.1, a, 1 << 40, a, 0, None)

    assert call(_lib.K2bGeom(1, 4, 128, 32, 64, 1, 3, 2, 1), 4000, 192) == _lib.BMXK_ERR_INVALID and b"batch=4000" in lib.bmxk_last_error()
    assert call(_lib.K2bGeom(2, 8, 128, 32, 64, 2, 3, 2, 1), 4, 9000) == _lib.BMXK_ERR_INVALID and b"tail_cap=9000" in lib.bmxk_last_error()


def agree(out, ref):
    out, ref = out.float(), ref.float()
    assert float((out - ref).norm() / ref.norm()) < 2 * P.REL / (1 - P.REL)
    assert float(((out - ref).abs().amax(-1) / ref.abs().amax(-1)).max()) < 10 * P.REL / (1 - 5 * P.REL)


def _layer(K, h_kv, G, n_slots, seqs, W, dev, tokens):
    from bmx_b200.paging import PagedK2bLayer
    from bmx_b200.rope import default_rope_tables

    cos, sin = (t.half() for t in default_rope_tables(500000.0, D, tokens, device=dev))
    geom = K.k2b_geom(h_kv, G, 128, 32, 64, h_kv)
    layer = PagedK2bLayer(geom, n_slots, seqs, W, dev, cos, sin)
    gen = torch.Generator().manual_seed(5)
    layer.set_basis(torch.randn(h_kv * D, 32, generator=gen).to(dev) / math.sqrt(D))
    x = lambda: torch.randn(h_kv, tokens, D, generator=gen).half().to(dev)  # noqa: E731
    layer.add_sequence(0)
    layer.append(0, x(), x(), x())
    return layer, gen


@pytest.mark.gpu
@pytest.mark.parametrize("h_kv,G,W,tokens,batch", [(1, 1, 32, 176, 2200), (2, 1, 32, 300, 2048), (8, 8, 5400, 6800, 12), (8, 4, 5400, 6800, 12)])
def test_many_sequences_and_long_windows(h_kv, G, W, tokens, batch):
    """Whatever the batch and the window, a step over shared prefixes gives what streaming gives; where attending them once is not served
    the layer streams."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from bmx_b200 import kernels as K

    dev = torch.device("cuda:0")
    layer, gen = _layer(K, h_kv, G, 40, batch, W, dev, tokens)
    layer.fork(0, *range(1, batch))
    assert layer.alloc.in_use == (tokens - W) // 128
    q = torch.randn(batch, h_kv * G, D, generator=gen).half().to(dev)
    out = layer.decode(list(range(batch)), q).float()
    served = batch <= K.SHARED_MAX_BATCH and (G <= 4 or W <= 5000)
    assert (layer._plan[4] is not None) == served
    layer.SHARED_MIN_TILES = 1 << 30
    ref = layer.decode(list(range(batch)), q).float()
    assert layer._plan[4] is None
    agree(out, ref)


@pytest.mark.gpu
@pytest.mark.parametrize("kw", [{}, dict(sliding_window=300, sinks=5)])
def test_steps_on_several_streams(kw):
    """Steps that take turns on two streams, with pages coming and going in between, keep nothing that the other stream still uses."""
    b = Bench(slots=40, **kw)
    b.start("a", 0, 900)
    b.fork("a", *range(12))
    b.layer.SHARED_MIN_TILES = 0
    side = torch.cuda.Stream()
    for i in range(6):
        seqs = ["a", *range(12)][i % 3:]
        if i % 2:
            side.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(side):
                b.check(seqs, tol=10 * P.REL)
                plan = b.layer._plan
            torch.cuda.current_stream().wait_stream(side)
            b.check(seqs, tol=10 * P.REL)
            assert b.layer._plan is not plan and b.layer._plan[0] != plan[0]
        else:
            b.check(seqs, tol=10 * P.REL)
        b.feed(i, 1, 140)


@pytest.mark.gpu
def test_the_prompt_kernel_asks_for_its_basis_without_pages():
    """The kernel reads the basis whether pages are held or not."""
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    from bmx_b200 import kernels as K

    dev = torch.device("cuda:0")
    g = K.k2b_geom(2, 4, 128, 32, 64, 2)
    pool = K.K2bPool(g, 1, dev)
    cos = torch.ones(128, D, dtype=torch.float16, device=dev)
    i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device=dev)  # noqa: E731
    q, win = torch.zeros(1, 8, 4, D, dtype=torch.float16, device=dev), torch.zeros(1, 2, 128, D, dtype=torch.float16, device=dev)
    signs, lut = torch.ones(D, device=dev), K.v_lut_tensor(K.GAUSSIAN_CODEBOOK[2], dev)
    for basis in (torch.zeros(2 * D, 16, dtype=torch.float16, device=dev), torch.zeros(2 * D, 32, device=dev)):
        with pytest.raises(AssertionError):
            K.k2b_prefill_sliding(pool, q, 0, basis, i32(1, 1), i32(1), 0, cos, cos, None, win, win, i32(1) + 4, lut, signs, 0.1, i32(4), 10)


@pytest.mark.gpu
def test_windows_longer_than_any_integer_of_the_device():
    """A window or sinks of 2^64 + 1 are longer than the context, not 1."""
    b = Bench(slots=40)
    b.start("a", 0, 900)
    st, K = b.layer, b.K
    q = torch.randn(1, 8, D, generator=b.gen).half().to(b.dev)
    want = st.decode(["a"], q)
    slots = torch.tensor([st.alloc.slots("a")], dtype=torch.int32, device=b.dev)
    n = torch.tensor([slots.shape[1]], dtype=torch.int32, device=b.dev)
    row = st._rows["a"]
    tails = (st.k_win[row: row + 1], st.v_win[row: row + 1], torch.tensor([st._tail["a"]], dtype=torch.int32, device=b.dev))
    ws = K.decode_workspace(st.geom, 1, slots.shape[1], b.dev)
    for window, sinks in ((2 ** 64 + 1, 0), (1, 2 ** 64 + 1)):
        out = K.k2b_decode_sliding(st.pool, q, st.basis_f16, slots, n, slots.shape[1], st.rope_cos, st.rope_sin, *tails, st.v_lut, st.signs, st.sm_scale, ws,
                                   window, sinks)
        agree(out, want)
        out = K.k2b_prefill_sliding(st.pool, q[:, :, None].contiguous(), 899, st.basis_f16, slots, n, slots.shape[1], st.rope_cos, st.rope_sin, None, *tails,
                                    st.v_lut, st.signs, st.sm_scale, ws[:256].view(torch.int32), window, sinks)
        agree(out[:, :, 0], want)


def test_shares_of_a_prefix_leave_room_for_the_pages_behind_it(monkeypatch):
    from bmx_b200 import kernels as K

    monkeypatch.setattr(K, "sm_count", lambda device: 148)
    for ctas, pages in ((8, 64), (8, 256), (12, 40), (32, 128), (4, 5), (300, 9), (1, 1)):
        most = K.split_walk(ctas, pages, "cpu")
        assert K.split_beside(ctas, pages, most, 0, "cpu") == most
        for own in (1, 40, 148, 900, 50000):
            s = K.split_beside(ctas, pages, most, own, "cpu")
            assert 1 <= s <= most
    assert K.split_beside(8, 256, 18, 307, "cpu") * 8 <= 148 - 32
    g = K.k2b_geom(8, 4)
    members, given = [list(range(32))], dict(own_pages=38)
    plan = K.PrefixGroups(g, 32, members, [256], "cpu", **given)
    assert plan.n_split == 18 and plan.split(3) == K.split_beside(8, 256, 18, 304, "cpu") < 18
    assert K.PrefixGroups(g, 32, members, [256], "cpu", own_pages=0).split(3) == 18
    assert K.PrefixGroups(g, 32, members, [256], "cpu").split(0) == 18
    assert K.PrefixGroups(g, 32, members, [256], "cpu", n_split=5).split(3) == 5


@pytest.mark.gpu
@pytest.mark.parametrize("own", [0, 2])
@pytest.mark.parametrize("rope", [True, False])
def test_shared_steps_with_and_without_pages_of_their_own_replayed(own, rope):
    """A step whose sequences hold nothing but prefix and window launches two kernels, one with more pages three: captured, replayed on other
    queries, against the plain form."""
    from bmx_b200 import kernels as K
    from tests.test_shared_prefix_gpu import World, _dev

    w = World(K, _dev(), [(6, [(0, 30), (own, 64), (0, 0), (0, 190)]), (3, [(own, 1), (0, 128)] * 20)], h_kv=3, G=4)
    want = w.decode(K, rope=rope)
    P.assert_attention(want, w.ref)
    q, out = torch.zeros_like(w.q), torch.empty_like(w.q)
    w.decode(K, rope=rope, q=q, out=out)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.decode(K, rope=rope, q=q, out=out)
        w.decode(K, rope=rope, q=q, out=out)
    for _ in range(3):
        q.copy_(w.q)
        out.zero_()
        graph.replay()
        assert torch.equal(out, want)
    K.check_status(w.ws)
