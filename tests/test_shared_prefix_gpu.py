"""A decode step of sequences that share prefixes, against a plain float64 form and against the step that streams every sequence."""

import ctypes
import math

import pytest
import torch

from bmx_b200 import _lib
from tests import k2b_plain as P

D = 128


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


class World:
    """groups: (prefix pages, [(own pages, window tokens) of each member]); alone: (pages, window tokens) of sequences in no group.
    Batch rows are shuffled; what lies behind a window's end is NaN."""

    def __init__(self, K, dev, groups, alone=(), h_kv=2, G=4, rank=32, group=64, per_head=True, cap=192, seed=3, n_split=None):
        self.geom = g = K.k2b_geom(h_kv, G, 128, rank, group, h_kv if per_head else 1)
        gen = torch.Generator().manual_seed(seed)
        seqs = [(i, P0, own, tail) for i, (P0, members) in enumerate(groups) for own, tail in members] + [(-1, 0, own, tail) for own, tail in alone]
        seqs = [seqs[i] for i in torch.randperm(len(seqs), generator=gen)]
        B = len(seqs)
        n_slots = 1 + sum(P0 for P0, _ in groups) + sum(own for _, _, own, _ in seqs)
        self.pool, self.basis, self.signs, self.cb = P.fill(K, g, n_slots, dev, seed)
        order = (torch.randperm(n_slots - 1, generator=gen) + 1).tolist()
        prefix = [[order.pop() for _ in range(P0)] for P0, _ in groups]
        rows = [(prefix[i] if i >= 0 else []) + [order.pop() for _ in range(own)] for i, _, own, _ in seqs]
        width = max(1, max(len(r) for r in rows))
        self.table = torch.tensor([r + [0] * (width - len(r)) for r in rows], dtype=torch.int32, device=dev)
        self.max_pages = width if any(rows) else 0
        from bmx_b200.rope import default_rope_tables

        cos, sin = default_rope_tables(500000.0, D, 128 * (width + 1), device=dev)
        self.cos, self.sin = cos.half(), sin.half()
        self.rope = K.rope_fragments(self.cos, self.sin, width)
        k_win, v_win = torch.randn(B, h_kv, cap, D, generator=gen).mul_(0.5).half(), torch.randn(B, h_kv, cap, D, generator=gen).half()
        self.q = torch.randn(B, h_kv * G, D, generator=gen).half()
        ref = []
        for b, (_, _, _, tail) in enumerate(seqs):
            k, v = P.pages(K, self.pool, rows[b], self.basis, self.signs, self.cb) if rows[b] else (torch.zeros(h_kv, 0, D, dtype=torch.float64),) * 2
            k = torch.cat([P.rotate(k, self.cos, self.sin, torch.arange(128 * len(rows[b]))), k_win[b, :, :tail].double()], 1)
            v = torch.cat([v, v_win[b, :, :tail].double()], 1)
            ref.append(P.attend(self.q[b][:, None], k, v, torch.ones(1, k.shape[1], dtype=torch.bool))[:, 0])
            k_win[b, :, tail:], v_win[b, :, tail:] = float("nan"), float("nan")
        self.ref, self.q, self.k_win, self.v_win = torch.stack(ref), self.q.to(dev), k_win.to(dev), v_win.to(dev)
        self.n_pages = torch.tensor([len(r) for r in rows], dtype=torch.int32, device=dev)
        self.tail_len = torch.tensor([t for *_, t in seqs], dtype=torch.int32, device=dev)
        members = [[b for b, s in enumerate(seqs) if s[0] == i] for i in range(len(groups))]
        self.groups = K.PrefixGroups(g, B, members, [P0 for P0, _ in groups], dev, n_split=n_split)
        self.v_lut = K.v_lut_tensor(K.GAUSSIAN_CODEBOOK[2], dev)
        self.ws = K.decode_shared_workspace(g, B, self.groups, dev)

    def decode(self, K, rope=True, q=None, **kw):
        return K.k2b_decode_shared(self.pool, self.q if q is None else q, self.basis, self.table, self.n_pages, self.max_pages, self.groups, self.cos, self.sin,
                                   self.rope if rope else None, self.k_win, self.v_win, self.tail_len, self.v_lut, self.signs, 1 / math.sqrt(D), self.ws, **kw)


MEMBERS = [(0, 64), (1, 1), (3, 130), (0, 0), (2, 191)]


@pytest.mark.gpu
@pytest.mark.parametrize("groups,alone", [
    ([(1, MEMBERS)], ()), ([(2, [(0, 5)])], ()), ([(9, MEMBERS * 3)], [(4, 60), (0, 3)]), ([(3, MEMBERS), (17, MEMBERS[:2]), (1, MEMBERS * 2)], [(1, 1)]),
    ([(40, [(0, 70), (1, 100)] * 40)], ()), ([(0, MEMBERS[:2])], [(3, 9)]), ([(5, [(0, 0)] * 33)], ()),
])
@pytest.mark.parametrize("split,fragments", [(None, True), (1, False), (7, True), (64, False)])
def test_groups_and_single_sequences(groups, alone, split, fragments):
    from bmx_b200 import kernels as K

    w = World(K, _dev(), groups, alone, n_split=split)
    P.assert_attention(w.decode(K, rope=fragments), w.ref)
    K.check_status(w.ws)


@pytest.mark.gpu
@pytest.mark.parametrize("h_kv,G,rank,group,per_head", [(1, 1, 16, 32, True), (3, 2, 16, 128, False), (2, 8, 32, 32, True), (2, 3, 32, 64, False), (1, 7, 16, 64, True),
                                                        (2, 5, 16, 64, False), (8, 4, 32, 64, True)])
def test_head_layouts(h_kv, G, rank, group, per_head):
    from bmx_b200 import kernels as K

    n = 140 if h_kv == 1 else 37
    w = World(K, _dev(), [(6, [(i % 3, 1 + i % 150) for i in range(n)])], [(2, 50)], h_kv=h_kv, G=G, rank=rank, group=group, per_head=per_head)
    P.assert_attention(w.decode(K), w.ref)
    out = torch.full((w.q.shape[0], h_kv * G, D), 9.0, device=w.q.device)
    P.assert_attention(w.decode(K, out=out), w.ref, "float32")


@pytest.mark.gpu
def test_no_groups_equals_the_plain_step_and_empty_sequences_give_zero():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [], [(5, 60), (1, 1), (9, 150)])
    plain = K.k2b_decode(w.pool, w.q, w.basis, w.table, w.n_pages, w.max_pages, w.cos, w.sin, w.k_win, w.v_win, w.tail_len, w.v_lut, w.signs, 1 / math.sqrt(D),
                         K.decode_workspace(w.geom, 3, w.max_pages, w.q.device))
    P.assert_one_step(w.decode(K), plain)
    w = World(K, _dev(), [(3, [(0, 9)] * 3)], [(0, 0)])
    out = w.decode(K)
    P.assert_attention(out, w.ref)
    assert not out[int((w.n_pages == 0).nonzero())].any()


@pytest.mark.gpu
def test_large_scores_stay_exact_across_the_merge():
    """Queries that single out keys in the prefix for some sequences and in their own part for others (scores tens of units apart)."""
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [(6, [(1, 50)] * 12)])
    out = w.decode(K, q=(w.q * 6).contiguous())
    ref = []
    for b in range(12):
        rows = w.table[b, : int(w.n_pages[b])].tolist()
        k, v = P.pages(K, w.pool, rows, w.basis, w.signs, w.cb)
        k = torch.cat([P.rotate(k, w.cos, w.sin, torch.arange(128 * len(rows))), w.k_win[b, :, :50].cpu().double()], 1)
        v = torch.cat([v, w.v_win[b, :, :50].cpu().double()], 1)
        ref.append(P.attend((w.q[b] * 6).half()[:, None], k, v, torch.ones(1, k.shape[1], dtype=torch.bool))[:, 0])
    # scores six times larger carry six times the key rounding's error: sqrt(36 + 2/3) u = 6.1 u = 3e-3
    out, ref = out.cpu().double(), torch.stack(ref)
    assert float((out - ref).norm() / ref.norm()) < 6e-3


@pytest.mark.gpu
def test_another_stream_and_a_replayed_graph():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [(9, MEMBERS * 3)], [(4, 60)])
    want = w.decode(K)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(w.decode(K), want)
    torch.cuda.current_stream().wait_stream(side)
    out, graph = torch.zeros_like(want), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        w.decode(K, out=out)
    for _ in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    w.q.mul_(-1)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out, w.decode(K)) and not torch.equal(out, want)


@pytest.mark.gpu
def test_fragments_that_end_before_a_prefix_are_refused_and_reported():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [(6, [(0, 10)] * 4)])
    with pytest.raises(AssertionError, match="rearranged"):
        K.k2b_decode_shared(w.pool, w.q, w.basis, w.table, w.n_pages, w.max_pages, w.groups, w.cos, w.sin, w.rope[:5], w.k_win, w.v_win, w.tail_len, w.v_lut,
                            w.signs, 0.1, w.ws)
    w.groups.max_prefix = 5                            # past the host's check: the kernel leaves the sixth page out and says so
    K.k2b_decode_shared(w.pool, w.q, w.basis, w.table, w.n_pages, w.max_pages, w.groups, w.cos, w.sin, w.rope[:5], w.k_win, w.v_win, w.tail_len, w.v_lut,
                        w.signs, 0.1, w.ws)
    with pytest.raises(_lib.BmxkError, match="rotation tables"):
        K.check_status(w.ws)


def test_refusals():
    lib = _lib.lib()
    a = 4096
    good = _lib.K2bGeom(2, 4, 128, 32, 64, 2, 3, 2, 1)

    def call(g=good, q=a, batch=2, skip=a, members=a, n_groups=1, max_members=2, n_split=1, frag=a, rope_pages=4, scale=0.1, nbytes=1 << 30, out=a, dtype=0,
             max_pages=3, own=2):
        return lib.bmxk_k2b_decode_shared(ctypes.byref(g), q, a, a, a, a, 3, a, batch, max_pages, own, skip, members, a, n_groups, max_members, n_split, a, a, frag,
                                          rope_pages, a, a, a, 192, (ctypes.c_uint32 * 4)(), a, scale, a, nbytes, out, dtype, None)

    for kw, word in ((dict(g=_lib.K2bGeom(2, 4, 64, 32, 64, 2, 3, 2, 0)), b"layout 1"), (dict(g=_lib.K2bGeom(2, 9, 128, 32, 64, 2, 3, 2, 1)), b"n_q_groups"),
                     (dict(g=_lib.K2bGeom(2, 4, 128, 8, 64, 2, 3, 2, 1)), b"rank"), (dict(g=_lib.K2bGeom(2, 4, 128, 32, 48, 2, 3, 2, 1)), b"group"),
                     (dict(g=_lib.K2bGeom(2, 4, 128, 32, 64, 3, 3, 2, 1)), b"n_coef_heads"), (dict(batch=0), b"batch"), (dict(n_groups=-1), b"n_groups"),
                     (dict(max_members=3), b"max_members"), (dict(n_split=0), b"n_split"), (dict(n_split=65), b"n_split"), (dict(skip=None), b"null"),
                     (dict(members=None), b"null"), (dict(own=-1), b"max_own_pages"), (dict(own=4), b"max_own_pages"), (dict(scale=0.0), b"sm_scale"), (dict(scale=-1.0), b"sm_scale"), (dict(nbytes=64), b"workspace"),
                     (dict(q=a + 4), b"16-byte"), (dict(rope_pages=0), b"rope_pages"), (dict(out=a + 8), b"16-byte")):
        assert call(**kw) == _lib.BMXK_ERR_INVALID and word in lib.bmxk_last_error(), (kw, lib.bmxk_last_error())
    # outputs are checked before anything is launched, whatever the prefixes
    for kw, word in ((dict(out=None), b"output"), (dict(dtype=1), b"out_dtype")):
        assert call(**kw) == _lib.BMXK_ERR_INVALID and word in lib.bmxk_last_error(), (kw, lib.bmxk_last_error())
    assert lib.bmxk_k2b_decode_shared_workspace_bytes(ctypes.byref(good), 0, 1) == 0
    from bmx_b200 import kernels as K

    g = K.k2b_geom(2, 4)
    for members, pages in (([[0, 1], [1]], [2, 2]), ([[0, 4]], [1]), ([[0, 0]], [1]), ([[-1]], [1]), ([[0]], [-1])):
        with pytest.raises(ValueError):
            K.PrefixGroups(g, 4, members, pages, "cpu", n_split=1)
