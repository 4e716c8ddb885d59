"""Sequences that fork, share their prompt, move and fall out of a sliding window over one page pool: the allocator's bookkeeping
(host) and the layer built on it (GPU), every live sequence decoding to what a state of its own gives."""

import math
import random

import pytest
import torch

from bmx_b200.paging import PageAllocator, _runs

D = 128


def test_shared_slots_are_free_again_when_the_last_holder_ends():
    a = PageAllocator(6)
    a.alloc("p", 3)
    assert a.share("p", "c1") == [0, 1, 2] and a.share("c1", "c2") == [0, 1, 2] and a.in_use == 3
    assert a.alloc("c1", 1) == [3] and a.slots("c1") == [0, 1, 2, 3] and a.slots("p") == [0, 1, 2]
    assert a.free("p") == 0 and a.in_use == 4
    assert a.free("c1") == 1 and a.free("c2") == 3 and a.in_use == 0
    a.alloc("x", 1)
    with pytest.raises(ValueError):
        a.share("x", "x")
    assert a.share("nobody", "y") == [] and a.free("y") == 0


def test_released_pages_leave_holes_and_shared_ones_stay():
    a = PageAllocator(8)
    a.alloc("p", 5)
    a.share("p", "c")
    assert a.available("p", 1, 4) == 3
    assert a.release("p", 1, 4) == 0 and a.slots("p") == [0, -1, -1, -1, 4] and a.in_use == 5
    assert a.available("c", 1, 4) == 6 and a.release("c", 1, 4) == 3 and a.in_use == 2 and a.release("c", 1, 4) == 0
    assert a.alloc("c", 2, [0, 2], 4) == [1, 2] and a.slots("c") == [0, -1, -1, -1, 4, 1, -1, 2, -1]
    for bad in ((2, 1), (-1, 2), (0, 99)):
        with pytest.raises(ValueError):
            a.release("c", *bad)
    assert a.free("p") == 0 and a.free("c") == 4 and a.in_use == 0 and sorted(a._free) == list(range(8))


def test_compaction_closes_the_holes_and_keeps_who_holds_what():
    rng = random.Random(4)
    for _ in range(200):
        a, data, pool = PageAllocator(rng.randint(1, 40)), {}, {}
        for step in range(rng.randint(1, 60)):
            what, seq = rng.random(), rng.randint(0, 6)
            if what < 0.5:
                n = rng.randint(0, 4)
                try:
                    got = a.alloc(seq, n)
                except MemoryError:
                    continue
                for s in got:
                    pool[s] = (seq, step, s)
                data.setdefault(seq, []).extend(pool[s] for s in got)
            elif what < 0.65:
                a.free(seq)
                data.pop(seq, None)
            elif what < 0.75 and seq in data and len(data[seq]) > 1:
                a.release(seq, 0, 1)
                data[seq][0] = None
            elif what < 0.85 and not a.slots(seq) and data.get((seq + 1) % 7):
                a.share((seq + 1) % 7, seq)
                data[seq] = list(data[(seq + 1) % 7])
            elif what < 0.95:
                moved, holes = a.compact()
                assert not set(moved) & set(holes) and len(set(holes)) == len(holes) and all(s < a.in_use for s in holes)
                for s, d in zip(moved, holes):
                    pool[d] = pool[s]
            for name, want in data.items():
                assert [None if s < 0 else pool[s] for s in a.slots(name)] == want
            held = {s for name in data for s in a.slots(name) if s >= 0}
            assert held | set(a._free) == set(range(a.n_slots)) and not held & set(a._free) and a.in_use == len(held) and len(a._free) == len(set(a._free))
        a.compact()
        a.shrink(max(1, a.in_use))
        assert a.n_slots == max(1, a.in_use)
        if a.in_use:
            with pytest.raises(ValueError):
                a.shrink(a.in_use - 1)


def test_runs():
    assert _runs([]) == [] and _runs([3]) == [(3, 4)] and _runs([0, 1, 4, 5, 6, 9]) == [(0, 2), (4, 7), (9, 10)]


# ---- on the GPU ----------------------------------------------------------------------------------------------------------

H_KV, G, RANK, GROUP = 2, 4, 32, 64


class Bench:
    """A layer, a state of its own per sequence, and tokens that are reproducible per (sequence, position)."""

    def __init__(self, slots=64, seqs=40, W=32, **kw):
        if not torch.cuda.is_available():
            pytest.skip("needs a CUDA device")
        from bmx_b200 import kernels as K
        from bmx_b200.paging import PagedK2bLayer
        from bmx_b200.rope import apply_rope, default_rope_tables
        from tests.test_k2b_gpu import make_k2b_inputs

        self.dev, self.K, self.W, self.kw = torch.device("cuda:0"), K, W, kw
        self.cos, self.sin = (t.half() for t in default_rope_tables(500000.0, D, 8192, device=self.dev))
        self.geom = K.k2b_geom(H_KV, G, 128, RANK, GROUP, H_KV)
        self.layer = PagedK2bLayer(self.geom, slots, seqs, W, self.dev, self.cos, self.sin, **kw)
        k, v, basis = make_k2b_inputs(11, 6, H_KV, 3000, RANK, True)
        self.k, self.v, self.basis = k.to(self.dev), v.to(self.dev), basis.to(self.dev)
        self.layer.set_basis(basis)
        self.rot = lambda x, t0: apply_rope(x.float(), self.cos[t0: t0 + x.shape[1]].float(), self.sin[t0: t0 + x.shape[1]].float()).half()
        self.text = {}                                 # sequence -> [(stream, begin, end)] of what it has been fed
        self.gen = torch.Generator().manual_seed(2)

    def feed(self, seq, stream, n, chunk=10 ** 9):
        t0 = self.layer.seq_len(seq)
        for a in range(t0, t0 + n, chunk):
            b = min(t0 + n, a + chunk)
            k = self.k[stream, :, a:b]
            self.layer.append(seq, k, self.rot(k, a), self.v[stream, :, a:b])
        self.text[seq] = self.text.get(seq, []) + [(stream, t0, t0 + n)]

    def start(self, seq, stream, n, chunk=10 ** 9):
        self.layer.add_sequence(seq)
        self.text.pop(seq, None)
        self.feed(seq, stream, n, chunk)

    def fork(self, seq, *children):
        self.layer.fork(seq, *children)
        for c in children:
            self.text[c] = list(self.text[seq])

    def check(self, seqs, tol=1e-3):
        """One decode step of these sequences against states of their own (same pages, another split of the walk: fp16 weights relative
        to another running maximum, 2^-11 each, and the output's rounding)."""
        from bmx_b200.engine import K2bLayerState

        q = torch.randn(len(seqs), H_KV * G, D, generator=self.gen).half().to(self.dev)
        out = self.layer.decode(seqs, q).float()
        for i, s in enumerate(seqs):
            k = torch.cat([self.k[st, :, a:b] for st, a, b in self.text[s]], 1)
            v = torch.cat([self.v[st, :, a:b] for st, a, b in self.text[s]], 1)
            st = K2bLayerState(self.geom, 1, max(128, k.shape[1]), self.W, self.dev, self.cos, self.sin,
                               **{x: y for x, y in self.kw.items() if x in ("sliding_window", "sinks")})
            st.set_basis(self.basis)
            st.append(k[None], self.rot(k, 0)[None], v[None])
            ref = st.decode(q[i][None])[0].float()
            assert float((out[i] - ref).abs().max() / ref.abs().max()) < tol, s
        return out


@pytest.mark.gpu
def test_forks_share_their_prompt_and_go_their_own_ways():
    b = Bench(slots=40)
    b.layer.SHARED_MIN_TILES = 0                          # share whatever can be shared
    b.start("doc", 0, 1500, 700)                          # 11 pages and 92 tokens in the window
    assert b.layer.alloc.in_use == 11
    kids = [f"k{i}" for i in range(9)]
    b.fork("doc", *kids)
    assert b.layer.alloc.in_use == 11
    b.check(["doc"] + kids)
    for i, c in enumerate(kids):
        b.feed(c, 1 + i % 5, 1 + 37 * i)                  # some of them commit pages of their own
    b.start("other", 3, 300)
    order = kids[:4] + ["other", "doc"] + kids[4:]
    b.check(order)
    assert b.layer._plan[4] is not None and b.layer._plan[4].max_members == 10     # the prompt was attended once
    plan = b.layer._plan
    b.feed("k1", 2, 1)                                    # a token that commits no page: tables and groups stay
    b.check(order)
    assert b.layer._plan is plan
    b.check(["k1", "k1", "k8"])                           # the same sequence twice
    assert b.layer._plan[4].max_members == 3
    b.layer.SHARED_MIN_TILES = 5                          # too little to save here
    b.check(["doc"] + kids)
    assert b.layer._plan[4] is None
    b.layer.SHARED_MIN_TILES = 0
    before = b.layer.alloc.in_use
    freed = b.layer.drop_sequence("doc")
    assert freed == 0 and b.layer.alloc.in_use == before  # the children hold the prompt
    b.check(kids)
    for c in kids[:-1]:
        b.layer.drop_sequence(c)
    b.check(["k8", "other"])
    assert b.layer.drop_sequence("k8") >= 11
    with pytest.raises(ValueError):
        b.fork("other", "x", "x")
    with pytest.raises(ValueError):
        b.fork("other", "other")
    with pytest.raises(MemoryError):
        b.fork("other", *range(100))
    assert set(b.layer._rows) == {"other"}


@pytest.mark.gpu
def test_forks_of_forks_and_forks_within_the_window():
    b = Bench()
    b.layer.SHARED_MIN_TILES = 0
    b.start("a", 0, 20)                                   # nothing committed yet
    b.fork("a", "b")
    b.feed("b", 1, 1300)
    b.fork("b", "c", "d", "e")
    b.feed("d", 2, 200)
    b.check(["a", "b", "c", "d", "e"])
    b.layer.add_sequence("empty")
    b.text["empty"] = []
    b.fork("empty", "empty2")
    b.feed("empty2", 4, 130)
    b.check(["empty2", "e"])


@pytest.mark.gpu
def test_compaction_growth_and_shrinking_keep_every_sequence():
    b = Bench(slots=30)
    b.layer.SHARED_MIN_TILES = 0
    for i, n in enumerate((500, 900, 260, 700)):
        b.start(i, i, n, 128)
    b.fork(1, "f")
    b.feed("f", 5, 300)
    b.layer.drop_sequence(0)
    b.layer.drop_sequence(2)
    live = [1, "f", 3]
    used = b.layer.alloc.in_use
    moved = b.layer.compact()
    assert moved > 0 and max(s for x in live for s in b.layer.alloc.slots(x)) == used - 1 and b.layer.compact() == 0
    b.check(live)
    with pytest.raises(MemoryError):
        b.layer.resize(used - 1)
    b.layer.resize(used)
    assert b.layer.pool.n_slots == used == b.layer.alloc.n_slots
    b.check(live)
    with pytest.raises(MemoryError):
        b.start("big", 4, 1000)
    b.layer.drop_sequence("big")
    b.layer.drop_sequence(3)
    b.layer.resize(50)
    b.start("big", 4, 2900)
    b.check([1, "f", "big"])


@pytest.mark.gpu
def test_a_sliding_window_frees_pages_and_everything_runs_together():
    """Prompt, forks, tokens one by one through page commits, pages falling out of the window, compaction, resize, join and leave."""
    b = Bench(slots=24, seqs=8, sliding_window=300, sinks=5)
    b.start("a", 0, 2000)                                 # 15 pages committed, of which the sinks' and the window's are kept
    kept = [s for s in b.layer.alloc.slots("a") if s >= 0]
    assert len(b.layer.alloc.slots("a")) == 15 and len(kept) == 3 and b.layer.alloc.in_use == 3
    b.check(["a"])
    b.fork("a", "b", "c")
    for i in range(140):
        b.feed("a", 1, 1), b.feed("b", 2, 1)
        if i % 35 == 0:
            b.check(["a", "b", "c"])
    b.feed("c", 3, 700, 90)
    b.check(["a", "b", "c"])
    assert all(b.layer.alloc.slots(s)[0] == kept[0] for s in "abc")        # the sinks' page is shared for good
    b.layer.drop_sequence("b")
    b.layer.compact()
    b.check(["c", "a"])
    b.layer.resize(b.layer.alloc.in_use + 5)
    b.start("d", 4, 100)
    b.feed("d", 4, 400)
    b.check(["c", "a", "d"])
    assert b.layer.alloc.in_use <= b.layer.alloc.n_slots
    # a prompt that needs more slots than are left changes nothing
    b.layer.add_sequence("e"), b.layer.append("e", b.k[5, :, :200], b.rot(b.k[5, :, :200], 0), b.v[5, :, :200])
    b.text["e"] = [(5, 0, 200)]
    state = (dict(b.layer._tail), dict(b.layer._committed), b.layer.alloc.in_use, b.layer.alloc.slots("e"))
    free = b.layer.alloc.n_slots - b.layer.alloc.in_use
    if free < 4:
        with pytest.raises(MemoryError):
            b.feed("e", 5, 900)
        assert state == (dict(b.layer._tail), dict(b.layer._committed), b.layer.alloc.in_use, b.layer.alloc.slots("e"))
    b.check(["e", "a", "c", "d"])


@pytest.mark.gpu
def test_what_a_layer_refuses():
    from bmx_b200 import kernels as K
    from bmx_b200.paging import PagedK2bLayer

    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    dev = torch.device("cuda:0")
    cos = torch.zeros(256, D, dtype=torch.float16, device=dev)
    for geom, kw in ((K.k2b_geom(1, 1), dict(sliding_window=0)), (K.k2b_geom(1, 1), dict(sliding_window=3, sinks=-1)), (K.k2b_geom(1, 1), dict(sinks=2)),
                     (K.k2b_geom(1, 1, page=64), dict(sliding_window=8))):
        with pytest.raises(ValueError):
            PagedK2bLayer(geom, 4, 2, 32, dev, cos, cos, **kw)
    # 64-token pages fork and compact too; their steps stream every sequence
    layer = PagedK2bLayer(K.k2b_geom(1, 1, page=64), 8, 4, 32, dev, cos, cos)
    x = torch.randn(1, 200, D, generator=torch.Generator().manual_seed(0)).half().to(dev)
    layer.add_sequence("a"), layer.append("a", x, x, x)
    layer.fork("a", "b")
    q = torch.randn(1, D).half().to(dev)
    out = layer.decode(["a", "b"], torch.stack([q, q]) / math.sqrt(D))
    assert torch.equal(out[0], out[1]) and layer.alloc.in_use == 2 and layer.compact() == 0
