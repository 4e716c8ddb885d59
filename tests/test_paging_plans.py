"""What PagedK2bLayer hands to a decode step, on the host: page table, page counts and window lengths are those of the sequences as they
are at the call, whatever a layer keeps between steps.  The kernels are replaced by functions that record their arguments."""

import random
import types

import pytest
import torch

from bmx_b200 import kernels as K
from bmx_b200 import paging
from bmx_b200.paging import PageAllocator, PagedK2bLayer

D = 128


class Steps:
    """A layer on the CPU whose kernel calls are recorded; every step's operands are compared with the layer's books."""

    def __init__(self, monkeypatch, slots=60, seqs=8, W=32, sms=1, n_q_groups=4, **kw):
        self.stream = types.SimpleNamespace(cuda_stream=7)
        monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: self.stream)
        monkeypatch.setattr(K, "k2b_append", lambda *a: None)
        monkeypatch.setattr(K, "copy_slots", lambda *a: None)
        monkeypatch.setattr(K, "sm_count", lambda device: sms)
        monkeypatch.setattr(K, "decode_workspace", lambda g, n, pages, device: torch.zeros(1))
        monkeypatch.setattr(K, "decode_shared_workspace", lambda *a: torch.zeros(1))
        monkeypatch.setattr(K, "rope_fragments", lambda cos, sin, n: torch.zeros(n, 8192, dtype=torch.int32))
        for name in ("k2b_decode", "k2b_decode_sliding", "k2b_decode_shared"):
            monkeypatch.setattr(K, name, lambda *a, _name=name, **k: self.handed.append((_name, a)))
        self.handed = []
        cos = torch.zeros(64 * 128, D, dtype=torch.float16)
        self.geom = K.k2b_geom(1, n_q_groups, 128, 16, 64, 1)
        self.layer = PagedK2bLayer(self.geom, slots, seqs, W, "cpu", cos, cos, max_pages_per_seq=64, **kw)
        self.layer.set_basis(torch.zeros(D, 16))

    def feed(self, seq, n):
        x = torch.zeros(1, n, D, dtype=torch.float16)
        self.layer.append(seq, x, x, x)

    def start(self, seq, n):
        self.layer.add_sequence(seq)
        self.feed(seq, n)

    def step(self, seqs):
        layer = self.layer
        layer.decode(seqs, torch.zeros(len(seqs), self.geom.n_q_groups, D, dtype=torch.float16))
        name, a = self.handed.pop()
        table, n_pages, max_pages = a[3], a[4], a[5]
        at = 10 if name == "k2b_decode_shared" else 8
        tail = a[at + 2]
        for i, s in enumerate(seqs):
            slots = layer.alloc.slots(s)
            assert int(n_pages[i]) == len(slots) == layer._committed[s] // 128 <= max_pages or not len(slots)
            assert table[i, : len(slots)].tolist() == slots
            assert int(tail[i]) == layer._tail[s]
            if layer.sliding_window is not None:  # every page that holds a visible token has a slot
                total = 128 * int(n_pages[i]) + int(tail[i])
                for p in range(int(n_pages[i])):
                    if 128 * p < layer.sinks or 128 * p + 127 >= total - layer.sliding_window:
                        assert 0 <= int(table[i, p]) < layer.alloc.n_slots
        if name == "k2b_decode_shared":
            groups = a[6]
            skip, info, members = groups.skip.tolist(), groups.info.view(-1, 4).tolist(), groups.members.tolist()
            for begin, end, first, pages in info:
                rows = members[begin:end]
                assert first in rows and all(skip[r] == pages for r in rows)
                assert all(table[r, :pages].tolist() == table[first, :pages].tolist() and int(n_pages[r]) >= pages for r in rows)
            assert max_pages - groups.min_prefix >= max(int(n) - s for n, s in zip(n_pages.tolist(), skip))
        return name


def test_freeing_a_sequence_without_a_page_left_is_a_change():
    a = PageAllocator(4)
    a.alloc("s", 2)
    a.release("s", 0, 2)
    before = a.version
    assert a.free("s") == 0 and a.version != before and a.slots("s") == []
    before = a.version
    assert a.free("s") == 0 and a.version == before          # nothing of it is left


@pytest.mark.parametrize("window,W,sinks", [(100, 32, 0), (128, 128, 0), (40, 64, 0), (100, 32, 3)])
def test_a_name_used_again_does_not_get_the_table_of_its_predecessor(monkeypatch, window, W, sinks):
    """Under a window that the recent tokens cover, a sequence's entries are all -1: ending it gives no slot back."""
    b = Steps(monkeypatch, W=W, sliding_window=window, sinks=sinks)
    b.start("s", 800)
    b.step(["s"])
    b.layer.drop_sequence("s")
    b.start("s", 10)
    b.step(["s"])
    b.feed("s", 600)
    b.step(["s"])


@pytest.mark.parametrize("kw", [{}, dict(sliding_window=150), dict(sliding_window=30), dict(sliding_window=60, sinks=1), dict(sliding_window=300, sinks=200)])
def test_steps_get_what_the_sequences_hold_whatever_happened_in_between(monkeypatch, kw):
    """Random joins, growth, forks, ends, compactions, resizes and streams; a step after each, often of the same sequences."""
    rng = random.Random(len(str(kw)))
    kinds = set()
    for _ in range(25):
        b = Steps(monkeypatch, slots=rng.randint(20, 60), **kw)
        layer, seqs = b.layer, []
        for _ in range(60):
            what, name = rng.random(), rng.choice("abcdef")
            try:
                if name not in layer._rows:
                    b.start(name, rng.choice([0, 1, 31, 160, 161, 300, 700]))
                elif what < 0.45:
                    b.feed(name, rng.choice([1, 1, 1, 20, 128, 200]))
                elif what < 0.6:
                    child = rng.choice("abcdef")
                    if child not in layer._rows:
                        layer.fork(name, child)
                elif what < 0.75:
                    layer.drop_sequence(name)
                elif what < 0.85:
                    layer.compact()
                elif what < 0.92:
                    layer.resize(max(layer.alloc.in_use, 1) + rng.randint(0, 30))
                else:
                    b.stream = types.SimpleNamespace(cuda_stream=rng.choice([7, 8]))
                    monkeypatch.setattr(torch.cuda, "current_stream", lambda device=None: b.stream)
            except (MemoryError, AssertionError):
                layer.drop_sequence(name)                     # out of slots or of table columns
            live = sorted(layer._rows)
            if not live:
                continue
            if not seqs or any(s not in layer._rows for s in seqs) or rng.random() < 0.3:
                seqs = rng.sample(live, rng.randint(1, len(live)))
            kinds.add(b.step(seqs))
    assert kinds == ({"k2b_decode", "k2b_decode_shared"} if not kw else {"k2b_decode_sliding"})


def test_a_pool_that_is_replaced_stays_until_the_copying_stream_is_through(monkeypatch):
    """A pool belongs to the stream it was made on; resized on another one, it is not free before that one has copied it."""

    class Held:
        is_cuda = True

        def __init__(self):
            self.streams = []

        def record_stream(self, stream):
            self.streams.append(stream)

    b = Steps(monkeypatch, slots=10)
    b.start("a", 500)
    old = b.layer.pool
    old.pages, old.coefs = Held(), Held()
    b.stream = types.SimpleNamespace(cuda_stream=9)
    b.layer.resize(20)
    assert b.layer.pool is not old and old.pages.streams == [b.stream] and old.coefs.streams == [b.stream]
    b.step(["a"])
