"""Attention under a sliding window with sinks, for single tokens and for blocks of prompt rows, against a plain float64 form; what is
hidden is not read or does not matter, whatever it holds."""

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
    """A pool, page tables and windows of sequences of the given lengths; hidden pages point at a slot full of NaN, hidden tokens and
    what lies behind the end of a window are NaN."""

    def __init__(self, K, dev, lens, window, sinks, rows=1, h_kv=2, G=4, rank=32, group=64, per_head=True, recent=64, seed=5, stride=0):
        self.geom = g = K.k2b_geom(h_kv, G, 128, rank, group, h_kv if per_head else 1)
        self.window, self.sinks, self.rows = window, sinks, rows
        self.held = [(max(0, n - recent) // 128, n - max(0, n - recent) // 128 * 128) for n in lens]
        self.cap = recent + 128
        gen = torch.Generator().manual_seed(seed)
        B, width = len(lens), max(1, max(p for p, _ in self.held))
        n_slots = 1 + sum(p for p, _ in self.held)
        self.pool, self.basis, self.signs, self.cb = P.fill(K, g, n_slots, dev, seed)
        order = (torch.randperm(n_slots - 1, generator=gen) + 1).tolist()
        bad = 0
        P.norms(self.pool)[bad] = float("nan")
        P.coefs(self.pool)[bad] = float("nan")
        table = torch.full((B, width + stride), bad, dtype=torch.int32)
        from bmx_b200.rope import default_rope_tables

        cos, sin = default_rope_tables(500000.0, D, 128 * (width + 2), device=dev)
        self.cos, self.sin = cos.half(), sin.half()
        self.k_win = torch.randn(B, h_kv, self.cap, D, generator=gen).mul_(0.5).half()
        self.v_win = torch.randn(B, h_kv, self.cap, D, generator=gen).half()
        self.q = torch.randn(B, h_kv * G, rows, D, generator=gen).half()
        self.pos0 = max(0, min(lens) - rows) if rows > 1 else None
        self.ref = []
        for b, (pages, tail) in enumerate(self.held):
            mine = [order.pop() for _ in range(pages)]
            k, v = P.pages(K, self.pool, mine, self.basis, self.signs, self.cb) if mine else (torch.zeros(h_kv, 0, D, dtype=torch.float64),) * 2
            k = P.rotate(k, self.cos, self.sin, torch.arange(128 * pages))
            k = torch.cat([k, self.k_win[b, :, :tail].double()], 1)
            v = torch.cat([v, self.v_win[b, :, :tail].double()], 1)
            total = 128 * pages + tail
            x = (total - 1 if rows == 1 else self.pos0) + torch.arange(rows)[:, None]
            t = torch.arange(total)
            seen = (t <= x) & ((t < sinks) | (t > x - window))
            self.ref.append(P.attend(self.q[b], k, v, seen))
            any_seen = seen.any(0)
            for j, slot in enumerate(mine):
                here = any_seen[128 * j: 128 * j + 128]
                if here.any():
                    table[b, j] = slot
                for r in (~here).nonzero().flatten().tolist():
                    P.norms(self.pool)[slot, :, r] = float("inf") if r % 2 else float("nan")
                    P.coefs(self.pool)[slot, :, r // 8, :, r % 8] = float("nan")
            hidden = torch.cat([~any_seen[128 * pages:], torch.ones(self.cap - tail, dtype=torch.bool)])
            self.k_win[b, :, hidden] = float("nan")
            self.v_win[b, :, hidden] = float("inf")
        self.ref = torch.stack(self.ref)
        self.table = table.to(dev)[:, :width]
        self.max_pages = width if any(p for p, _ in self.held) else 0
        self.n_pages = torch.tensor([p for p, _ in self.held], dtype=torch.int32, device=dev)
        self.tail_len = torch.tensor([t for _, t in self.held], dtype=torch.int32, device=dev)
        self.k_win, self.v_win, self.q = self.k_win.to(dev), self.v_win.to(dev), self.q.to(dev)
        self.v_lut = K.v_lut_tensor(K.GAUSSIAN_CODEBOOK[2], dev)
        self.ws = K.decode_workspace(g, B, width, dev)

    def decode(self, K, **kw):
        return K.k2b_decode_sliding(self.pool, self.q[:, :, 0].contiguous(), self.basis, self.table, self.n_pages, self.max_pages, self.cos, self.sin,
                                    self.k_win, self.v_win, self.tail_len, self.v_lut, self.signs, 1 / math.sqrt(D), self.ws, self.window, self.sinks,
                                    **kw)

    def prompt(self, K, rope=None, **kw):
        return K.k2b_prefill_sliding(self.pool, self.q, self.pos0, self.basis, self.table, self.n_pages, self.max_pages, self.cos, self.sin, rope,
                                     self.k_win, self.v_win, self.tail_len, self.v_lut, self.signs, 1 / math.sqrt(D), self.ws, self.window, self.sinks,
                                     **kw)


LENS = [1500, 700, 64, 1, 191, 192, 193, 1023]


@pytest.mark.gpu
@pytest.mark.parametrize("sinks", [0, 1, 4, 128, 130, 10 ** 9, 2 ** 63 - 1])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 65, 127, 128, 129, 500, 10 ** 12, 2 ** 63 - 1])
def test_decode_sees_the_window_and_the_sinks(window, sinks):
    from bmx_b200 import kernels as K

    w = World(K, _dev(), LENS, window, sinks)
    P.assert_attention(w.decode(K), w.ref[:, :, 0], f"window {window} sinks {sinks}")
    K.check_status(w.ws)


@pytest.mark.gpu
@pytest.mark.parametrize("h_kv,G,rank,group,per_head", [(1, 1, 16, 32, True), (3, 2, 16, 128, False), (8, 8, 32, 64, True), (5, 3, 32, 32, False),
                                                        (2, 7, 16, 64, False)])
def test_decode_head_layouts_and_odd_tables(h_kv, G, rank, group, per_head):
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [1333, 400, 77], 300, 5, h_kv=h_kv, G=G, rank=rank, group=group, per_head=per_head, stride=3)
    P.assert_attention(w.decode(K), w.ref[:, :, 0])
    out = torch.full((3, h_kv * G, D), 7.0, device=w.q.device)
    P.assert_attention(w.decode(K, out=out), w.ref[:, :, 0], "float32")
    host = torch.zeros(3, h_kv * G, D, dtype=torch.float16).pin_memory()
    w.decode(K, out=host)
    torch.cuda.synchronize()
    P.assert_attention(host, w.ref[:, :, 0], "pinned")


@pytest.mark.gpu
def test_decode_of_empty_sequences_and_without_a_window_is_defined():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [0, 900, 0], 200, 4)
    out = w.decode(K)
    assert not out[0].any() and not out[2].any()
    P.assert_attention(out, w.ref[:, :, 0])
    empty = World(K, _dev(), [0, 0], 5, 0)
    assert not empty.decode(K).any()
    # no fp16 window at all: 128 * pages tokens are held, and the newest of them is the query's (a world whose last page has no
    # poisoned tokens: under a window of 200 its first 60 would be NaN, and visible to this query)
    w = World(K, _dev(), [0, 900, 0], 400, 4)
    g = w.geom
    none = K.k2b_decode_sliding(w.pool, w.q[1:2, :, 0].contiguous(), w.basis, w.table[1:2], w.n_pages[1:2].contiguous(), w.max_pages, w.cos, w.sin, None,
                                None, None, w.v_lut, w.signs, 1 / math.sqrt(D), w.ws, 128, 0)
    pages = w.held[1][0]
    k, v = P.pages(K, w.pool, [int(w.table[1, pages - 1])], w.basis, w.signs, w.cb)
    k = P.rotate(k, w.cos, w.sin, torch.arange(128 * (pages - 1), 128 * pages))
    assert g.n_q_groups == 4
    P.assert_attention(none[0], P.attend(w.q[1, :, :1], k, v, torch.ones(1, 128, dtype=torch.bool))[:, 0])


@pytest.mark.gpu
def test_decode_equals_the_plain_step_when_everything_is_visible():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [1500, 700, 64, 193], 10 ** 9, 0)
    plain = K.k2b_decode(w.pool, w.q[:, :, 0].contiguous(), w.basis, w.table, w.n_pages, w.max_pages, w.cos, w.sin, w.k_win, w.v_win, w.tail_len, w.v_lut,
                         w.signs, 1 / math.sqrt(D), K.decode_workspace(w.geom, 4, w.max_pages, w.q.device))
    P.assert_one_step(w.decode(K), plain)


@pytest.mark.gpu
@pytest.mark.parametrize("rows,lens,window,sinks", [(2, [700], 300, 4), (33, [1500, 1500], 200, 0), (150, [900, 900], 1, 0), (150, [900, 900], 64, 129),
                                                    (257, [1900], 129, 1), (40, [40], 7, 2), (600, [600], 256, 130), (64, [3000], 500, 300),
                                                    (100, [1200, 1200, 1200], 10 ** 12, 0)])
@pytest.mark.parametrize("split,fragments", [(None, True), (1, False), (5, False)])
def test_prompt_rows_see_their_windows_and_the_sinks(rows, lens, window, sinks, split, fragments):
    from bmx_b200 import kernels as K

    w = World(K, _dev(), lens, window, sinks, rows=rows, recent=128)
    rope = K.rope_fragments(w.cos, w.sin, w.cos.shape[0] // 128) if fragments else None
    P.assert_attention(w.prompt(K, rope, n_split=split), w.ref, f"{rows} rows window {window} sinks {sinks}")
    K.check_status(w.ws)


@pytest.mark.gpu
@pytest.mark.parametrize("h_kv,G,rank,group,per_head", [(1, 1, 16, 32, True), (3, 2, 16, 128, False), (4, 8, 32, 32, True)])
def test_prompt_head_layouts(h_kv, G, rank, group, per_head):
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [1333], 300, 5, rows=130, h_kv=h_kv, G=G, rank=rank, group=group, per_head=per_head, recent=128)
    P.assert_attention(w.prompt(K), w.ref)


@pytest.mark.gpu
def test_prompt_rows_that_see_nothing_give_zero_and_missing_fragments_are_reported():
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [800], 100, 0, rows=64, recent=128)
    w.pos0 = 1000                                     # rows 200 tokens behind the last key: nothing within 100 of them
    assert not w.prompt(K, n_split=1).any() and not w.prompt(K, n_split=3).any()
    w = World(K, _dev(), [800], 100, 4, rows=64, recent=128)
    w.prompt(K, K.rope_fragments(w.cos, w.sin, 2))
    with pytest.raises(_lib.BmxkError, match="rotation tables"):
        K.check_status(w.ws)


@pytest.mark.gpu
def test_plain_decode_takes_queries_that_begin_on_any_fp16():
    """The plain step reads queries by words where it can and by halves where it cannot."""
    from bmx_b200 import kernels as K

    w = World(K, _dev(), [700, 1500], 10 ** 9, 0)
    q = w.q[:, :, 0].contiguous()
    args = (w.basis, w.table, w.n_pages, w.max_pages, w.cos, w.sin, w.k_win, w.v_win, w.tail_len, w.v_lut, w.signs, 1 / math.sqrt(D), w.ws)
    shifted = torch.empty(q.numel() + 1, dtype=torch.float16, device=q.device)[1:].view(q.shape)
    shifted.copy_(q)
    assert shifted.data_ptr() % 4 == 2 and torch.equal(K.k2b_decode(w.pool, shifted, *args), K.k2b_decode(w.pool, q, *args))


@pytest.mark.gpu
def test_another_stream_and_a_replayed_graph():
    from bmx_b200 import kernels as K

    dev = _dev()
    w = World(K, dev, [1500, 700, 64], 200, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        P.assert_attention(w.decode(K), w.ref[:, :, 0])
    torch.cuda.current_stream().wait_stream(side)
    out = torch.zeros_like(w.q[:, :, 0])
    graph = torch.cuda.CUDAGraph()
    q, want = w.q.clone(), w.decode(K)
    with torch.cuda.graph(graph):
        K.k2b_decode_sliding(w.pool, q[:, :, 0].contiguous(), w.basis, w.table, w.n_pages, w.max_pages, w.cos, w.sin, w.k_win, w.v_win, w.tail_len,
                             w.v_lut, w.signs, 1 / math.sqrt(D), w.ws, w.window, w.sinks, out=out)
    for _ in range(2):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want)
    # lengths live on the device: a captured step follows them (the second sequence's window then reaches back to tokens that are NaN
    # here, so the bits are compared)
    w.tail_len.copy_(torch.tensor([w.held[0][1], 0, 10], dtype=torch.int32))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(out.view(torch.int16), w.decode(K).view(torch.int16)) and not torch.equal(out[2], want[2])


@pytest.mark.gpu
def test_a_layer_state_with_a_window_streams_and_its_step_graph_agrees():
    """Token by token through append / decode and through the captured step, across steps that commit pages; prompt rows by prefill_attend."""
    from bmx_b200 import kernels as K
    from bmx_b200.engine import DecodeStepGraph, K2bLayerState
    from bmx_b200.rope import apply_rope, default_rope_tables
    from tests.test_k2b_gpu import make_k2b_inputs

    dev = _dev()
    h_kv, G, B, W, T0, steps, window, sinks = 2, 4, 2, 64, 400, 300, 150, 3
    k, v, basis = make_k2b_inputs(3, B, h_kv, T0 + steps, 32, True)
    k, v = k.to(dev), v.to(dev)
    cos, sin = default_rope_tables(500000.0, D, 1024, device=dev)
    post = apply_rope(k.float(), cos[: T0 + steps], sin[: T0 + steps]).half()
    geom = K.k2b_geom(h_kv, G, 128, 32, 64, h_kv)
    states = [K2bLayerState(geom, B, 1024, W, dev, cos.half(), sin.half(), sliding_window=window, sinks=sinks) for _ in range(2)]
    for st in states:
        st.set_basis(basis.to(dev))
        st.append(k[:, :, :T0], post[:, :, :T0], v[:, :, :T0])
    gen = torch.Generator().manual_seed(1)
    qs = torch.randn(steps, B, h_kv * G, D, generator=gen).half()
    hin = torch.zeros(B * (h_kv * G + 3 * h_kv) * D, dtype=torch.float16).pin_memory()
    hout = torch.zeros(B, h_kv * G, D, dtype=torch.float16).pin_memory()
    graph = DecodeStepGraph(states[1], hin, hout)
    for i in range(steps):
        t = slice(T0 + i, T0 + i + 1)
        states[0].append(k[:, :, t], post[:, :, t], v[:, :, t])
        want = states[0].decode(qs[i].to(dev))
        hin.copy_(torch.cat([x.reshape(-1) for x in (qs[i], post[:, :, t].cpu(), v[:, :, t].cpu(), k[:, :, t].cpu())]))
        graph.step()
        torch.cuda.synchronize()
        assert torch.equal(want.cpu(), hout), i
    st, total = states[0], T0 + steps
    ref, rows = [], 70
    q = torch.randn(B, h_kv * G, rows, D, generator=gen).half()
    for b in range(B):
        kd, vd = P.pages(K, st.pool, st.page_table[b, : st.committed // 128].tolist(), st.basis_f16, st.signs, st.codebook)
        kd = torch.cat([P.rotate(kd, cos.half(), sin.half(), torch.arange(st.committed)), st.k_win[b, :, : st.tail_len].cpu().double()], 1)
        vd = torch.cat([vd, st.v_win[b, :, : st.tail_len].cpu().double()], 1)
        x, t = torch.arange(total - rows, total)[:, None], torch.arange(total)
        seen = (t <= x) & ((t < sinks) | (t > x - window))
        ref.append(P.attend(q[b], kd, vd, seen))
        P.assert_attention(want[b], P.attend(qs[-1][b][:, None], kd, vd, seen[-1:])[:, 0], "last step")
    P.assert_attention(st.prefill_attend(q.to(dev), total - rows), torch.stack(ref), "prompt rows")
    with pytest.raises(NotImplementedError):
        st.decode(qs[0].to(dev), pos_offset=128)


def test_refusals():
    """Checked on the host, before any launch (made-up addresses that nothing reads)."""
    lib = _lib.lib()
    a = 4096

    def decode(g, window=10, sinks=0, batch=2, max_pages=3, out=a, dtype=0, ws_bytes=1 << 30, tail_cap=256, q=a):
        return lib.bmxk_k2b_decode_sliding(ctypes.byref(g), q, a, a, a, a, 3, a, batch, max_pages, a, a, a, a, a, tail_cap, (ctypes.c_uint32 * 4)(), a,
                                           0.1, window, sinks, a, ws_bytes, out, dtype, None)

    good = _lib.K2bGeom(2, 4, 128, 32, 64, 2, 3, 2, 1)
    for kw, word in ((dict(window=0), b"window"), (dict(window=-3), b"window"), (dict(sinks=-1), b"sinks"), (dict(batch=0), b"batch"),
                     (dict(out=None), b"output"), (dict(dtype=1), b"out_dtype"), (dict(ws_bytes=100), b"workspace"), (dict(q=a + 2), b"16-byte"),
                     (dict(out=a + 8), b"16-byte")):
        assert decode(good, **kw) == _lib.BMXK_ERR_INVALID and word in lib.bmxk_last_error(), (kw, lib.bmxk_last_error())
    for g in (_lib.K2bGeom(2, 4, 64, 32, 64, 2, 3, 2, 0), _lib.K2bGeom(2, 4, 128, 32, 64, 2, 3, 2, 0)):
        assert decode(g) == _lib.BMXK_ERR_INVALID and b"layout 1" in lib.bmxk_last_error()

    def prompt(g=good, q=a, window=10, sinks=0, pos0=0, scale=0.1, frag=None, rope_pages=0, n_split=1, ws=None, nbytes=0):
        return lib.bmxk_k2b_prefill_sliding(ctypes.byref(g), q, 8, pos0, a, a, a, a, 3, a, 1, a, a, frag, rope_pages, a, a, a, 256, (ctypes.c_uint32 * 4)(),
                                            a, scale, window, sinks, a, a, n_split, ws, nbytes, None)

    for kw, word in ((dict(window=0), b"window"), (dict(sinks=-1), b"sinks"), (dict(pos0=-1), b"q_pos0"), (dict(scale=0.0), b"sm_scale"),
                     (dict(scale=float("nan")), b"sm_scale"), (dict(q=a + 8), b"16-byte"), (dict(frag=a, rope_pages=0), b"rope_pages"),
                     (dict(n_split=65), b"n_split"), (dict(n_split=4), b"workspace"), (dict(g=_lib.K2bGeom(2, 3, 128, 32, 64, 2, 3, 2, 1)), b"n_q_groups")):
        assert prompt(**kw) == _lib.BMXK_ERR_INVALID and word in lib.bmxk_last_error(), (kw, lib.bmxk_last_error())
    assert lib.bmxk_k2b_rope_fragments(a, a, 0, a, None) == _lib.BMXK_ERR_INVALID
    assert lib.bmxk_k2b_rope_fragments(a, a + 2, 1, a, None) == _lib.BMXK_ERR_INVALID
    from bmx_b200 import kernels as K
    from bmx_b200.engine import K2bLayerState

    cos = torch.zeros(256, D, dtype=torch.float16)
    for kw in (dict(sliding_window=0), dict(sliding_window=5, sinks=-1), dict(sinks=3)):
        with pytest.raises(ValueError):
            K2bLayerState(K.k2b_geom(1, 1), 1, 128, 64, "cpu", cos, cos, **kw)
    with pytest.raises(ValueError):
        K2bLayerState(K.k2b_geom(1, 1, page=64), 1, 128, 64, "cpu", cos, cos, sliding_window=5)
