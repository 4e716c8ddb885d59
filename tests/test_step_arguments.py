"""What the steps under a sliding window and over shared prefixes make of their arguments on the host, before any launch: the library call is
replaced by one that records, so no GPU is needed."""

import contextlib
import ctypes
import warnings

import pytest
import torch

from bmx_b200 import _lib
from bmx_b200 import kernels as K

D = 128


@pytest.fixture
def calls(monkeypatch):
    """The library calls that were made; tensors on the CPU pass for the device's."""
    made = []
    K.v_lut_tensor(K.GAUSSIAN_CODEBOOK[2], "cpu")                 # made by the library once, kept from then on
    monkeypatch.setattr(K, "call", lambda name, *a: made.append((name, a)))
    monkeypatch.setattr(K, "_on_device_of", lambda *ts: contextlib.nullcontext())
    monkeypatch.setattr(K, "_stream", lambda: None)
    monkeypatch.setattr(K, "sm_count", lambda device: 148)
    return made


def _operands(batch=2, h_kv=1, G=4, columns=8, cap=192):
    g = K.k2b_geom(h_kv, G, 128, 16, 64, h_kv)
    cos = torch.zeros(128 * columns, D, dtype=torch.float16)
    win = torch.zeros(batch, h_kv, cap, D, dtype=torch.float16)
    return dict(pool=K.K2bPool(g, 4, "cpu"), basis=torch.zeros(h_kv * D, 16, dtype=torch.float16), table=torch.zeros(batch, columns, dtype=torch.int32),
                n_pages=torch.zeros(batch, dtype=torch.int32), cos=cos, win=win, tail=torch.zeros(batch, dtype=torch.int32),
                lut=K.v_lut_tensor(K.GAUSSIAN_CODEBOOK[2], "cpu"), signs=torch.ones(D), ws=torch.zeros(1 << 16, dtype=torch.uint8))


def _prompt(o, rows, pos0, max_pages, fragments, **kw):
    q = torch.zeros(2, 4, rows, D, dtype=torch.float16)
    rope = None if fragments is None else torch.zeros(fragments, 8192, dtype=torch.int32)
    return K.k2b_prefill_sliding(o["pool"], q, pos0, o["basis"], o["table"], o["n_pages"], max_pages, o["cos"], o["cos"], rope, o["win"], o["win"], o["tail"],
                                 o["lut"], o["signs"], 0.1, o["ws"], 100, 4, **kw)


@pytest.mark.parametrize("rows,pos0,max_pages,enough", [(64, 736, 5, 5), (64, 736, 8, 7), (1, 0, 8, 1), (200, 0, 8, 2), (128, 0, 8, 1), (129, 0, 8, 2), (64, 5000, 6, 6)])
def test_a_prompt_beyond_its_rearranged_tables_draws_a_warning(calls, rows, pos0, max_pages, enough):
    o = _operands()
    for n in (enough, enough + 1, None):
        with warnings.catch_warnings():
            warnings.simplefilter("error")
            _prompt(o, rows, pos0, max_pages, n)
    assert len(calls) == 3 and all(name == "bmxk_k2b_prefill_sliding" for name, _ in calls)
    if enough > 1:
        with pytest.warns(RuntimeWarning, match="left out"):
            _prompt(o, rows, pos0, max_pages, enough - 1)


@pytest.mark.parametrize("G", [3, 5, 6, 7])
def test_prompt_rows_under_a_window_have_no_dense_route(G):
    """None sends the caller to attention over everything held: a state with a window never answers so."""
    from bmx_b200.engine import K2bLayerState

    cos = torch.zeros(256, D, dtype=torch.float16)
    q = torch.zeros(1, G, 5, D, dtype=torch.float16)
    assert K2bLayerState(K.k2b_geom(1, G), 1, 256, 64, "cpu", cos, cos).prefill_attend(q, 0) is None
    with pytest.raises(NotImplementedError):
        K2bLayerState(K.k2b_geom(1, G), 1, 256, 64, "cpu", cos, cos, sliding_window=50, sinks=4).prefill_attend(q, 0)


class _On:
    """Stands for a tensor of a device (None: pinned host memory)."""

    def __init__(self, device, like):
        self.device_index, self.is_cuda = device, device is not None
        self.dtype, self.shape = like.dtype, like.shape

    def is_contiguous(self):
        return True

    def is_pinned(self):
        return True

    def get_device(self):
        return -1 if self.device_index is None else self.device_index


def test_an_output_on_another_device_is_refused():
    like = torch.zeros(2, 4, D, dtype=torch.float16)
    q = _On(1, like)
    for where in (1, None):
        out = _On(where, like)
        assert K._check_out(out, q, (torch.float16,)) is out
    with pytest.raises(RuntimeError, match="different devices: 1 and 0"):
        K._check_out(_On(0, like), q, (torch.float16,))


def _step(which, layout=1, page=128, rank=16, G=4, a=4096, tail_cap=192, **at):
    """A step on made-up addresses that nothing reads; `at` moves operands.  (status, message)."""
    lib, g = _lib.lib(), _lib.K2bGeom(2, G, page, rank, 64, 2, 3, 2, layout)
    p = {k: a + at.get(k, 0) for k in ("q", "basis", "cos", "sin", "k", "v", "out", "ws")}
    head = (ctypes.byref(g), p["q"], a, a, p["basis"], a, 3, a)
    lut, big = (ctypes.c_uint32 * 4)(), 1 << 40
    if which == "plain":
        rc = lib.bmxk_k2b_decode(*head, 2, 3, p["cos"], p["sin"], 0, p["k"], p["v"], a, tail_cap, lut, a, 0.1, p["ws"], big, p["out"], 0, None, 3, None)
    elif which == "sliding":
        rc = lib.bmxk_k2b_decode_sliding(*head, 2, 3, p["cos"], p["sin"], p["k"], p["v"], a, tail_cap, lut, a, 0.1, 100, 4, p["ws"], big, p["out"], 0, None)
    elif which == "shared":
        rc = lib.bmxk_k2b_decode_shared(*head, 2, 3, 2, a, a, a, 0, 0, 1, p["cos"], p["sin"], None, 0, p["k"], p["v"], a, tail_cap, lut, a, 0.1, p["ws"], big,
                                        p["out"], 0, None)
    else:
        rc = lib.bmxk_k2b_prefill_sliding(ctypes.byref(g), p["q"], 8, 0, a, a, p["basis"], a, 3, a, 1, p["cos"], p["sin"], None, 0, p["k"], p["v"], a, tail_cap,
                                          lut, a, 0.1, 100, 4, p["ws"], p["out"], 1, None, 0, None)
    return rc, lib.bmxk_last_error()


@pytest.mark.parametrize("which", ["plain", "sliding", "shared", "prompt"])
@pytest.mark.parametrize("operand,by", [("cos", 2), ("sin", 2), ("basis", 8), ("basis", 2), ("k", 8), ("v", 2)])
def test_operands_that_are_read_by_words_are_aligned(which, operand, by):
    """Whatever a kernel reads by words or 16 bytes at a time is refused elsewhere, not met on the device."""
    rc, message = _step(which, **{operand: by})
    assert rc == _lib.BMXK_ERR_INVALID and b"align" in message, message


def test_64_token_pages_and_status_words_are_aligned_too():
    for operand, by in (("cos", 2), ("basis", 2), ("k", 8)):
        rc, message = _step("plain", layout=0, page=64, **{operand: by})
        assert rc == _lib.BMXK_ERR_INVALID and b"align" in message, message
    rc, message = _step("prompt", ws=1)
    assert rc == _lib.BMXK_ERR_INVALID and b"align" in message, message


@pytest.mark.parametrize("which,G,tail_cap", [("sliding", 8, 9000), ("sliding", 5, 6000), ("sliding", 4, 12000), ("shared", 8, 9000), ("plain", 4, 12000)])
def test_a_window_that_the_merge_cannot_hold_is_refused_before_the_first_launch(which, G, tail_cap):
    rc, message = _step(which, G=G, tail_cap=tail_cap)
    assert rc == _lib.BMXK_ERR_INVALID and b"tail_cap=%d" % tail_cap in message, message


@pytest.mark.parametrize("rows,fine", [(1024, True), (1023, False), (900, False)])
def test_rotation_tables_that_end_inside_a_prefix_are_refused(calls, rows, fine):
    """The prefix kernel reads the row of every position of its pages where the tables are not rearranged."""
    o = _operands()
    groups = K.PrefixGroups(o["pool"].geom, 2, [[0, 1]], [8], "cpu", n_split=1)

    def step(cos, sin):
        K.k2b_decode_shared(o["pool"], torch.zeros(2, 4, D, dtype=torch.float16), o["basis"], o["table"], o["n_pages"], 8, groups, cos, sin, None, o["win"],
                            o["win"], o["tail"], o["lut"], o["signs"], 0.1, o["ws"])

    for cos, sin in ((o["cos"][:rows], o["cos"]), (o["cos"], o["cos"][:rows])):
        if fine:
            step(cos, sin)
        else:
            with pytest.raises(AssertionError, match="8 pages"):
                step(cos, sin)
    assert len(calls) == 2 * fine
