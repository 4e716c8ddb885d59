"""Steps over shared prefixes and under sliding windows at the edges that the other tests' sizes do not meet: shares without pages."""

import pytest
import torch

from tests import k2b_plain as P

D = 128


def _dev():
    if not torch.cuda.is_available():
        pytest.skip("needs a CUDA device")
    return torch.device("cuda:0")


@pytest.mark.gpu
@pytest.mark.parametrize("pages,split,G,rank,group", [(1, 64, 4, 32, 64), (5, 7, 4, 32, 32), (9, 64, 8, 16, 128), (17, 12, 1, 16, 64), (3, 2, 3, 32, 128)])
def test_a_query_of_nan_stays_in_its_sequence_where_shares_have_no_pages(pages, split, G, rank, group):
    """64 shares of one page, or 7 of five: some of them have none and leave records of zeros, whatever the other rows' queries are.  The
    bits of this NaN are one as fp16 and, in pairs, as float32."""
    from bmx_b200 import kernels as K
    from tests.test_shared_prefix_gpu import World

    w = World(K, _dev(), [(pages, [(0, 30), (1, 64), (0, 0), (0, 190)] * 9)], h_kv=2, G=G, rank=rank, group=group, n_split=split)
    want = w.decode(K)
    P.assert_attention(want, w.ref)
    bad = [3, 8, 20, 35]
    q = w.q.clone()
    q.view(torch.int16)[bad] = 0x7FFF
    good = [b for b in range(q.shape[0]) if b not in bad]
    for _ in range(20):
        out = w.decode(K, q=q)
        assert torch.equal(out[good], want[good])
        assert torch.isnan(out[bad]).all()
    K.check_status(w.ws)
    assert torch.equal(w.decode(K), want)


@pytest.mark.gpu
@pytest.mark.parametrize("report", [2, 3])
def test_a_bounded_wait_runs_its_time_whatever_an_earlier_call_reported(report):
    """A report about a call's arguments (a full window, too few rearranged tables) is none about a wait."""
    from bmx_b200 import kernels as K
    from bmx_b200._lib import BmxkError

    status = torch.zeros(64, dtype=torch.int32, device=_dev())
    status[:3] = torch.tensor([report, 5, 9])
    K.selftest_bounded_wait(status, 2_000_000)
    torch.cuda.synchronize()
    assert status[:4].tolist() == [1, 0, 77, 2]
    with pytest.raises(BmxkError, match="site 77"):
        K.check_status(status.view(torch.uint8))


@pytest.mark.gpu
def test_steps_after_a_reported_prompt_give_what_they_gave_before():
    """Too few rearranged tables for a prompt are reported in the status word of the workspace; the steps that follow on it do not stop at
    their waits (walks of several sequences and heads per CTA, whose basis buffers and stages are waited for)."""
    from bmx_b200 import kernels as K
    from bmx_b200._lib import BmxkError
    from tests import test_shared_prefix_gpu as S
    from tests import test_sliding_gpu as T

    dev = _dev()
    w = T.World(K, dev, [1500, 1500], 700, 4, rows=64, recent=128)
    enough = K.rope_fragments(w.cos, w.sin, w.cos.shape[0] // 128)
    want = w.prompt(K, enough)
    step = T.World(K, dev, [700, 1500, 900, 130, 2000] * 12, 10 ** 9, 0, h_kv=5)
    slid = step.decode(K)
    plain = (step.basis, step.table, step.n_pages, step.max_pages, step.cos, step.sin, step.k_win, step.v_win, step.tail_len, step.v_lut, step.signs, D ** -0.5)
    q = step.q[:, :, 0].contiguous()
    streamed = K.k2b_decode(step.pool, q, *plain, step.ws)
    shared = S.World(K, dev, [(40, [(3, 40), (1, 130), (0, 7), (5, 60)] * 20)], h_kv=4)
    joined = shared.decode(K)
    for ws in (w.ws, step.ws, shared.ws):
        w.ws = ws
        w.prompt(K, enough[:2])
        for _ in range(3):
            assert torch.equal(w.prompt(K, enough), want)
            if ws is step.ws:
                assert torch.equal(K.k2b_decode(step.pool, q, *plain, ws), streamed)
                assert torch.equal(step.decode(K), slid)
            if ws is shared.ws:
                assert torch.equal(shared.decode(K), joined)
        with pytest.raises(BmxkError, match="rotation tables"):
            K.check_status(ws)
