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
