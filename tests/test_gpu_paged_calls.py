"""Calls over a paged cache that go beside the usual ones: batches with entries that cannot be, queries that are not numbers, other streams, captured
calls whose lengths change, calls under the profile."""
import numpy as np
import pytest
import torch

from tests import paged_util as pu
from tests.gpu_util import ctx, host
from tests.test_gpu_paged import SENTINEL, handles

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("wrong", [-5, 0, 10 ** 6])
@pytest.mark.parametrize("many,entry", [(900, 450), (900, 1), (1300, 650), (1300, 325), (1300, 975), (1300, 701), (1300, 1), (1300, 1299), (1300, 1300)])
def test_a_wrong_entry_of_first_costs_the_two_sequences_beside_it_alone(many, entry, wrong):
    """Whatever the number of sequences: those that the entry ends and begins are left out and reported, all others stored.  Entries that a search by
    halving meets first are among them."""
    from heirloom_b200 import cuda
    from heirloom_b200._lib import HeirloomError
    c, dim = ctx(), 64
    b = pu.make([(2, 20)] * many, 1, 1, dim, 16, BF16, spare_rows=5)
    g = torch.Generator("cuda").manual_seed(entry)
    q, k, v = (torch.randn(b.tokens, dim, device="cuda", generator=g).to(BF16) for _ in range(3))
    b.first_dev[entry] = wrong
    left_out = {s for s in (entry - 1, entry) if 0 <= s < many}
    b.k_pages.fill_(SENTINEL)
    b.v_pages.fill_(SENTINEL)
    q_out = torch.full_like(q, SENTINEL)
    cuda.paged_append(c, *handles(b), k, v, q, q_out=q_out)
    with pytest.raises(HeirloomError, match="out-of-range"):
        c.sync()
    want_k, want_q = np.full((*b.k_pages.shape[:2], dim), SENTINEL), np.full(tuple(q.shape), SENTINEL)
    want_v = want_k.copy()
    t, (qn, kn, vn) = np.arange(18, 20), (host(x) for x in (q, k, v))
    for s in set(range(many)) - left_out:
        r, at = b.first[s] + np.arange(2), (b.table[s, t // 16], t % 16)
        want_k[at], want_v[at], want_q[r] = kn[r], vn[r], qn[r]
    assert np.array_equal(host(b.k_pages)[:, :, 0], want_k) and np.array_equal(host(b.v_pages)[:, :, 0], want_v)
    assert np.array_equal(host(q_out), want_q)
