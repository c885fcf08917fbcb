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


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 80), (F32, 64), (F32, 80), (F32, 256)])
@pytest.mark.parametrize("sequences", [[(1, 40), (1, 3000), (1, 1)], [(3, 40), (70, 3000), (9, 9), (2, 1)]], ids=["steps", "chunks"])
def test_a_query_that_is_not_a_number_shows_in_its_own_result_alone(sequences, dtype, dim):
    """Whole rows and those of which several pieces are joined: one head of the last token of every sequence."""
    from heirloom_b200 import cuda
    b = pu.make(sequences, 4, 2, dim, 16, dtype, seed=dim)
    want, want_lse, bound, lse_bound = pu.attention(b)
    spoilt = np.zeros((b.used, 4), bool)
    for s in range(len(sequences)):
        row, head = int(b.first[s + 1]) - 1, s % 4
        b.q[row, head * dim + 3] = float("nan")
        spoilt[row, head] = True
    out, lse = cuda.paged_attention(ctx(), *handles(b), b.q, 4)
    out, lse = host(out).reshape(b.used, 4, dim), host(lse)
    want, bound = want.reshape(out.shape), bound.reshape(out.shape)
    assert np.isnan(out[spoilt]).all() and np.isnan(lse[spoilt]).all()
    assert (np.abs(out - want) <= bound)[~spoilt].all()
    seen = ~spoilt & np.isfinite(want_lse)
    assert (np.abs(lse - np.where(np.isfinite(want_lse), want_lse, 0)) <= lse_bound)[seen].all() and np.isneginf(lse[~spoilt & ~seen]).all()


def test_the_profile_counts_attention_by_what_the_host_knows():
    """Lengths stand on the device: no flops are made up from what the page table could hold, and the bytes are those of queries and results."""
    import ctypes
    from heirloom_b200 import cuda
    from heirloom_b200._lib import Profile
    c = ctx()
    for sequences, dtype in (([(1, 40)] * 3, BF16), ([(200, 300), (1, 5)], BF16), ([(3, 9)], F32)):
        b = pu.make(sequences, 4, 2, 64, 16, dtype, spare_width=500)
        cache, batch = handles(b)
        c.sync()
        cuda.check(c.lib.hl_profile_enable(c.handle, ctypes.c_int(1)))
        try:
            cuda.paged_attention(c, cache, batch, b.q, 4)
            p = Profile()
            cuda.check(c.lib.hl_profile_read(c.handle, ctypes.byref(p)))
        finally:
            cuda.check(c.lib.hl_profile_enable(c.handle, ctypes.c_int(0)))
        assert p.work[1] == 0 and p.scopes[1] == 0  # products of attention
        assert p.scopes[8] == 1 and p.work[8] == b.tokens * 4 * (2 * 64 * b.q.element_size() + 4) and p.ms[8] > 0


@pytest.mark.parametrize("dtype,dim,n,length", [(BF16, 64, 1, 14), (BF16, 128, 1, 9), (BF16, 64, 1, 1500), (F32, 80, 1, 16)])
def test_strides_of_single_rows_and_pages_say_nothing(dtype, dim, n, length):
    """One token, of rows and pages that lie an odd number of elements from where the next ones would."""
    from heirloom_b200 import cuda
    page = 16 if length <= 16 else 2048
    b = pu.make([(n, length)], 2, 1, dim, page, dtype, seed=length, spare_width=0)
    at = int(b.table[0, 0])

    def odd(x):
        wide = torch.full((x[:1].numel() + 1 + 16 // x.element_size(),), float("nan"), dtype=x.dtype, device="cuda")
        t = wide.as_strided(x[:1].shape, (x[0].numel() + 1, *x.stride()[1:]))
        t.copy_(x[:1])
        return t

    b.k_pages, b.v_pages = odd(b.k_pages[at:at + 1]), odd(b.v_pages[at:at + 1])
    b.page_table.fill_(0)
    b.q = odd(b.q)
    want, want_lse, bound, lse_bound = pu.attention(b)
    out, lse = odd(torch.zeros_like(b.q)), odd(torch.zeros(1, 2, device="cuda"))
    cuda.paged_attention(ctx(), *handles(b), b.q, 2, out=out, lse=lse)
    assert (np.abs(host(out) - want) <= bound).all() and (np.abs(host(lse) - want_lse) <= lse_bound).all()
    k, v = (odd(torch.randn(1, dim, device="cuda").to(dtype)) for _ in range(2))
    cuda.paged_append(ctx(), *handles(b), k, v, b.q, q_out=out)
    assert np.array_equal(host(b.k_pages)[0, length - 1, 0], host(k)[0]) and np.array_equal(host(b.v_pages)[0, length - 1, 0], host(v)[0])
    assert np.array_equal(host(out), host(b.q))
    tokens, _ = cuda.sample_rows(ctx(), odd(torch.tensor([[0.0, 9.0, 1.0]], device="cuda")), torch.tensor([0.5], dtype=torch.float64, device="cuda"))
    assert host(tokens).tolist() == [1]
