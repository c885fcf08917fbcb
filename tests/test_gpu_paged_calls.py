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
@pytest.mark.parametrize("many,entry", [(900, 450), (900, 1), (1300, 650), (1300, 325), (1300, 975), (1300, 701), (1300, 1), (1300, 1299), (1300, 1300), (5000, 2500), (5000, 4999)])
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


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 48)])
@pytest.mark.parametrize("sequences", [[(1, 40), (1, 1500)], [(90, 1500), (1, 7)]], ids=["steps", "chunks"])
@pytest.mark.parametrize("own_buffers", [True, False])
def test_calls_under_another_current_stream(sequences, dtype, dim, own_buffers):
    """Inputs that another stream is still making when the call is issued, and results that it takes: the calls run on the context's stream, which is
    told to wait, as the other one is afterwards."""
    from heirloom_b200 import cuda
    c = ctx()
    b = pu.make(sequences, 4, 2, dim, 16, dtype, seed=dim)
    want, _, bound, _ = pu.attention(b)
    cache, batch = handles(b)
    late = torch.empty_like(b.q)
    k = torch.randn(b.tokens, 2 * dim, device="cuda").to(dtype)
    logits = torch.randn(3, 5000, device="cuda")
    late_logits, draws = torch.empty_like(logits), torch.rand(3, dtype=torch.float64, device="cuda")
    chosen = cuda.sample_rows(c, logits, draws, top_k=torch.full((3,), 700, dtype=torch.int32, device="cuda"))
    top_k = torch.full((3,), 700, dtype=torch.int32, device="cuda")
    work = torch.empty(cuda.paged_attention_workspace(c, dtype, 4, 2, dim), dtype=torch.uint8, device="cuda")
    given = [torch.empty_like(b.q), torch.empty_like(b.q), torch.empty(b.tokens, 4, device="cuda"), torch.empty(3, dtype=torch.int64, device="cuda"),
             torch.empty(3, device="cuda")]
    other = torch.cuda.Stream()
    other.wait_stream(c.stream)
    with torch.cuda.stream(other):
        torch.cuda._sleep(20_000_000)  # ten milliseconds
        late.copy_(b.q)
        late_logits.copy_(logits)
        c.stream.wait_stream(other)
        if own_buffers:
            q, out, lse, tokens, chances = given
            cuda.paged_attention(c, cache, batch, late, 4, out=out, lse=lse, workspace=work)
            cuda.paged_append(c, cache, batch, k, k, late, q_out=q)
            cuda.sample_rows(c, late_logits, draws, top_k=top_k, tokens=tokens, probabilities=chances)
        else:
            out, lse = cuda.paged_attention(c, cache, batch, late, 4)
            q = cuda.paged_append(c, cache, batch, k, k, late)
            tokens, chances = cuda.sample_rows(c, late_logits, draws, top_k=top_k)
        other.wait_stream(c.stream)
        got = [x.clone() for x in (out, q, tokens, chances)]
    c.stream.wait_stream(other)
    out, q, tokens, chances = map(host, got)
    assert (np.abs(out - want) <= bound).all() and np.array_equal(q, host(b.q))
    assert np.array_equal(tokens, host(chosen[0])) and np.array_equal(chances, host(chosen[1]))


def recast(b, sequences):
    """The batch with other new tokens and lengths, no longer than those that it was made with, written where they stand."""
    first = np.concatenate([[0], np.cumsum([n for n, _ in sequences])]).astype(np.int32)
    b.sequences, b.first, b.used = sequences, first, int(first[-1])
    b.lengths.copy_(torch.tensor([length for _, length in sequences], dtype=torch.int32))
    if b.first_dev is not None:
        b.first_dev.copy_(torch.from_numpy(first))


GRAPHS = {
    "steps": ([(1, 3000), (1, 1200), (1, 5000)], [[(1, 1), (1, 1200), (1, 4999)], [(1, 3000), (1, 0), (1, 17)], [(1, 64), (1, 65), (1, 66)], [(1, 0)] * 3]),
    "chunks": ([(200, 3000), (1, 1200), (40, 5000)], [[(1, 1), (40, 40), (200, 4999)], [(0, 0), (200, 1200), (1, 17)], [(129, 129), (1, 1100), (70, 2049)],
                                                      [(5, 2), (0, 40), (0, 0)]]),
}


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("kind", GRAPHS)
def test_captured_calls_follow_the_lengths_that_stand_there(kind, dtype, dim):
    """Tables of more than a thousand positions: work is dealt out and pieces are joined anew at every replay.  Two graphs in turn and, at last, both at
    once on streams of their own, each with the workspace of its capture."""
    from heirloom_b200 import cuda
    c = ctx()
    start, others = GRAPHS[kind]
    b = pu.make(start, 4, 2, dim, 16, dtype, seed=dim, spare_rows=4 if kind == "chunks" else 0, with_first=kind == "chunks")
    cache, batch = handles(b)
    out, lse = [torch.empty_like(b.q) for _ in range(2)], [torch.empty(b.tokens, 4, device="cuda") for _ in range(2)]
    cuda.paged_attention(c, cache, batch, b.q, 4, out=out[0], lse=lse[0])
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for graph, o, s in zip(graphs, out, lse):
        with torch.cuda.graph(graph, stream=c.stream):
            cuda.paged_attention(c, cache, batch, b.q, 4, out=o, lse=s)

    def compare(i):
        want, want_lse, bound, lse_bound = pu.attention(b)
        got, got_lse, blind = host(out[i]), host(lse[i]), np.isneginf(want_lse)
        assert (np.abs(got[:b.used] - want) <= bound).all() and (got[b.used:] == SENTINEL).all() and (got_lse[b.used:] == SENTINEL).all()
        assert np.array_equal(np.isneginf(got_lse[:b.used]), blind)
        assert (np.abs(np.where(blind, 0, got_lse[:b.used]) - np.where(blind, 0, want_lse)) <= lse_bound).all()

    for step, sequences in enumerate([start, *others]):
        recast(b, sequences)
        i = step % 2
        out[i].fill_(SENTINEL)
        lse[i].fill_(SENTINEL)
        graphs[i].replay()
        c.sync()
        compare(i)
    recast(b, start)
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i in range(2):
        out[i].fill_(SENTINEL)
        lse[i].fill_(SENTINEL)
    for graph, stream in zip(graphs, streams):
        stream.wait_stream(c.stream)
        with torch.cuda.stream(stream):
            for _ in range(20):
                graph.replay()
    torch.cuda.synchronize()
    compare(0)
    compare(1)


@pytest.mark.parametrize("last", [2000, 131072, (1 << 24) - 1])
def test_sines_are_off_by_their_own_rounding(last):
    """Channel pairs (1, 0) and (0, 1), which a rotation turns into its cosine and sine."""
    from heirloom_b200 import cuda
    n, pairs, page = 997, 32, 1 << 16
    step = last // n
    positions = (np.arange(n) + 1) * step
    table = torch.zeros(n, -(-(last + 1) // page), dtype=torch.int32, device="cuda")
    pages = torch.zeros(1, page, 1, 64, device="cuda")
    lengths = torch.tensor(positions + 1, dtype=torch.int32, device="cuda")
    f = torch.tensor(10000.0 ** (-np.arange(pairs) / pairs), dtype=F32, device="cuda")
    batch = cuda.PagedBatch(table, lengths)
    x = torch.zeros(n, 2 * 64, device="cuda")
    x[:, :pairs], x[:, 64 + pairs:] = 1.0, 1.0  # two heads
    q = host(cuda.paged_append(ctx(), cuda.PagedCache(pages, pages.clone()), batch, x[:, :64].contiguous(), x[:, :64].contiguous(), x, f))
    angle = positions.astype(np.longdouble)[:, None] * f.double().cpu().numpy()
    want = np.concatenate([np.cos(angle), np.sin(angle), -np.sin(angle), np.cos(angle)], 1)
    # an ulp of the function, 2^-24 below 1, and the rounding of the correction; products with 0 and 1 are exact.  The angle in turns is a product of 64 bits: off by
    # 2^-53 of itself and, reduced, as much again
    off = 1.5 * 2.0 ** -24 + 2 * np.abs(angle) * 2.0 ** -53
    assert (np.abs(q - want) <= np.tile(off, 4)).all(), float((np.abs(q - want) * 2.0 ** 24).max())


@pytest.mark.parametrize("heads_first", [False, True])
def test_offsets_beyond_32_bits(heads_first):
    """Caches of more than 2^32 elements a tensor, sequences in their last pages; rows of logits and of queries as far apart."""
    from heirloom_b200 import cuda
    page, kv_heads, dim = 256, 4, 128
    pages = (1 << 32) // (page * kv_heads * dim) + 40
    shape = (pages, kv_heads, page, dim) if heads_first else (pages, page, kv_heads, dim)
    try:
        k, v = (torch.empty(shape, dtype=BF16, device="cuda") for _ in range(2))
        if heads_first:
            k, v = k.transpose(1, 2), v.transpose(1, 2)
        for sequences in ([(1, 300), (1, 2000), (1, 1)], [(150, 300), (40, 2000), (1, 1)], [(1, 700), (1, 3)]):
            b = pu.make(sequences, 8, kv_heads, dim, page, BF16, seed=len(sequences))
            offset = pages - b.k_pages.shape[0]
            k[offset:], v[offset:] = b.k_pages, b.v_pages
            used = torch.from_numpy((b.table >= 0) & (b.table < b.k_pages.shape[0])).cuda()
            b.page_table = torch.where(used, b.page_table + offset, b.page_table)
            b.table = np.where(used.cpu().numpy(), b.table + offset, b.table)
            b.k_pages, b.v_pages = k, v
            out, lse = cuda.paged_attention(ctx(), *handles(b), b.q, 8)
            want, want_lse, bound, lse_bound = pu.attention(b)
            assert (np.abs(host(out) - want) <= bound).all() and (np.abs(host(lse) - want_lse) <= lse_bound).all()
            x, y = (torch.randn(b.tokens, kv_heads * dim, device="cuda").to(BF16) for _ in range(2))
            cuda.paged_append(ctx(), *handles(b), x, y)
            for s, (n, length) in enumerate(sequences):
                t = np.arange(length - n, length)
                at = torch.from_numpy(b.table[s, t // page]).cuda().long(), torch.from_numpy(t % page).cuda()
                rows = slice(int(b.first[s]), int(b.first[s + 1]))
                assert torch.equal(k[at].reshape(n, -1), x[rows]) and torch.equal(v[at].reshape(n, -1), y[rows])
    finally:
        k = v = b = None
        torch.cuda.empty_cache()
    if heads_first:
        return
    # rows 2^31 elements and more apart
    wide = torch.empty(3, (1 << 31) + 8, dtype=BF16, device="cuda")
    q = wide[:, 8:8 + 4 * 64]
    for sequences in ([(1, 40), (1, 1300), (1, 7)], [(3, 50)]):
        b = pu.make(sequences, 4, 2, 64, 16, BF16, seed=1)
        q.copy_(b.q)
        got, _ = cuda.paged_attention(ctx(), *handles(b), q, 4, out=wide[:, 1024:1024 + 4 * 64])
        want, _, bound, _ = pu.attention(b)
        assert (np.abs(host(got) - want) <= bound).all()
    logits = torch.randn(3, 5000, device="cuda").to(BF16)
    wide[:, 16:5016] = logits
    draws, controls = torch.rand(3, dtype=torch.float64, device="cuda"), dict(top_p=torch.full((3,), 0.9, device="cuda"))
    far, near = cuda.sample_rows(ctx(), wide[:, 16:5016], draws, **controls), cuda.sample_rows(ctx(), logits, draws, **controls)
    assert np.array_equal(host(far[0]), host(near[0])) and np.array_equal(host(far[1]), host(near[1]))
    wide = q = got = far = None
    torch.cuda.empty_cache()


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 80)])
def test_two_contexts_at_once(dtype, dim):
    """A stream, and a kept workspace, each: calls that overlap."""
    from heirloom_b200 import cuda
    c = ctx()
    other = cuda.Context(0)
    try:
        batches = [pu.make(s, 4, 2, dim, 16, dtype, seed=i) for i, s in enumerate(([(1, 3000), (1, 500)], [(60, 3000), (1, 1200)]))]
        made = [handles(b) for b in batches]
        torch.cuda.synchronize()
        results = [[], []]
        for _ in range(10):
            for i, x in enumerate((c, other)):
                results[i].append(cuda.paged_attention(x, *made[i], batches[i].q, 4))
        torch.cuda.synchronize()
        for b, got in zip(batches, results):
            want, _, bound, _ = pu.attention(b)
            for out, _ in got:
                assert (np.abs(out.double().cpu().numpy() - want) <= bound).all()
    finally:
        torch.cuda.synchronize()
        other.close()


@pytest.mark.parametrize("dtype,dim,pairs", [(BF16, 80, 20), (BF16, 128, 4), (BF16, 64, 12), (BF16, 256, 124), (F32, 80, 10), (F32, 64, 2), (F32, 8, 2)])
@pytest.mark.parametrize("sequences", [[(1, 1)], [(1, 17), (1, 0), (1, 1023)], [(1, 90), (37, 300), (0, 4), (130, 131), (3, 1)]], ids=["one", "steps", "mixed"])
def test_halves_of_turned_channels_that_end_within_16_bytes(sequences, dtype, dim, pairs):
    from tests.test_gpu_paged import check_append, inverse
    for more in (dict(), dict(strided=True, in_place=True), dict(with_q=False)):
        check_append(pu.make(sequences, 6, 2, dim, 16, dtype, spare_rows=2, seed=dim), inverse(pairs), False, **more)
