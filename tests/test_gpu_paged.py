"""The paged cache on the GPU: appending with rotation, attention over it, against the formulas in 64 bits."""
import numpy as np
import pytest
import torch

from tests import paged_util as pu
from tests.gpu_util import ctx, host

pytestmark = pytest.mark.gpu
BF16, F32 = torch.bfloat16, torch.float32
SENTINEL = 7.0


def handles(b, max_length=0):
    from heirloom_b200 import cuda
    return cuda.PagedCache(b.k_pages, b.v_pages), cuda.PagedBatch(b.page_table, b.lengths, b.first_dev, b.tokens, b.max_new, max_length)


def attend(b, max_length=0, **more):
    from heirloom_b200 import cuda
    cache, batch = handles(b, max_length)
    out = torch.full((b.tokens, b.heads * b.dim), SENTINEL, dtype=b.dtype, device="cuda")
    lse = torch.full((b.tokens, b.heads), SENTINEL, device="cuda")
    got = cuda.paged_attention(ctx(), cache, batch, b.q, b.heads, out=out, lse=lse, **more)
    return host(got[0]), host(got[1])


def check_attention(b, scale=None, **more):
    out, lse = attend(b, scale=scale, **more)
    want, want_lse, bound, lse_bound = pu.attention(b, scale)
    assert (out[b.used:] == SENTINEL).all() and (lse[b.used:] == SENTINEL).all()  # rows of no sequence
    out, lse = out[:b.used], lse[:b.used]
    blind = np.isneginf(want_lse)
    assert np.array_equal(np.isneginf(lse), blind)
    off = np.abs(out - want)
    assert np.isfinite(out).all() and (off <= bound).all(), (off - bound).max()
    off = np.abs(np.where(blind, 0, lse) - np.where(blind, 0, want_lse))
    assert (off <= lse_bound).all(), (off - lse_bound).max()


STEPS = [(1, 1), (1, 17), (1, 0), (1, 200), (1, 64), (1, 65), (1, 1023), (1, 16), (1, 2)]
MIXED = [(1, 90), (5, 5), (0, 40), (37, 300), (0, 0), (130, 131), (3, 1), (64, 64), (1, 0), (200, 513), (2, 129)]


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (BF16, 32), (BF16, 80), (BF16, 256), (F32, 64), (F32, 8), (F32, 80), (F32, 256)])
@pytest.mark.parametrize("heads,kv_heads", [(3, 3), (8, 2), (10, 2), (20, 1)])
@pytest.mark.parametrize("sequences", [STEPS, MIXED], ids=["steps", "mixed"])
def test_attention_of_ragged_batches(sequences, heads, kv_heads, dtype, dim):
    check_attention(pu.make(sequences, heads, kv_heads, dim, 16, dtype, seed=dim + heads, spare_rows=3))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 96)])
@pytest.mark.parametrize("page", [16, 32, 64, 128, 256, 1024])
@pytest.mark.parametrize("heads_first", [False, True])
def test_attention_of_page_sizes_and_layouts(page, heads_first, dtype, dim):
    for seed, sequences in enumerate(([(1, 333), (1, 1025), (1, 31)], [(70, 333), (257, 1025), (31, 31), (1, 500)])):
        check_attention(pu.make(sequences, 4, 2, dim, page, dtype, heads_first, seed=seed))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("sequences", [[(1, 40000)], [(1, 5), (1, 30000), (1, 0), (1, 9000)], [(9, 20000), (1, 3)], [(300, 9000)]],
                         ids=["one", "uneven", "few", "chunk"])
def test_attention_of_long_sequences_that_many_streams_share(sequences, dtype, dim):
    check_attention(pu.make(sequences, 4, 1, dim, 32, dtype, seed=3))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("n", [1, 2, 15, 16, 17, 31, 32, 33, 127, 128, 129])
def test_attention_of_every_number_of_rows(n, dtype):
    for group in (1, 3, 8):
        check_attention(pu.make([(n, n), (n, n + 1), (n, n + 127)], group * 2, 2, 64, 16, dtype, seed=n))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
def test_attention_with_scores_of_all_sizes(dtype, dim):
    """Scores far apart, rising and falling along the keys, so that maxima are raised by far more than 2^8; a scale of the caller's."""
    for seed, scale in ((1, None), (2, 1.0)):
        for sequences in ([(1, 700), (1, 90)], [(50, 700), (140, 300)]):
            b = pu.make(sequences, 4, 2, dim, 16, dtype, seed=seed)
            for s, (n, length) in enumerate(sequences):
                k = b.stored[s][0]
                k *= np.abs(np.sin(np.arange(length) / 37.0))[:, None, None] * 6
                k[:] = torch.from_numpy(k).to(dtype).double().numpy()
                t = torch.arange(length)
                page = torch.from_numpy(b.table[s].astype(np.int64))[t // b.page]
                b.k_pages[page.cuda(), (t % b.page).cuda()] = torch.from_numpy(k).to("cuda", dtype)
            check_attention(b, scale=scale)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 80)])
def test_attention_without_first_without_lse_and_with_a_bound_on_lengths(dtype, dim):
    from heirloom_b200 import cuda
    b = pu.make(STEPS, 6, 3, dim, 16, dtype, with_first=False, spare_width=40)
    check_attention(b, max_length=1023)
    cache, batch = handles(b)
    want = attend(b)[0]
    out = torch.empty(b.tokens, b.heads * dim, dtype=dtype, device="cuda")
    c = ctx()
    size = cuda.paged_attention_workspace(c, dtype, b.heads, b.kv_heads, dim)
    work = torch.full((size,), 255, dtype=torch.uint8, device="cuda")  # NaN: it needs no clearing
    import ctypes
    rc = c.lib.hl_paged_attention(c.handle, ctypes.byref(cache.desc), ctypes.byref(batch.desc), ctypes.c_void_p(b.q.data_ptr()), ctypes.c_longlong(b.heads * dim),
                                  ctypes.c_void_p(out.data_ptr()), ctypes.c_longlong(b.heads * dim), None, ctypes.c_int(b.heads),
                                  ctypes.c_float(dim ** -0.5), ctypes.c_void_p(work.data_ptr()), ctypes.c_size_t(size))
    assert rc == 0 and np.array_equal(host(out), want)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
def test_attention_of_strided_rows_and_caches(dtype, dim):
    """Queries and results as columns of wider buffers, keys and values as halves of one, pages and heads with gaps between them."""
    for sequences in (STEPS, MIXED):
        b = pu.make(sequences, 4, 2, dim, 16, dtype, seed=5)
        pages = b.k_pages.shape[0]
        both = torch.full((pages, 2, 16, 3, dim + 16), float("nan"), dtype=dtype, device="cuda")
        both[:, 0, :, :2, :dim], both[:, 1, :, :2, :dim] = b.k_pages, b.v_pages
        b.k_pages, b.v_pages = both[:, 0, :, :2, :dim], both[:, 1, :, :2, :dim]
        wide = torch.full((b.tokens, 3 * 4 * dim), float("nan"), dtype=dtype, device="cuda")
        wide[:, 4 * dim:8 * dim] = b.q
        b.q = wide[:, 4 * dim:8 * dim]
        out = torch.full((b.tokens, 8 * dim), SENTINEL, dtype=dtype, device="cuda")
        from heirloom_b200 import cuda
        got, _ = cuda.paged_attention(ctx(), *handles(b), b.q, 4, out=out[:, 8 * dim // 2:])
        want, _, bound, _ = pu.attention(b)
        assert (np.abs(host(got)[:b.used] - want) <= bound).all() and (host(out)[:, :4 * dim] == SENTINEL).all()


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
def test_attention_gives_the_same_bits_again_and_on_a_used_workspace(dtype, dim):
    from heirloom_b200 import cuda
    c = ctx()
    work = torch.empty(cuda.paged_attention_workspace(c, dtype, 4, 2, dim), dtype=torch.uint8, device="cuda")
    for sequences in ([(1, 3000), (1, 77)], [(200, 3000), (1, 1000)]):
        b = pu.make(sequences, 4, 2, dim, 16, dtype)
        first = attend(b, workspace=work)
        work.fill_(255)
        again = attend(b, workspace=work)
        assert all(np.array_equal(x, y) for x, y in zip(first, again))


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (BF16, 128), (F32, 64)])
@pytest.mark.parametrize("sequences", [[(1, 3000), (1, 500)], [(200, 3000), (1, 700)]], ids=["steps", "chunks"])
def test_attention_without_lse_where_pieces_are_joined(sequences, dtype, dim):
    import ctypes
    from heirloom_b200 import cuda
    c, b = ctx(), pu.make(sequences, 4, 2, dim, 64, dtype)
    cache, batch = handles(b)
    want = attend(b)[0]
    out = torch.full((b.tokens, 4 * dim), SENTINEL, dtype=dtype, device="cuda")
    work = torch.empty(cuda.paged_attention_workspace(c, dtype, 4, 2, dim), dtype=torch.uint8, device="cuda")
    assert c.lib.hl_paged_attention(c.handle, cache.address, batch.address, b.q.data_ptr(), 4 * dim, out.data_ptr(), 4 * dim, None, 4, dim ** -0.5,
                                    work.data_ptr(), work.numel()) == 0
    assert np.array_equal(host(out), want)


@pytest.mark.parametrize("dtype,dim", [(BF16, 64), (F32, 48)])
@pytest.mark.parametrize("new", [1, 2, 21])
def test_thousands_of_sequences(new, dtype, dim):
    """More than a block's threads, of all lengths, some empty; without `first` where each has one token."""
    rng = np.random.default_rng(new)
    many = 1500
    n = np.full(many, 1) if new == 1 else rng.integers(0, new + 1, many)
    sequences = [(int(a), int(a + rng.integers(0, 60)) if i % 7 else 0) for i, a in enumerate(n)]
    for with_first in ((True, False) if new == 1 else (True,)):
        b = pu.make(sequences, 2, 1, dim, 16, dtype, seed=new, with_first=with_first)
        check_attention(b)
        check_append(b, inverse(dim // 2), False)


def test_attention_reports_what_it_cannot_follow_and_leaves_it_out():
    """A length beyond its bound, `first` that falls, pages that the cache does not have: reported once, nothing else disturbed."""
    from heirloom_b200 import cuda
    from heirloom_b200._lib import HeirloomError
    c = ctx()
    for dtype, dim in ((BF16, 64), (BF16, 128), (F32, 64)):
        for sequences in ([(1, 40), (1, 50), (1, 60)], [(20, 40), (30, 50), (1, 60)]):
            b = pu.make(sequences, 2, 2, dim, 16, dtype)
            want, _, bound, _ = pu.attention(b)
            good = slice(0, int(b.first[1])), slice(int(b.first[2]), b.used)
            b.lengths[1] = 1000
            with pytest.raises(HeirloomError, match="out-of-range"):
                attend(b)
            c.sync()
            out = torch.full((b.tokens, 2 * dim), SENTINEL, dtype=dtype, device="cuda")
            cuda.paged_attention(c, *handles(b), b.q, 2, out=out)
            with pytest.raises(HeirloomError, match="out-of-range"):
                c.sync()
            got = host(out)
            assert all((np.abs(got[r] - want[r]) <= bound[r]).all() for r in good) and (got[int(b.first[1]):int(b.first[2])] == SENTINEL).all()
            b.lengths[1] = 50
            b.page_table[1, 0] = b.k_pages.shape[0]
            out.fill_(SENTINEL)
            cuda.paged_attention(c, *handles(b), b.q, 2, out=out)
            with pytest.raises(HeirloomError, match="out-of-range"):
                c.sync()
            got = host(out)
            assert all((np.abs(got[r] - want[r]) <= bound[r]).all() for r in good) and np.isfinite(got).all()


# ---- appending --------------------------------------------------------------------------------------------------------------
def check_append(b, frequencies, interleaved, strided=False, in_place=False, with_q=True):
    from heirloom_b200 import cuda
    rng = np.random.default_rng(len(b.sequences))
    wide, dim, dtype = b.kv_heads * b.dim, b.dim, b.dtype
    rows = torch.from_numpy(rng.standard_normal((b.tokens, b.heads * dim + 2 * wide))).to("cuda", dtype)
    q, k, v = rows[:, :b.heads * dim], rows[:, b.heads * dim:b.heads * dim + wide], rows[:, b.heads * dim + wide:]
    if not strided:
        q, k, v = q.contiguous(), k.contiguous(), v.contiguous()
    qn, kn, vn = (host(x).reshape(b.tokens, -1, dim) for x in (q, k, v))
    b.k_pages.fill_(SENTINEL)
    b.v_pages.fill_(SENTINEL)
    q_out = q if in_place else torch.full((b.tokens, b.heads * dim), SENTINEL, dtype=dtype, device="cuda")
    f = torch.tensor(frequencies, dtype=F32, device="cuda")
    got = cuda.paged_append(ctx(), *handles(b), k, v, q if with_q else None, f, interleaved, q_out=q_out if with_q else None)
    want_k = np.full(tuple(b.k_pages.shape), SENTINEL)
    want_v = want_k.copy()
    # a rotation is two products and a sum of f32 (3 u of |x| + |y|) with a sine and cosine off by 2^-22 (their own rounding and the angle's); bf16
    # and f32 results are rounded once
    bound_k, half = np.zeros_like(want_k), 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    fr = f.double().cpu().numpy()
    for s, (n, length) in enumerate(b.sequences):
        r, t = b.first[s] + np.arange(n), length - n + np.arange(n)
        if with_q:
            want = pu.rotate(qn[r], t.clip(0), fr, interleaved)
            size = np.abs(qn).max()
            assert (np.abs(host(got).reshape(b.tokens, -1, dim)[r] - want) <= half * np.abs(want) + 4 * 2.0 ** -22 * size).all()
        r, t = r[t >= 0], t[t >= 0]
        at = b.table[s, t // b.page], t % b.page
        want_k[at], want_v[at] = pu.rotate(kn[r], t, fr, interleaved), vn[r]
        bound_k[at] = half * np.abs(want_k[at]) + 4 * 2.0 ** -22 * np.abs(kn).max()
    assert (np.abs(host(b.k_pages) - want_k) <= bound_k).all() and np.array_equal(host(b.v_pages), want_v)
    if with_q:  # rows of no sequence
        rest = host(got).reshape(b.tokens, -1, dim)[b.used:]
        assert np.array_equal(rest, qn[b.used:]) if in_place else (rest == SENTINEL).all()


def inverse(pairs):
    return 10000.0 ** (-np.arange(pairs) / max(1, pairs))


@pytest.mark.parametrize("dtype,dim,pairs,interleaved", [
    (BF16, 64, 32, False), (BF16, 128, 64, False), (BF16, 128, 64, True), (BF16, 64, 0, False), (BF16, 80, 16, False), (BF16, 80, 13, True), (BF16, 256, 128, False),
    (F32, 64, 32, False), (F32, 80, 20, True), (F32, 8, 4, False), (F32, 256, 128, True), (F32, 96, 20, False)])
@pytest.mark.parametrize("sequences", [STEPS, MIXED, [(1, 1)], [(3000, 3001)]], ids=["steps", "mixed", "one", "long"])
def test_append(sequences, dtype, dim, pairs, interleaved):
    check_append(pu.make(sequences, 4, 2, dim, 16, dtype, spare_rows=2, seed=dim), inverse(pairs), interleaved)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("heads_first,page", [(False, 64), (True, 16), (True, 256)])
def test_append_of_columns_in_place_without_queries_and_in_other_layouts(dtype, heads_first, page):
    for more in (dict(strided=True), dict(in_place=True), dict(with_q=False), dict(strided=True, in_place=True)):
        check_append(pu.make(MIXED, 6, 3, 64, page, dtype, heads_first, spare_rows=1), inverse(32), False, **more)
    check_append(pu.make(STEPS, 6, 3, 64, page, dtype, heads_first, with_first=False), inverse(16), True)


def test_append_of_many_sequences_leaves_out_what_cannot_be():
    from heirloom_b200 import cuda
    from heirloom_b200._lib import HeirloomError
    c = ctx()
    b = pu.make([(2, 20)] * 1300, 2, 1, 64, 16, BF16)
    x = torch.randn(b.tokens, 64, device="cuda").to(BF16)
    for spoil in (lambda: b.lengths[700].fill_(10 ** 6), lambda: b.page_table[700].fill_(-3), lambda: b.first_dev[701].fill_(10 ** 6),
                  lambda: b.first_dev[701].fill_(-5)):
        table, lengths, first = b.page_table.clone(), b.lengths.clone(), b.first_dev.clone()
        spoil()
        b.v_pages.fill_(SENTINEL)
        cuda.paged_append(c, *handles(b), x, x)
        with pytest.raises(HeirloomError, match="out-of-range"):
            c.sync()
        written = (host(b.v_pages) != SENTINEL).any(-1)[..., 0]
        t = np.arange(18, 20)
        for s in range(1300):  # a spoilt entry of `first` is the end of one sequence and the start of the next, and may mislead the search for others
            if s in (700, 701):
                continue
            if abs(s - 700) < 50 or s % 13 == 0:
                at = written[b.table[s, t // 16], t % 16]
                assert at.all() or (spoil.__code__.co_consts[1] == 701), s
        assert written.sum() <= 2 * 1300 and not written[b.table[700, 1], :2].all()
        b.page_table.copy_(table)
        b.lengths.copy_(lengths)
        b.first_dev.copy_(first)


def test_append_at_far_positions():
    """Angles of positions near 2^30, where an f32 product would be off by whole turns; only the pages that are used exist."""
    from heirloom_b200 import cuda
    page, length = 1 << 20, (1 << 30) - 5
    width = -(-length // page)
    table = torch.full((1, width), -1, dtype=torch.int32, device="cuda")
    table[0, -1] = 0
    k_pages = torch.zeros(1, page, 1, 8, device="cuda")
    v_pages = torch.zeros_like(k_pages)
    x = torch.randn(3, 8, device="cuda", generator=torch.Generator("cuda").manual_seed(1))
    f = torch.tensor([1.0, 0.37, 0.011, 1e-4], device="cuda")
    batch = cuda.PagedBatch(table, torch.tensor([length], dtype=torch.int32, device="cuda"), torch.tensor([0, 3], dtype=torch.int32, device="cuda"), 3, 3)
    q = cuda.paged_append(ctx(), cuda.PagedCache(k_pages, v_pages), batch, x, x, x, f)
    t = length - 3 + np.arange(3)
    want = pu.rotate(host(x).reshape(3, 1, 8), t, f.double().cpu().numpy(), False)
    # the turns, below 2^28, are two products of 64 bits: off by 2^-24 of a turn or 2^-21.3 of a radian; the rest is f32
    assert (np.abs(host(q).reshape(3, 1, 8) - want) <= 2.0 ** -19 * np.abs(host(x)).max()).all()
    assert np.array_equal(host(k_pages)[0, t % page, 0], host(q)) and np.array_equal(host(v_pages)[0, t % page, 0], host(x))


def test_append_reports_what_it_cannot_follow_and_writes_nothing_there():
    from heirloom_b200 import cuda
    from heirloom_b200._lib import HeirloomError
    c = ctx()
    b = pu.make([(1, 20), (3, 40), (2, 7)], 2, 1, 64, 16, BF16)
    x = torch.randn(b.tokens, 64, device="cuda").to(BF16)
    for spoil, good in ((lambda: b.page_table[1].fill_(b.k_pages.shape[0]), (0, 2)), (lambda: b.page_table[1].fill_(-3), (0, 2)),
                        (lambda: b.lengths[1].fill_(10 ** 6), (0, 2)), (lambda: b.lengths[1].fill_(-1), (0, 2)),
                        (lambda: b.first_dev[1].fill_(100), (2,))):  # the end of one and the start of the next
        table, lengths, first = b.page_table.clone(), b.lengths.clone(), b.first_dev.clone()
        spoil()
        b.k_pages.fill_(SENTINEL)
        b.v_pages.fill_(SENTINEL)
        cuda.paged_append(c, *handles(b), x, x)
        with pytest.raises(HeirloomError, match="out-of-range"):
            c.sync()
        c.sync()
        wanted = np.zeros((b.k_pages.shape[0], 16), bool)
        for s in good:
            n, length = b.sequences[s]
            t = length - n + np.arange(n)
            wanted[b.table[s, t // 16], t % 16] = True
        for pages in (b.k_pages, b.v_pages):
            assert np.array_equal((host(pages) != SENTINEL).any(-1)[..., 0], wanted)
        b.page_table.copy_(table)
        b.lengths.copy_(lengths)
        b.first_dev.copy_(first)


def test_calls_follow_their_context_whatever_device_and_stream_are_current():
    """Another stream of the caller's, ordered by events, changes nothing."""
    b = pu.make(STEPS, 4, 2, 64, 16, BF16)
    want = attend(b)
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        cache_batch = handles(b)
    ctx().stream.wait_stream(other)
    from heirloom_b200 import cuda
    out, lse = cuda.paged_attention(ctx(), *cache_batch, b.q, b.heads)
    assert np.array_equal(host(out), want[0]) and np.array_equal(host(lse), want[1])


# ---- a server's steps -------------------------------------------------------------------------------------------------------
class Server:
    """One layer and a head over a paged cache: rotated keys, attention, logits, a token a sequence."""

    def __init__(self, dtype, heads, kv_heads, dim, vocab, page, pages, seed):
        from heirloom_b200 import cuda
        g = torch.Generator("cuda").manual_seed(seed)
        self.dtype, self.heads, self.kv_heads, self.dim, self.page = dtype, heads, kv_heads, dim, page
        width = (heads + 2 * kv_heads) * dim
        self.embedding = (torch.randn(vocab, width, device="cuda", generator=g)).to(dtype)  # q, k and v of a token
        self.head = (torch.randn(heads * dim, vocab, device="cuda", generator=g) * 0.4).to(dtype)
        self.k_pages, self.v_pages = (torch.full((pages, page, kv_heads, dim), float("nan"), dtype=dtype, device="cuda") for _ in range(2))
        self.frequencies = torch.tensor(inverse(dim // 2), dtype=F32, device="cuda")
        self.cache = cuda.PagedCache(self.k_pages, self.v_pages)

    def run(self, batch, ids, last_rows, draws, controls):
        from heirloom_b200 import cuda
        c = ctx()
        rows = self.embedding[ids]
        a, b = self.heads * self.dim, (self.heads + self.kv_heads) * self.dim
        q = cuda.paged_append(c, self.cache, batch, rows[:, a:b], rows[:, b:], rows[:, :a], self.frequencies)
        out, _ = cuda.paged_attention(c, self.cache, batch, q, self.heads)
        logits = (out[last_rows].float() @ self.head.float())
        return cuda.sample_rows(c, logits, draws, *controls)[0], out, logits


def whole_prompt(server, ids):
    """The layer's output for one sequence from its ids alone, in 64 bits, keys and queries rounded as the cache holds them."""
    x = server.embedding.double().cpu().numpy()[ids]
    n, (h, g, d) = len(ids), (server.heads, server.kv_heads, server.dim)
    f = server.frequencies.double().cpu().numpy()
    t = np.arange(n)
    stored = lambda y: torch.from_numpy(y).to(server.dtype).double().numpy()  # noqa: E731
    q = stored(pu.rotate(x[:, :h * d].reshape(n, h, d), t, f, False))
    k = stored(pu.rotate(x[:, h * d:(h + g) * d].reshape(n, g, d), t, f, False))
    v = x[:, (h + g) * d:].reshape(n, g, d)
    z = np.einsum("nhd,lhd->hnl", q, np.repeat(k, h // g, 1)) / np.sqrt(d)
    z = np.where(np.tril(np.ones((n, n), bool)), z, -np.inf)
    p = np.exp(z - z.max(-1, keepdims=True))
    p /= p.sum(-1, keepdims=True)
    return np.einsum("hnl,lhd->nhd", p, np.repeat(v, h // g, 1)).reshape(n, -1), np.einsum("hnl,lhd->nhd", p, np.abs(np.repeat(v, h // g, 1))).reshape(n, -1)


@pytest.mark.parametrize("dtype,heads,kv_heads,dim", [(BF16, 4, 4, 64), (BF16, 8, 2, 128), (F32, 4, 2, 48)])
def test_prompts_in_chunks_and_steps_captured_into_a_graph(dtype, heads, kv_heads, dim):
    """Four conversations: prompts in ragged chunks, then steps of a captured graph whose lengths and page table are rewritten between
    replays, one slot of the batch empty.  The layer's outputs are those of whole prompts; tokens are those that the rules choose from the logits."""
    from heirloom_b200 import cuda
    page, vocab, slots, width = 16, 300, 5, 12
    server = Server(dtype, heads, kv_heads, dim, vocab, page, 60, 1)
    rng = np.random.default_rng(3)
    prompts = [list(rng.integers(0, vocab, n)) for n in (37, 1, 120, 64)]
    table_host = rng.permutation(60)[:slots * width].reshape(slots, width).astype(np.int32)
    table = torch.from_numpy(table_host).cuda()
    held, ids = [0] * slots, [[] for _ in range(slots)]
    half = 2.0 ** -8 if dtype == BF16 else 2.0 ** -24
    chosen = dict(temperature=0.9, top_k=40, top_p=0.95, min_p=0.01)
    # a key or query off by one rounding (where the f32 rotation fell on the other side) moves a score by |q| |k| of that: bounded with the
    # values' spread, and a rounding of P and of the result
    def compare(slot, rows, outputs):
        want, reach = whole_prompt(server, ids[slot])
        got = outputs[rows]
        assert (np.abs(got - want[-len(rows):]) <= half * np.abs(want[-len(rows):]) + 10 * half * reach[-len(rows):] + 2.0 ** -16 * reach[-len(rows):]).all()

    def check_tokens(tokens, logits, draws, rows):
        x = host(logits)
        for r in rows:
            want, _ = pu.sample(x[r], draws[r], float(np.float32(0.9)), 40, float(np.float32(0.95)), float(np.float32(0.01)))
            assert host(tokens)[r] == want

    def controls(n):
        return (torch.full((n,), 0.9, device="cuda"), torch.full((n,), 40, dtype=torch.int32, device="cuda"),
                torch.full((n,), 0.95, device="cuda"), torch.full((n,), 0.01, device="cuda"))

    newest = {}
    for chunk in (30, 200):
        parts = [p[held[s]:held[s] + chunk] for s, p in enumerate(prompts)] + [[]]
        for s, p in enumerate(parts):
            ids[s] += p
            held[s] += len(p)
        first = np.concatenate([[0], np.cumsum([len(p) for p in parts])]).astype(np.int32)
        flat = torch.tensor(sum(parts, []), device="cuda")
        batch = cuda.PagedBatch(table, torch.tensor(held, dtype=torch.int32, device="cuda"), torch.from_numpy(first).cuda(), len(flat), max(map(len, parts)))
        with_tokens = [s for s, p in enumerate(parts) if p]
        draws = rng.random(len(with_tokens))
        tokens, out, logits = server.run(batch, flat, torch.tensor([int(first[s + 1]) - 1 for s in with_tokens], device="cuda"),
                                         torch.from_numpy(draws).cuda(), controls(len(with_tokens)))
        check_tokens(tokens, logits, draws, range(len(with_tokens)))
        for i, s in enumerate(with_tokens):
            compare(s, np.arange(first[s], first[s + 1]), host(out))
            newest[s] = int(tokens[i])
    # steps: static buffers, one token a slot, the fifth slot empty
    step_ids = torch.zeros(slots, dtype=torch.int64, device="cuda")
    lengths = torch.zeros(slots, dtype=torch.int32, device="cuda")
    draws_dev = torch.zeros(slots, dtype=torch.float64, device="cuda")
    batch, step_controls, all_rows = cuda.PagedBatch(table, lengths), controls(slots), torch.arange(slots, device="cuda")
    server.run(batch, step_ids, all_rows, draws_dev, step_controls)  # all slots empty
    torch.cuda.synchronize()
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]  # two, replayed in turn
    results = []
    for graph in graphs:
        with torch.cuda.graph(graph, stream=ctx().stream):
            results.append(server.run(batch, step_ids, all_rows, draws_dev, step_controls))
    for step in range(6):
        for s in range(4):
            ids[s].append(newest[s])
            held[s] += 1
        draws = rng.random(slots)
        step_ids.copy_(torch.tensor([ids[s][-1] if ids[s] else 0 for s in range(slots)]))
        lengths.copy_(torch.tensor(held, dtype=torch.int32))
        draws_dev.copy_(torch.from_numpy(draws))
        graphs[step % 2].replay()
        ctx().sync()
        tokens, out, logits = results[step % 2]
        check_tokens(tokens, logits, draws, range(4))
        outputs = host(out)
        assert (outputs[4] == 0).all()  # the empty slot
        for s in range(4):
            compare(s, np.array([s]), outputs)
            newest[s] = int(tokens[s])
    used = np.zeros(60, bool)
    for s in range(slots):
        used[table_host[s, :-(-held[s] // page)]] = True
    assert np.isnan(host(server.k_pages)[~used]).all()  # pages of nobody are as they were
