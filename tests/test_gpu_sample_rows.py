"""Choosing the next tokens of many rows on the GPU, against the rules in 64 bits."""
import numpy as np
import pytest
import torch

from tests import paged_util as pu
from tests.gpu_util import ctx, host

pytestmark = pytest.mark.gpu


def run(logits, draws, **controls):
    from heirloom_b200 import cuda
    types = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    given = {n: torch.tensor(np.broadcast_to(v, len(draws)).copy(), dtype=types[n], device="cuda") for n, v in controls.items()}
    tokens, p = cuda.sample_rows(ctx(), logits, torch.tensor(draws, dtype=torch.float64, device="cuda"), **given)
    return host(tokens), host(p), {n: host(v) for n, v in given.items()}


def check(logits, draws, **controls):
    tokens, p, given = run(logits, draws, **controls)
    x = logits.double().cpu().numpy()
    for r in range(len(x)):
        token, chance = pu.sample(x[r], draws[r], **{n: (int(v[r]) if n == "top_k" else float(v[r])) for n, v in given.items()})
        assert tokens[r] == token, (r, tokens[r], token, {n: v[r] for n, v in given.items()})
        # one rounding to f32; weights are whole multiples of 2^-40 of the largest or finer
        assert abs(p[r] - chance) <= 2.0 ** -24 * chance + 2.0 ** -40


def logits_of(rows, vocab, dtype=torch.float32, seed=0, wide=None, spread=2.5):
    g = torch.Generator("cuda").manual_seed(seed)
    x = (torch.randn(rows, wide or vocab, device="cuda", generator=g) * spread).to(dtype)
    return x[:, :vocab]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab", [1, 2, 7, 33, 1000, 1023, 1025, 4097, 50304, 128001, 300007])
def test_all_filters_of_all_sizes(vocab, dtype):
    rng = np.random.default_rng(vocab)
    rows = 24
    x = logits_of(rows, vocab, dtype, vocab, wide=vocab + vocab % 3)
    check(x, rng.random(rows))
    check(x, rng.random(rows), temperature=rng.choice([0.0, 0.3, 1.0, 2.0], rows))
    check(x, rng.random(rows), temperature=0.7, top_k=rng.integers(-1, min(vocab, 3000) + 2, rows))
    check(x, rng.random(rows), temperature=1.1, top_p=rng.choice([0.0, 1e-6, 0.3, 0.9, 0.99, 0.9999, 1.0], rows))
    check(x, rng.random(rows), min_p=rng.choice([0.0, 0.001, 0.3, 1.0, 2.0], rows))
    check(x, rng.random(rows), temperature=rng.choice([0.0, 0.5, 0.8, 1.0], rows), top_k=rng.choice([0, 1, 2, 50, 700], rows),
          top_p=rng.choice([0.2, 0.9, 0.95, 1.0], rows), min_p=rng.choice([0.0, 0.02, 0.1], rows))


@pytest.mark.parametrize("rows", [160, 300])
def test_rows_of_a_cta_each_with_controls_of_all_kinds(rows):
    """Slices that are read again from L2, with cuts of every length: of few ranks, by a list, by a short list of what can stay, by crowds."""
    rng = np.random.default_rng(rows)
    for vocab, dtype in ((50304, torch.float32), (50305, torch.bfloat16)):
        x = logits_of(rows, vocab, dtype, seed=rows, spread=1.5)
        x[::9] = x[::9].round()  # crowds
        check(x, rng.random(rows), temperature=rng.choice([0.0, 0.5, 1.0, 1.4], rows), top_k=rng.choice([0, 1, 50, 384, 400, 5000, 30000], rows),
              top_p=rng.choice([0.1, 0.5, 0.9, 0.999, 1.0], rows), min_p=rng.choice([0.0, 0.0, 1e-3, 0.05], rows))


@pytest.mark.parametrize("rows", [1, 2, 3, 17, 150, 400])
def test_numbers_of_rows(rows):
    rng = np.random.default_rng(rows)
    check(logits_of(rows, 5003, seed=rows), rng.random(rows), temperature=0.8, top_k=60, top_p=0.9, min_p=0.01)
    check(logits_of(rows, 5003, seed=rows + 1), rng.random(rows))


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_equal_logits_go_by_index(dtype):
    """Few values, many ties: every filter cuts within a group of equal ones."""
    g = torch.Generator("cuda").manual_seed(5)
    for vocab in (40, 3001, 50304):
        rng = np.random.default_rng(vocab)
        x = torch.randint(-2, 3, (16, vocab), device="cuda", generator=g).to(dtype)
        x[0] = 1.5                       # all the same
        x[1] = 0.0
        x[1, ::2] = -0.0                 # so are these
        u = rng.random(16)
        check(x, u, temperature=0.0)
        check(x, u, top_k=rng.integers(1, vocab, 16))
        check(x, u, top_p=rng.choice([0.1, 0.5, 0.77, 0.9], 16))
        check(x, u, top_k=rng.integers(1, vocab, 16), top_p=0.6, min_p=0.05)
    x = torch.zeros(3, 64, device="cuda", dtype=dtype)  # whole numbers: token i begins at the draw i / 64
    draws = np.array([0.0, 0.25, 63 / 64])
    assert run(x, draws)[0].tolist() == [0, 16, 63]
    assert run(x, np.array([0.0, 0.5, 1 - 2.0 ** -53]), top_k=[4, 4, 4])[0].tolist() == [0, 2, 3]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_infinities_nan_and_extremes(dtype):
    x = logits_of(12, 2000, dtype, 9).clone()
    low = torch.finfo(dtype).min
    x[0, 5:] = -torch.inf                        # a mask that leaves five
    x[1, :] = -torch.inf
    x[1, 1234] = -3.0                            # one
    x[2, :] = -torch.inf                         # none
    x[3, ::3] = torch.nan
    x[4, 7] = torch.inf                          # no probability either
    x[5, :] = torch.nan
    x[6, 100:] = low                             # the type's lowest value as a mask
    x[7, :] = low                                # equal all the same
    x[8, 3] = torch.finfo(dtype).max             # far above everything
    x[9] = torch.linspace(-3e4, 3e4, 2000, device="cuda").to(dtype)
    x[10, :] = torch.finfo(dtype).max
    x[11, 1::2] = -0.0
    u = np.linspace(0.0, 0.999, 12)
    check(x, u)
    check(x, u, top_k=3)
    check(x, u, top_p=0.5, min_p=0.1)
    check(x, u, temperature=0.0)
    check(x, u, temperature=[1e-30, 1e-3, 1.0, 1e30, np.inf, 1.0, 1e-3, 1.0, 1.0, 1e4, 1e-6, 5.0], top_p=0.9)
    tokens, p, _ = run(x, u)
    assert tokens[[2, 5]].tolist() == [-1, -1] and p[[2, 5]].tolist() == [0, 0]
    # controls that say nothing: less than 0 or NaN is the largest logit, shares outside (0, 1) no filter
    greedy = run(x, u, temperature=0.0)[0]
    assert np.array_equal(run(x, u, temperature=-1.0)[0], greedy) and np.array_equal(run(x, u, temperature=np.nan)[0], greedy)
    assert np.array_equal(run(x, u, top_p=-0.5, top_k=-7, min_p=-1.0)[0], tokens) and np.array_equal(run(x, u, top_p=np.nan, min_p=np.nan)[0], tokens)
    # draws outside [0, 1) are its ends
    ends = run(x, np.full(12, -0.5))[0], run(x, np.full(12, 1.0))[0]
    assert np.array_equal(ends[0], run(x, np.zeros(12))[0]) and np.array_equal(ends[1], run(x, np.full(12, 1 - 2.0 ** -53))[0])


def test_far_cuts():
    """A rank behind all fine bins of the first histogram, and shares so near to one that the tail counts."""
    x = torch.linspace(40.0, -400.0, 30000, device="cuda")[None].repeat(6, 1)
    x[3:] = torch.linspace(1e-3, -1e-3, 30000, device="cuda")
    check(x, np.linspace(0.01, 0.99, 6), temperature=100.0, top_k=[29999, 20000, 9000, 29999, 20000, 15000])
    check(x, np.linspace(0.01, 0.99, 6), temperature=50.0, top_p=[0.999999, 0.99, 0.9, 0.999999, 0.5, 0.25])


@pytest.mark.parametrize("rows", [6, 320])
def test_smallest_temperatures(rows):
    """Logits that only such a temperature tells apart: few have a weight, beside thousands of others nearly as large."""
    g = torch.Generator("cuda").manual_seed(rows)
    x = -torch.rand(rows, 50304, device="cuda", generator=g) * 1e-30
    x[::3] = logits_of(len(x[::3]), 50304, seed=rows)  # and the usual ones
    u = np.random.default_rng(rows).random(rows)
    for temperature in (1e-33, 1e-35, 1e-36):
        check(x, u, temperature=temperature)
        check(x, u, temperature=temperature, top_p=0.9)
        check(x, u, temperature=temperature, top_k=5000, top_p=0.999, min_p=1e-3)


def test_rows_of_millions():
    """Slices whose sums are kept in tiles of more than the usual size, and crowds in one of them."""
    x = logits_of(2, 4_400_001, seed=3, wide=4_400_003)
    x[1, 1_000_000:1_050_000] = x[1].max() + 1.0
    check(x, np.array([0.3, 0.7]), temperature=0.9)
    check(x, np.array([0.3, 0.7]), temperature=1.5, top_k=[60000, 49999], top_p=[0.9, 0.99])


def test_frequencies_follow_the_probabilities():
    """Evenly spread draws hit every token as often as it is probable, to one draw a border."""
    x = logits_of(1, 12, seed=4, spread=1.0)
    n = 4096
    tokens, _, _ = run(x.expand(n, 12).contiguous(), (np.arange(n) + 0.5) / n)
    share = np.exp(x.double().cpu().numpy()[0])
    assert np.abs(np.bincount(tokens, minlength=12) / n - share / share.sum()).max() <= 1.01 / n


def test_rows_give_the_same_tokens_alone_and_together():
    x, u = logits_of(300, 20000, seed=8), np.random.default_rng(2).random(300)
    together = run(x, u, temperature=0.9, top_p=0.97)
    for r in (0, 1, 150, 299):
        alone = run(x[r:r + 1], u[r:r + 1], temperature=0.9, top_p=0.97)
        assert alone[0][0] == together[0][r] and alone[1][0] == together[1][r]
