"""Weights of sampled rows whose sums show how near they are: logits far below the largest beside it, tails of millions."""
import numpy as np
import pytest
import torch

from tests.gpu_util import ctx, host

pytestmark = pytest.mark.gpu


def sample(x, draws, **controls):
    from heirloom_b200 import cuda
    types = dict(temperature=torch.float32, top_k=torch.int32, top_p=torch.float32, min_p=torch.float32)
    given = {n: torch.full((len(draws),), v, dtype=types[n], device="cuda") for n, v in controls.items()}
    tokens, p = cuda.sample_rows(ctx(), x, torch.tensor(draws, dtype=torch.float64, device="cuda"), **given)
    return host(tokens), host(p)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("vocab,rows", [(2982, 3), (2982, 200), (128001, 5), (128001, 200)])
def test_logits_far_smaller_than_the_largest(vocab, rows, dtype):
    """A top of 8 over logits around 2^-22, whose difference from it does not fit the type in which it is formed; probabilities of the top and of
    others, by all ways to an answer."""
    g = torch.Generator("cuda").manual_seed(vocab)
    x = (torch.randn(rows, vocab, device="cuda", generator=g) * 2.0 ** -22).to(dtype)
    x[:, 77] = 8.0
    weight = np.exp(x.double().cpu().numpy() - 8.0)
    share = weight[:, 77] / weight.sum(1)
    for draws, kept, controls in ((np.zeros(rows), None, {}), (np.full(rows, 0.999), None, {}), (np.full(rows, 0.5), None, dict(top_p=0.9999)),
                                  (np.zeros(rows), 200, dict(top_k=200)), (np.full(rows, 0.999), 200, dict(top_k=200)), (np.zeros(rows), 2000, dict(top_k=2000))):
        tokens, p = sample(x, draws, **controls)
        if "top_p" in controls:  # the shortest prefix by falling logit
            kept = 1 + np.array([int(np.searchsorted(np.cumsum(np.sort(w)[::-1]), float(np.float32(0.9999)) * w.sum())) for w in weight])
        total = np.array([np.sort(w)[::-1][:vocab if kept is None else (kept if np.isscalar(kept) else kept[r])].sum() for r, w in enumerate(weight)])
        want = weight[np.arange(rows), tokens] / total
        # a rounding to f32, 2^-24; weights to 2^-28, and of so many units of 2^-45 of the largest one that is shifted out
        bound = (2.0 ** -24 + 2 * 2.0 ** -28 + vocab * 2.0 ** -45 / total + 2.0 ** -45 / weight[np.arange(rows), tokens]) * want
        # of a cut that falls between tokens of nearly one weight, one more or less may stay
        bound = bound + (want * np.exp(-8.0) / total if "top_p" in controls else 0)
        assert (np.abs(p - want) <= bound).all(), (controls, np.abs(p - want).max())
    assert (share < 0.6 if vocab < 10000 else share < 0.03).all()


@pytest.mark.parametrize("vocab,dtype", [(1 << 24, torch.float32), ((1 << 24) - 3, torch.bfloat16), (1_000_003, torch.float32), (270_001, torch.bfloat16),
                                         (131_073, torch.bfloat16)])
def test_tails_of_small_weights_count(vocab, dtype):
    """One large logit and a tail of the smallest that still show together, about 2^-14 of it for 2^24 logits."""
    g = torch.Generator("cuda").manual_seed(vocab % 1000)
    x = (torch.rand(1, vocab, device="cuda", generator=g) - 27.0).to(dtype)  # 2^-38.2 of the large one on the average
    x[0, 5] = 0.0
    weight = np.exp(x[0].double().cpu().numpy())
    # in 64 bits of mantissa: sums of 53 drift by 3e-10 where millions of equal weights round alike
    reached = np.cumsum(weight.astype(np.longdouble))
    total, tail = reached[-1], float(reached[-1] - 1)
    reached = reached / total
    # weights to 2^-28, the largest to nothing; what is shifted out, a unit each at most
    unit = 2.0 ** -60 if vocab > 1 << 18 else 2.0 ** -44
    off = 2 * 2.0 ** -28 * tail + 2 * vocab * unit
    draws = np.array([0.5, 1.0 - tail / 2, 1.0 - tail / 7, 1.0 - 2.0 ** -53])
    rows = x.expand(len(draws), vocab).contiguous()
    tokens, p = sample(rows, draws)
    assert tokens[0] == 5 and (tokens[1:] != 5).all()
    for r, token in enumerate(tokens):
        assert (reached[token - 1] if token > 0 else 0.0) - off <= draws[r] <= reached[token] + off
        want = weight[token] / total
        assert abs(p[r] - want) <= (2.0 ** -24 + 2 * 2.0 ** -28 + 2 * vocab * unit) * want + unit
    # half of the tail by rank, and by weight; a draw of 0 is the first token that stays, whichever that is
    order = np.argsort(-weight, kind="stable")
    falling = weight[order]

    def halved(kept, few, **controls):
        slack = few * falling[1]
        tokens, p = sample(rows[:2], np.array([0.0, 0.5]), **controls)
        assert tokens[1] == 5 and abs(p[1] * float(falling[:kept].astype(np.longdouble).sum()) - 1.0) <= 2.0 ** -24 + 2 * off + slack
        want = weight[tokens[0]] / falling[:kept].sum()
        # of a cut by weight, some of the tokens of nearly one weight at its end may or may not stay
        assert (tokens[0] in order[:kept + few] and tokens[0] <= order[:kept - few].min()) if few else tokens[0] == order[:kept].min()
        assert abs(p[0] - want) <= (2.0 ** -24 + 2 * 2.0 ** -28 + 2 * off + slack) * want + 2 * unit

    halved(vocab // 2, 0, top_k=vocab // 2)
    share = float(np.float32(1.0 - tail / 2)) if tail > 2.0 ** -20 else 0.0
    kept = 1 + int(np.searchsorted(np.cumsum(falling.astype(np.longdouble)), share * total)) if 0 < share < 1 else vocab
    halved(kept, min(kept - 1, 2 + int(2 * off / falling[-1])), top_p=share)


@pytest.mark.parametrize("temperature", [1e-36, 0.5, 1e30, float("inf")])
def test_wide_rows_of_all_temperatures(temperature):
    """Sums from one weight to as many as there are logits, from which the units of wide rows follow."""
    vocab = 300_001
    g = torch.Generator("cuda").manual_seed(1)
    x = torch.randn(5, vocab, device="cuda", generator=g)
    x[1, 10:] = -torch.inf
    x[2, 1:] = torch.finfo(torch.float32).min
    x[3, ::2] = torch.nan
    x[4, :] = -torch.inf
    draws = np.array([0.25, 0.9, 0.9, 0.6, 0.5])
    tokens, p = sample(x, draws, temperature=temperature)
    t = float(np.float32(temperature))
    for r, row in enumerate(x.double().cpu().numpy()):
        row = np.where(np.isfinite(row), row, -np.inf)
        if r == 4:
            assert tokens[r] == -1 and p[r] == 0
            continue
        with np.errstate(invalid="ignore"):
            weight = np.where(np.isneginf(row), 0.0, np.exp((row - row.max()) / t))
        total = weight.sum()
        reached = np.cumsum(weight) / total
        off = 2 * 2.0 ** -28 + 2 * vocab * 2.0 ** -60
        assert (reached[tokens[r] - 1] if tokens[r] > 0 else 0.0) - off <= draws[r] <= reached[tokens[r]] + off
        assert abs(p[r] * total / weight[tokens[r]] - 1.0) <= 2.0 ** -24 + 2 * off
