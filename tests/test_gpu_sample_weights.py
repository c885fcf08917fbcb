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
