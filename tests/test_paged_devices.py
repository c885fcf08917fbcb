"""Tensors on another device than the context's are refused before anything is launched; on the CPU, with stand-ins for devices that are not here."""
from types import SimpleNamespace

import pytest
import torch

from heirloom_b200 import cuda
from heirloom_b200._lib import HeirloomError


class Library:
    def __getattr__(self, name):
        raise AssertionError(name + " was called")


class OnDevice:
    """As much of a CUDA tensor as the checks look at."""

    is_cuda = True

    def __init__(self, t, device):
        self.t, self.index = t, device

    def get_device(self):
        return self.index

    @property
    def device(self):
        return torch.device("cuda", self.index)

    def __getattr__(self, name):
        return getattr(self.t, name)


@pytest.mark.parametrize("context,tensors", [(0, 1), (1, 0)])
def test_tensors_on_another_device_than_the_contexts(context, tensors):
    ctx = SimpleNamespace(device=context, handle=None, lib=Library(), attention_workspace=Library())
    pages = OnDevice(torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), tensors)
    cache = cuda.PagedCache(pages, pages)
    batch = cuda.PagedBatch(OnDevice(torch.zeros(3, 2, dtype=torch.int32), tensors), OnDevice(torch.ones(3, dtype=torch.int32), tensors))
    rows = OnDevice(torch.zeros(3, 128, dtype=torch.bfloat16), tensors)
    logits, draws = OnDevice(torch.zeros(3, 100), tensors), OnDevice(torch.zeros(3, dtype=torch.float64), tensors)
    for call in (lambda: cuda.paged_append(ctx, cache, batch, rows, rows, rows), lambda: cuda.paged_append(ctx, cache, batch, rows, rows),
                 lambda: cuda.paged_attention(ctx, cache, batch, rows, 2), lambda: cuda.paged_attention(ctx, cache, batch, rows, 2, workspace=rows),
                 lambda: cuda.sample_rows(ctx, logits, draws)):
        with pytest.raises(HeirloomError, match=f"context's device cuda:{context}"):
            call()


@pytest.mark.parametrize("what", ["k", "v", "q", "batch", "frequencies", "q_out"])
def test_tensors_on_another_device_than_the_caches(what):
    ctx = SimpleNamespace(device=0, handle=None, lib=Library())
    at = lambda name: 1 if name == what else 0  # noqa: E731
    pages = OnDevice(torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16), 0)
    batch = cuda.PagedBatch(OnDevice(torch.zeros(3, 2, dtype=torch.int32), at("batch")), OnDevice(torch.ones(3, dtype=torch.int32), at("batch")))
    k, v, q, q_out = (OnDevice(torch.zeros(3, 128, dtype=torch.bfloat16), at(n)) for n in ("k", "v", "q", "q_out"))
    frequencies = OnDevice(torch.zeros(32), at("frequencies"))
    with pytest.raises(HeirloomError):
        cuda.paged_append(ctx, cuda.PagedCache(pages, pages), batch, k, v, q, frequencies, q_out=q_out)
