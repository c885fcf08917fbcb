"""What the entry points for many sequences refuse, on the CPU: every refusal comes before the context's device is touched."""
import ctypes
import struct

import pytest
import torch

from ctypes import byref, c_float, c_int, c_longlong, c_size_t, c_void_p


@pytest.fixture(scope="module")
def lib():
    import __graft_entry__
    __graft_entry__.build()
    from heirloom_b200 import _lib
    return _lib.load()


CTX = ctypes.create_string_buffer(struct.pack("ii", 0, 148), 4096)  # of a context only the number of SMs is looked at
AT = 1 << 20                             # an aligned address that nobody follows


def cache(**changes):
    from heirloom_b200._lib import PagedCacheDesc
    d = dict(k_pages=AT, v_pages=AT, dtype=1, pages=4, page_size=16, kv_heads=2, head_dim=64, page_stride=16 * 128, position_stride=128,
             head_stride=64)
    return PagedCacheDesc(**{**d, **changes})


def batch(**changes):
    from heirloom_b200._lib import PagedBatchDesc
    d = dict(page_table=AT, lengths=AT, first=AT, ld_table=4, table_width=4, sequences=3, tokens=9, max_new=5, max_length=0)
    return PagedBatchDesc(**{**d, **changes})


BAD_CACHE = [
    (dict(k_pages=0), "null"), (dict(v_pages=0), "null"), (dict(dtype=2), "bf16 or f32"), (dict(pages=0), "pages"), (dict(kv_heads=0), "heads"),
    (dict(page_size=0), "power of two"), (dict(page_size=8), "power of two"), (dict(page_size=48), "power of two"), (dict(head_dim=60), "multiple of 8"),
    (dict(head_dim=264), "up to 256"), (dict(position_stride=63), "overlap"), (dict(head_stride=32), "overlap"), (dict(position_stride=132), "16 bytes"),
    (dict(page_stride=2052), "16 bytes"), (dict(k_pages=AT + 8), "aligned"), (dict(v_pages=AT + 2), "aligned"),
]
BAD_BATCH = [
    (dict(page_table=0), "null"), (dict(lengths=0), "null"), (dict(sequences=0), "requires"), (dict(tokens=0), "requires"), (dict(max_new=0), "requires"),
    (dict(table_width=0), "requires"), (dict(ld_table=3), "overlap"), (dict(first=0), "one new token"), (dict(first=0, tokens=3), "one new token"),
    (dict(max_length=65), "max_length"), (dict(max_length=-1), "max_length"), (dict(table_width=1 << 28, ld_table=1 << 28), "give max_length"),
]


def append(lib, c=None, b=None, **changes):
    d = dict(ctx=CTX, q=AT, ld_q=256, q_out=AT, ld_q_out=256, heads=4, k=AT, ld_k=128, v=AT, ld_v=128, frequencies=AT, rotary=64, interleaved=0)
    d.update(changes)
    c, b = c or cache(), b or batch()
    return lib.hl_paged_append(d["ctx"], ctypes.addressof(c), ctypes.addressof(b), c_void_p(d["q"]), c_longlong(d["ld_q"]), c_void_p(d["q_out"]),
                               c_longlong(d["ld_q_out"]), c_int(d["heads"]), c_void_p(d["k"]), c_longlong(d["ld_k"]), c_void_p(d["v"]),
                               c_longlong(d["ld_v"]), c_void_p(d["frequencies"]), c_int(d["rotary"]), c_int(d["interleaved"]))


def attend(lib, c=None, b=None, **changes):
    d = dict(ctx=CTX, q=AT, ld_q=256, out=AT, ld_out=256, lse=AT, heads=4, scale=0.125, workspace=AT, size=1 << 40)
    d.update(changes)
    c, b = c or cache(), b or batch()
    return lib.hl_paged_attention(d["ctx"], ctypes.addressof(c), ctypes.addressof(b), c_void_p(d["q"]), c_longlong(d["ld_q"]), c_void_p(d["out"]),
                                  c_longlong(d["ld_out"]), c_void_p(d["lse"]), c_int(d["heads"]), c_float(d["scale"]), c_void_p(d["workspace"]),
                                  c_size_t(d["size"]))


def refused(lib, rc, words):
    message = lib.hl_last_error().decode()
    assert rc == -1 and words in message, (rc, message)


@pytest.mark.parametrize("changes,words", BAD_CACHE)
def test_bad_caches(lib, changes, words):
    refused(lib, append(lib, cache(**changes)), words)
    refused(lib, attend(lib, cache(**changes)), words)


@pytest.mark.parametrize("changes,words", BAD_BATCH)
def test_bad_batches(lib, changes, words):
    refused(lib, append(lib, b=batch(**changes)), words)
    refused(lib, attend(lib, b=batch(**changes)), words)


@pytest.mark.parametrize("changes,words", [
    (dict(ctx=None), "null"), (dict(k=0), "null"), (dict(v=0), "null"), (dict(q=0), "null"), (dict(q_out=0), "null"), (dict(heads=0), "heads"),
    (dict(q=0, q_out=0), "heads goes with q"), (dict(rotary=63), "even"), (dict(rotary=66), "even"), (dict(rotary=-2), "even"), (dict(frequencies=0), "frequencies"),
    (dict(rotary=20), "halves"), (dict(ld_k=120), "cover"), (dict(ld_v=120), "cover"), (dict(ld_q=248), "cover"), (dict(ld_q_out=248), "cover"),
    (dict(ld_k=132), "16 bytes"), (dict(ld_q=260), "16 bytes"), (dict(k=AT + 4), "aligned"), (dict(q=AT + 8), "aligned"), (dict(q_out=AT + 8), "aligned"),
    (dict(heads=1 << 20, ld_q=1 << 26, ld_q_out=1 << 26), "too many heads")])
def test_bad_appends(lib, changes, words):
    refused(lib, append(lib, **changes), words)


@pytest.mark.parametrize("changes,words", [
    (dict(ctx=None), "null"), (dict(q=0), "null"), (dict(out=0), "null"), (dict(workspace=0), "null"), (dict(heads=0), "multiple of kv_heads"),
    (dict(heads=3), "multiple of kv_heads"), (dict(scale=0.0), "scale"), (dict(scale=float("nan")), "scale"), (dict(scale=float("inf")), "scale"),
    (dict(ld_q=248), "cover"), (dict(ld_out=248), "cover"), (dict(ld_q=260), "16 bytes"), (dict(ld_out=260), "16 bytes"), (dict(q=AT + 8), "aligned"),
    (dict(out=AT + 8), "aligned"), (dict(workspace=AT + 8), "aligned"), (dict(size=100), "workspace")])
def test_bad_attention(lib, changes, words):
    refused(lib, attend(lib, **changes), words)


def test_sequences_too_long_for_their_heads(lib):
    refused(lib, attend(lib, b=batch(table_width=1 << 26, ld_table=1 << 26, max_length=1 << 30)), "too long")


def test_more_sequences_and_channels_than_are_counted(lib):
    refused(lib, attend(lib, b=batch(sequences=1 << 30)), "too many sequences")
    wide = cache(kv_heads=1 << 25, position_stride=1 << 31, page_stride=1 << 35)
    refused(lib, attend(lib, wide, heads=1 << 25, ld_q=1 << 31, ld_out=1 << 31), "too many heads")


@pytest.mark.parametrize("args,words", [
    ((None, 1, 4, 2, 64), "null"), ((CTX, 2, 4, 2, 64), "bf16 or f32"), ((CTX, 1, 3, 2, 64), "multiple"), ((CTX, 1, 0, 2, 64), "multiple"),
    ((CTX, 1, 4, 0, 64), "multiple"), ((CTX, 1, 4, 2, 12), "head_dim"), ((CTX, 1, 4, 2, 512), "head_dim")])
def test_bad_workspace_questions(lib, args, words):
    size = c_size_t()
    refused(lib, lib.hl_paged_attention_workspace(args[0], *map(c_int, args[1:]), byref(size)), words)
    refused(lib, lib.hl_paged_attention_workspace(CTX, c_int(1), c_int(4), c_int(2), c_int(64), None), "null")


@pytest.mark.parametrize("changes,words", [
    (dict(ctx=None), "null"), (dict(logits=0), "null"), (dict(draws=0), "null"), (dict(tokens=0), "null"), (dict(dtype=2), "f32 or bf16"),
    (dict(rows=0), "requires"), (dict(vocab=0), "requires"), (dict(vocab=(1 << 24) + 1, ld=1 << 31), "2^24"), (dict(ld=99), "stride"),
    (dict(logits=AT + 2), "misaligned"), (dict(logits=AT + 1, dtype=1), "misaligned")])
def test_bad_samples(lib, changes, words):
    d = dict(ctx=CTX, logits=AT, dtype=0, ld=100, rows=3, vocab=100, draws=AT, tokens=AT)
    d.update(changes)
    rc = lib.hl_sample_rows(d["ctx"], c_void_p(d["logits"]), c_int(d["dtype"]), c_longlong(d["ld"]), c_int(d["rows"]), c_int(d["vocab"]), None, None,
                            None, None, c_void_p(d["draws"]), c_void_p(d["tokens"]), None)
    refused(lib, rc, words)


def test_wrappers_refuse_what_they_cannot_describe():
    from heirloom_b200 import cuda
    from heirloom_b200._lib import HeirloomError
    k = torch.zeros(4, 16, 2, 64, dtype=torch.bfloat16)
    for bad in (lambda: cuda.PagedCache(k, k), lambda: cuda.PagedCache(k, k[:, :, :1]), lambda: cuda.PagedCache(k[0], k[0]),
                lambda: cuda.PagedCache(k.half(), k.half()), lambda: cuda.PagedBatch(torch.zeros(2, 3, dtype=torch.int32), torch.zeros(2, dtype=torch.int32)),
                lambda: cuda.sample_rows(None, torch.zeros(2, 3), torch.zeros(2, dtype=torch.float64)),
                lambda: cuda.sample_rows(None, torch.zeros(3), torch.zeros(3, dtype=torch.float64))):
        with pytest.raises(HeirloomError):
            bad()
