"""The operators of batched serving, measured: keys and values appended to a paged cache (rotated on the way), attention of new
tokens over that cache, and the choice of the next tokens.

`listed()` and `draw()` give cases, `prepare()` the tensors that a serving program has in hand, `run()` one pass: with `own`
the library's entry points, otherwise the same formulas in elementary torch operations.  `exact()` is the definition in 64
bits, written by itself.
"""
import math
import random

import numpy as np
import torch

own = False

_TYPES = {"bf16": torch.bfloat16, "f32": torch.float32}
_BYTES = {"bf16": 2, "f32": 4}


def listed():
    return [
        # one token of each of 64 conversations enters the cache of a 12 x 64 decoder: the smallest call, all latency
        {"name": "append_step", "op": "append", "sequences": 64, "new_min": 1, "new_max": 1, "len_min": 1, "len_max": 1024,
         "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "rotary": 64, "interleaved": False, "dtype": "bf16",
         "heads_first": False},
        # prompts of many lengths in chunks of up to 2048 tokens, shared key heads, pages of 64 positions with a head's rows together
        {"name": "append_chunks", "op": "append", "sequences": 13, "new_min": 7, "new_max": 2048, "len_min": 2048, "len_max": 40000,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "rotary": 128, "interleaved": False, "dtype": "bf16",
         "heads_first": True},
        # the f32 route with an odd head size, rotated in neighbouring pairs over half of its channels
        {"name": "append_f32", "op": "append", "sequences": 37, "new_min": 1, "new_max": 300, "len_min": 300, "len_max": 2000,
         "heads": 6, "kv_heads": 3, "head_dim": 80, "page": 32, "rotary": 40, "interleaved": True, "dtype": "f32",
         "heads_first": False},
        # one-token steps of eight sequences of the 12 x 64 decoder in its context of 1024: latency
        {"name": "attend_step_small", "op": "attend", "sequences": 8, "new_min": 1, "new_max": 1, "len_min": 5, "len_max": 1024,
         "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "dtype": "bf16", "heads_first": False},
        # one-token steps of a full server: 64 ragged sequences, four query heads to a key head
        {"name": "attend_step_batch", "op": "attend", "sequences": 64, "new_min": 1, "new_max": 1, "len_min": 100, "len_max": 8192,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64, "dtype": "bf16", "heads_first": False},
        # two very long conversations: few rows, so that the keys have to be shared out over the chip
        {"name": "attend_step_long", "op": "attend", "sequences": 2, "new_min": 1, "new_max": 1, "len_min": 60001, "len_max": 131071,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 32, "dtype": "bf16", "heads_first": True},
        # one-token steps and pieces of prompts in one batch, as a scheduler mixes them
        {"name": "attend_mixed", "op": "attend", "sequences": 19, "new_min": 1, "new_max": 511, "len_min": 511, "len_max": 4000,
         "heads": 12, "kv_heads": 12, "head_dim": 64, "page": 16, "dtype": "bf16", "heads_first": False},
        # a chunk of 4096 tokens of a long prompt over the 4096 before it: products
        {"name": "attend_chunk", "op": "attend", "sequences": 1, "new_min": 4096, "new_max": 4096, "len_min": 8192, "len_max": 8192,
         "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 128, "dtype": "bf16", "heads_first": False},
        # the f32 route with an odd head size: short chunks of a small model
        {"name": "attend_f32", "op": "attend", "sequences": 9, "new_min": 1, "new_max": 40, "len_min": 40, "len_max": 700,
         "heads": 6, "kv_heads": 3, "head_dim": 80, "page": 32, "dtype": "f32", "heads_first": False},
        # the next token of one conversation
        {"name": "sample_one", "op": "sample", "rows": 1, "vocab": 50304, "dtype": "f32", "padded": False, "filters": "all"},
        # the next tokens of a full server, each row with controls of its own
        {"name": "sample_batch", "op": "sample", "rows": 256, "vocab": 50304, "dtype": "f32", "padded": False, "filters": "mixed"},
        # bf16 logits of a wide, odd vocabulary, drawn from the whole distribution
        {"name": "sample_wide", "op": "sample", "rows": 48, "vocab": 128001, "dtype": "bf16", "padded": True, "filters": "none"},
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    kind = rng.choice(["append", "attend", "attend", "attend", "sample"])
    if kind == "sample":
        vocab = _log(rng, 300, 200000)
        return {"op": "sample", "rows": _log(rng, 1, max(1, min(512, 12_000_000 // vocab))), "vocab": vocab,
                "dtype": rng.choice(["f32", "bf16"]), "padded": rng.random() < 0.5, "filters": rng.choice(["none", "all", "mixed", "mixed"])}
    dtype = rng.choice(["bf16", "bf16", "bf16", "f32"])
    head_dim = rng.choice([64, 128, 64, 128, 32, 80, 96, 256])
    kv_heads = rng.choice([1, 2, 3, 4, 8, 12])
    group = rng.choice([1, 1, 2, 3, 4, 5, 8]) if kv_heads <= 8 else 1
    fast = dtype == "bf16" and head_dim in (64, 128)
    steps = rng.random() < 0.5
    sequences = _log(rng, 1, 200 if steps else 24)
    new_max = 1 if steps else _log(rng, 2, 2048 if fast or kind == "append" else 64)
    # keys and work are kept below those of the listed cases: positions x key heads x channels, and the scores of a chunk
    positions = 250_000_000 // (2 * kv_heads * head_dim) // sequences if fast else 4_000_000 // (kv_heads * head_dim) // sequences
    if not steps and kind == "attend":
        scores = 400_000_000 if fast else 1_500_000
        positions = min(positions, scores // (sequences * new_max * kv_heads * group))
    len_max = _log(rng, new_max, max(new_max, min(131072, positions)))
    case = {"op": kind, "sequences": sequences, "new_min": rng.choice([1, new_max]), "new_max": new_max, "len_min": rng.choice([new_max, len_max]),
            "len_max": len_max, "heads": kv_heads * group, "kv_heads": kv_heads, "head_dim": head_dim, "page": rng.choice([16, 32, 64, 128, 256]),
            "dtype": dtype, "heads_first": rng.random() < 0.3}
    if kind == "append":
        case["rotary"] = rng.choice([0, head_dim // 2, head_dim])
        case["interleaved"] = rng.random() < 0.5
    return case


def _between(case, what, low, high, n):
    """n whole numbers of [low, high], low and high among them where there are two: the case's own, the same for every seed."""
    rng = random.Random("%s %d %d %d" % (what, low, high, n))
    got = [rng.randint(low, high) for _ in range(n)]
    got[-1] = high
    if n > 1:
        got[0] = low
    return got


def _sizes(case):
    """(new tokens, lengths with them) of the sequences."""
    n = case["sequences"]
    return _between(case, "new", case["new_min"], case["new_max"], n), _between(case, "length", case["len_min"], case["len_max"], n)


def _generator(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def prepare(case, seed):
    return _prepare_sample(case, seed) if case["op"] == "sample" else _prepare_paged(case, seed)


def _prepare_paged(case, seed):
    g, dtype = _generator(seed), _TYPES[case["dtype"]]
    new, lengths = _sizes(case)
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["head_dim"], case["page"]
    tokens, wide = sum(new), -(-max(lengths) // page)
    pages = sum(-(-n // page) for n in lengths) + 3
    shape = (pages, kv_heads, page, dim) if case["heads_first"] else (pages, page, kv_heads, dim)
    k_pages, v_pages = (torch.randn(shape, generator=g, device="cuda", dtype=torch.float32).to(dtype) for _ in range(2))
    if case["heads_first"]:  # seen as [page, position, head, channel] all the same
        k_pages, v_pages = k_pages.transpose(1, 2), v_pages.transpose(1, 2)
    # pages in the order that sequences came for them, which is none
    order = torch.randperm(pages, generator=torch.Generator().manual_seed(seed)).tolist()
    table = np.full((len(lengths), wide), -1, np.int32)
    at = 0
    for i, n in enumerate(lengths):
        need = -(-n // page)
        table[i, :need] = order[at:at + need]
        at += need
    first = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
    state = {
        "case": dict(case), "k_pages": k_pages, "v_pages": v_pages, "page_table": torch.from_numpy(table).cuda(),
        "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "first": torch.from_numpy(first).cuda(),
        "tokens": tokens, "max_new": max(new), "max_length": max(lengths),
    }
    rows = torch.randn(tokens, (heads + 2 * kv_heads) * dim, generator=g, device="cuda", dtype=torch.float32).to(dtype)
    if case["op"] == "append":  # the fused projection's columns
        state["q"], state["k"], state["v"] = rows[:, :heads * dim], rows[:, heads * dim:(heads + kv_heads) * dim], rows[:, (heads + kv_heads) * dim:]
        half = case["rotary"] // 2
        state["frequencies"] = (10000.0 ** (-torch.arange(half, dtype=torch.float64) / max(1, half))).to(torch.float32).cuda()
    else:
        state["q"] = rows[:, :heads * dim].contiguous()
    return state


def _prepare_sample(case, seed):
    g = _generator(seed)
    rows, vocab, dtype = case["rows"], case["vocab"], _TYPES[case["dtype"]]
    wide = -(-vocab // 64) * 64 if case["padded"] else vocab
    # logits of a language model: a broad bulk and a few tokens far above it
    x = torch.randn(rows, wide, generator=g, device="cuda", dtype=torch.float32) * 2.5
    top = torch.rand(rows, 24, generator=g, device="cuda")
    x.scatter_add_(1, torch.randint(0, vocab, (rows, 24), generator=g, device="cuda"), 4.0 + 8.0 * top)
    state = {"case": dict(case), "logits": x.to(dtype)[:, :vocab],
             "draws": torch.rand(rows, generator=g, device="cuda", dtype=torch.float64)}
    if case["filters"] == "none":
        state["temperature"] = torch.full((rows,), 0.9, device="cuda")
        state["top_k"] = state["top_p"] = state["min_p"] = None
        return state
    rng = random.Random(seed)
    mixed = case["filters"] == "mixed"
    state["temperature"] = torch.tensor([rng.choice([0.0, 0.6, 0.8, 1.0, 1.3]) if mixed else 0.8 for _ in range(rows)], device="cuda")
    state["top_k"] = torch.tensor([rng.choice([0, 1, 20, 50, 400, 5000]) if mixed else 50 for _ in range(rows)], dtype=torch.int32, device="cuda")
    state["top_p"] = torch.tensor([rng.choice([1.0, 0.5, 0.9, 0.95, 0.999]) if mixed else 0.95 for _ in range(rows)], device="cuda")
    state["min_p"] = torch.tensor([rng.choice([0.0, 0.0, 0.02, 0.1]) if mixed else 0.02 for _ in range(rows)], device="cuda")
    return state


# ---- the library's calls --------------------------------------------------------------------------------------------------
_open = {}


def _library():
    if not _open:
        from heirloom_b200 import cuda
        _open["cuda"], _open["ctx"] = cuda, cuda.Context(torch.cuda.current_device())
    return _open["cuda"], _open["ctx"]


def _handles(state):
    """The descriptions of cache and batch that a serving program makes once and keeps."""
    cuda, _ = _library()
    if "handles" not in state:
        cache = cuda.PagedCache(state["k_pages"], state["v_pages"])
        batch = cuda.PagedBatch(state["page_table"], state["lengths"], state["first"], tokens=state["tokens"], max_new=state["max_new"],
                                max_length=state["max_length"])
        state["handles"] = cache, batch
    return state["handles"]


def _run_own(state):
    cuda, ctx = _library()
    case = state["case"]
    if case["op"] == "sample":
        return cuda.sample_rows(ctx, state["logits"], state["draws"], state["temperature"], state["top_k"], state["top_p"], state["min_p"])
    cache, batch = _handles(state)
    if case["op"] == "append":
        q = cuda.paged_append(ctx, cache, batch, state["k"], state["v"], state["q"], state["frequencies"], case["interleaved"])
        return q, state["k_pages"], state["v_pages"]
    return cuda.paged_attention(ctx, cache, batch, state["q"], case["heads"])


# ---- the plain forms ------------------------------------------------------------------------------------------------------
def run(state):
    if own:
        return _run_own(state)
    return {"append": _plain_append, "attend": _plain_attend, "sample": _plain_sample}[state["case"]["op"]](state)


def _rows_of(state):
    """(sequence, number within it) of every new token."""
    rows = torch.arange(state["tokens"], device="cuda")
    sequence = (rows[:, None] >= state["first"][None, 1:]).sum(1)
    return sequence, rows - state["first"][sequence]


def _rotated(x, angle, dims, interleaved):
    """x [tokens, heads, channels] in f32, its first `dims` channels turned by angle [tokens, dims / 2]."""
    if dims == 0:
        return x
    c, s = angle.cos().float()[:, None], angle.sin().float()[:, None]
    if interleaved:
        a, b = x[..., 0:dims:2], x[..., 1:dims:2]
        turned = torch.stack([a * c - b * s, a * s + b * c], -1).reshape(*x.shape[:-1], dims)
    else:
        a, b = x[..., :dims // 2], x[..., dims // 2:dims]
        turned = torch.cat([a * c - b * s, a * s + b * c], -1)
    return torch.cat([turned, x[..., dims:]], -1)


def _plain_append(state):
    case, page, dim = state["case"], state["case"]["page"], state["case"]["head_dim"]
    sequence, i = _rows_of(state)
    lengths, first = state["lengths"].long(), state["first"].long()
    position = lengths[sequence] - (first[sequence + 1] - first[sequence]) + i
    angle = position[:, None].double() * state["frequencies"].double()
    dtype, dims, turn = state["q"].dtype, case["rotary"], case["interleaved"]
    q = _rotated(state["q"].reshape(-1, case["heads"], dim).float(), angle, dims, turn).to(dtype)
    k = _rotated(state["k"].reshape(-1, case["kv_heads"], dim).float(), angle, dims, turn).to(dtype)
    at = state["page_table"].long()[sequence, position // page], position % page
    state["k_pages"].index_put_(at, k)
    state["v_pages"].index_put_(at, state["v"].reshape(-1, case["kv_heads"], dim))
    return q.reshape(-1, case["heads"] * dim), state["k_pages"], state["v_pages"]


def _plain_attend(state):
    case, dim, kv_heads = state["case"], state["case"]["head_dim"], state["case"]["kv_heads"]
    group, most, new = case["heads"] // kv_heads, state["max_length"], state["max_new"]
    lengths, first = state["lengths"].long(), state["first"].long()
    pages = state["page_table"].long().clamp(min=0)

    def dense(x):  # [sequence, head, position, channel]
        x = x[pages].float()
        return x.reshape(x.shape[0], -1, kv_heads, dim)[:, :most].transpose(1, 2)

    count = first[1:] - first[:-1]
    i = torch.arange(new, device="cuda")
    row = (first[:-1, None] + i).clamp(max=state["tokens"] - 1)
    q = state["q"].float().reshape(-1, kv_heads, group, dim)[row]  # [sequence, token, head, group, channel]
    q = q.permute(0, 2, 1, 3, 4).reshape(len(lengths), kv_heads, new * group, dim)
    j = torch.arange(most, device="cuda")
    seen = (j <= (lengths - count)[:, None, None] + i[None, :, None]) & (j < lengths[:, None, None])
    seen = seen.repeat_interleave(group, 1)[:, None]
    scores = torch.matmul(q, dense(state["k_pages"]).transpose(-1, -2)) * dim ** -0.5
    top = torch.where(seen, scores, -math.inf).amax(-1, keepdim=True)
    p = torch.where(seen, torch.exp(scores - torch.where(top == -math.inf, 0.0, top)), 0.0)
    total = p.sum(-1, keepdim=True)
    values = torch.where((j < lengths[:, None])[:, None, :, None], dense(state["v_pages"]), 0.0)
    out = torch.matmul(p, values) / torch.where(total == 0, 1.0, total)
    lse = top + torch.log(total)
    sequence, i = _rows_of(state)
    out = out.reshape(len(lengths), kv_heads, new, group, dim).permute(0, 2, 1, 3, 4)[sequence, i]
    lse = lse.reshape(len(lengths), kv_heads, new, group).permute(0, 2, 1, 3)[sequence, i]
    return out.reshape(-1, case["heads"] * dim).to(state["q"].dtype), lse.reshape(-1, case["heads"])


def _plain_sample(state):
    # in 64 bits: a token is chosen by which side of a border a sum lies on
    x = state["logits"].double()
    rows, vocab = x.shape
    t = state["temperature"].double()[:, None]
    sorted_x, order = torch.sort(x, dim=1, descending=True, stable=True)
    w = torch.exp((sorted_x - sorted_x[:, :1]) / torch.where(t > 0, t, 1.0))
    rank = torch.arange(vocab, device="cuda")
    if state["top_k"] is not None:
        k = state["top_k"].long()[:, None]
        w = torch.where((k <= 0) | (rank < k), w, 0.0)
    if state["top_p"] is not None:
        p = state["top_p"].double()[:, None]
        before = torch.cumsum(w, 1) - w
        w = torch.where((p <= 0) | (p >= 1) | (before < p * w.sum(1, keepdim=True)), w, 0.0)
    if state["min_p"] is not None:
        w = torch.where(w >= state["min_p"].double()[:, None].clamp(max=1), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)  # by token again
    total = w.sum(1, keepdim=True)
    token = (torch.cumsum(w, 1) <= state["draws"][:, None] * total).sum(1, keepdim=True).clamp(max=vocab - 1)
    token = torch.where(t > 0, token, order[:, :1])
    p = torch.where(t > 0, w.gather(1, token) / total, 1.0)
    return token[:, 0], p[:, 0].float()


# ---- work and definition --------------------------------------------------------------------------------------------------
def work(case):
    if case["op"] == "sample":
        return {"bytes": case["rows"] * (case["vocab"] * _BYTES[case["dtype"]] + 36), "flops": 4 * case["rows"] * case["vocab"]}
    size, dim, heads, kv_heads = _BYTES[case["dtype"]], case["head_dim"], case["heads"], case["kv_heads"]
    new, lengths = _sizes(case)
    tokens = sum(new)
    if case["op"] == "append":
        return {"bytes": 2 * tokens * (heads + 2 * kv_heads) * dim * size, "flops": 3 * tokens * (heads + kv_heads) * case["rotary"]}
    pairs = sum(n * length - n * (n - 1) // 2 for n, length in zip(new, lengths))
    return {"bytes": size * dim * (2 * kv_heads * sum(lengths) + 2 * heads * tokens) + 4 * heads * tokens, "flops": 4 * pairs * heads * dim}


def exact(case, seed):
    state = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](case, state)


def _exact_append(case, state):
    new, lengths = _sizes(case)
    page, dim, dims = case["page"], case["head_dim"], case["rotary"]
    position = torch.from_numpy(np.concatenate([np.arange(m - n, m) for n, m in zip(new, lengths)])).cuda()
    sequence = torch.from_numpy(np.repeat(np.arange(len(new)), new)).cuda()
    turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"), position.double()[:, None] * state["frequencies"].double())[:, None]

    def rotated(x, heads):
        x = x.double().reshape(-1, heads, dim)
        z, rest = x[..., :dims], x[..., dims:]
        if case["interleaved"]:
            z = torch.view_as_real(torch.complex(z[..., ::2], z[..., 1::2]) * turn).flatten(-2)
        else:
            z = torch.complex(*z.chunk(2, -1)) * turn
            z = torch.cat([z.real, z.imag], -1)
        return torch.cat([z, rest], -1)

    q, k = (rotated(state["q"], case["heads"]), rotated(state["k"], case["kv_heads"])) if dims else (
        state["q"].double(), state["k"].double().reshape(-1, case["kv_heads"], dim))
    k_pages, v_pages = state["k_pages"].double(), state["v_pages"].double()
    at = state["page_table"].long()[sequence, torch.div(position, page, rounding_mode="floor")], torch.remainder(position, page)
    k_pages[at] = k
    v_pages[at] = state["v"].double().reshape(-1, case["kv_heads"], dim)
    return q.reshape(-1, case["heads"] * dim), k_pages, v_pages


def _exact_attend(case, state):
    dim, kv_heads, page = case["head_dim"], case["kv_heads"], case["page"]
    group = case["heads"] // kv_heads
    outs, lses, at = [], [], 0
    for s, (n, length) in enumerate(zip(*_sizes(case))):
        pages = state["page_table"][s, :-(-length // page)].long()
        q = state["q"][at:at + n].double().reshape(n, kv_heads, group, dim)
        at += n
        out = torch.empty(n, kv_heads, group, dim, dtype=torch.float64, device="cuda")
        lse = torch.empty(n, kv_heads, group, dtype=torch.float64, device="cuda")
        hidden = torch.ones(n, length, dtype=torch.bool, device="cuda").triu(length - n + 1)
        for h in range(kv_heads):
            k, v = (x[pages, :, h].double().reshape(-1, dim)[:length] for x in (state["k_pages"], state["v_pages"]))
            z = torch.einsum("ngd,ld->ngl", q[:, h], k) / math.sqrt(dim)
            z = z.masked_fill(hidden[:, None], -math.inf)
            lse[:, h] = torch.logsumexp(z, -1)
            out[:, h] = torch.einsum("ngl,ld->ngd", torch.softmax(z, -1), v)
        outs.append(out.reshape(n, -1))
        lses.append(lse.reshape(n, -1))
    return torch.cat(outs), torch.cat(lses)


def _exact_sample(case, state):
    logits = state["logits"].double().cpu().numpy()
    controls = {name: None if state[name] is None else state[name].double().cpu().numpy() for name in ("temperature", "top_k", "top_p", "min_p")}
    draws = state["draws"].cpu().numpy()
    tokens, chances = [], []
    for r, x in enumerate(logits):
        t = controls["temperature"][r]
        if t == 0:
            tokens.append(int(np.argmax(x)))  # the first of the largest
            chances.append(1.0)
            continue
        weight = np.exp((x - x.max()) / t)
        ranked = np.lexsort((np.arange(len(x)), -x))
        if controls["top_k"] is not None and 0 < controls["top_k"][r] < len(x):
            ranked = ranked[:int(controls["top_k"][r])]
        if controls["top_p"] is not None and 0 < controls["top_p"][r] < 1:
            reached = np.cumsum(weight[ranked])
            ranked = ranked[:1 + int(np.searchsorted(reached, controls["top_p"][r] * reached[-1], side="left"))]
        if controls["min_p"] is not None:
            ranked = ranked[weight[ranked] >= min(1.0, controls["min_p"][r])]
        stays = np.sort(ranked)
        reached = np.cumsum(weight[stays])
        at = min(int(np.searchsorted(reached, draws[r] * reached[-1], side="right")), len(stays) - 1)
        tokens.append(int(stays[at]))
        chances.append(weight[stays[at]] / reached[-1])
    return torch.tensor(tokens), torch.tensor(chances, dtype=torch.float64)
