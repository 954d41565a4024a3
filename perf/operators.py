"""The operators of the paged key/value cache: what a serving program has them do, at the sizes it has it done.

``listed()`` names the cases, ``draw(rng)`` draws one more from the same ranges, ``prepare`` makes on the GPU what the
program holds before the call, ``run`` is one pass, in the plain form or, with ``own``, through the framework's entry
points, ``work`` says what the pass cannot do without, and ``exact`` gives its outputs in 64 bits.

Kinds:
  append     new tokens' keys and values written to the paged cache, keys (and queries) rotated to their positions
  attention  a chunk of new tokens per sequence (one token in a decode step) over the sequence's whole paged cache
  selected   each new token over the cached keys that its index list names, as the indexer's top-k gives them
"""

from __future__ import annotations

import math

import torch

own = False

THETA = 10_000.0
E4M3_MOST = 448.0
LEAST_SCALE = 2.0**-126
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.bfloat16}  # of the rows; an fp8 cache takes bf16 rows
# Bounds of the drawn cases: tokens x heads of an append, cached key/value elements and score pairs of an attention, and
# gathered key elements of a selected one.  Each is the largest listed case's.
MOST_APPEND = 8192 * 48
MOST_CACHED = 16 * 32768 * 8 * 128
MOST_PAIRS = 2048 * 32768 * 32
MOST_GATHERED = 4096 * 512 * 8 * 128
MOST_DRAWS = 2**28  # random numbers that the lists of a selected case are made from


def listed() -> list[dict]:
    return [
        # One interactive sequence's new token: the smallest call, where launches and latency count.
        {"name": "append_one", "kind": "append", "dtype": "bf16", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128,
         "rope_dim": 128, "page": 64, "pages": 512, "queries": True},
        # A prefill chunk of a server that rotates its queries in the same pass.
        {"name": "append_chunk_bf16", "kind": "append", "dtype": "bf16", "tokens": 8192, "heads": 32, "kv_heads": 8,
         "dim": 128, "rope_dim": 128, "page": 64, "pages": 512, "queries": True},
        # A ragged chunk written to a quantised cache with half of each head rotated, queries rotated elsewhere.
        {"name": "append_chunk_fp8", "kind": "append", "dtype": "fp8", "tokens": 6001, "heads": 32, "kv_heads": 8,
         "dim": 128, "rope_dim": 64, "page": 32, "pages": 1024, "queries": False},
        # Interactive decoding: one sequence of 4K keys.
        {"name": "decode_one_4k", "kind": "attention", "dtype": "bf16", "batch": 1, "chunk": 1, "length": 4096,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # A full decode batch: 16 sequences of 32K keys.
        {"name": "decode_batch_32k", "kind": "attention", "dtype": "bf16", "batch": 16, "chunk": 1, "length": 32768,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # Long contexts of unlike lengths on a quantised cache.
        {"name": "decode_long_fp8", "kind": "attention", "dtype": "fp8", "batch": 4, "chunk": 1, "length": 131072,
         "ragged": True, "heads": 64, "kv_heads": 8, "dim": 128, "page": 32, "lse": False},
        # A whole prompt at once: causal prefill of 4K tokens.
        {"name": "prefill_4k", "kind": "attention", "dtype": "bf16", "batch": 1, "chunk": 4096, "length": 4096,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": True},
        # Chunked prefill: the next 2048 tokens of a prompt whose context has reached 32K.
        {"name": "chunk_2k_of_32k", "kind": "attention", "dtype": "bf16", "batch": 1, "chunk": 2048, "length": 32768,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # A mixed batch: chunks from one token to some hundreds over contexts of unlike lengths, an odd group of heads.
        {"name": "chunks_ragged_f16", "kind": "attention", "dtype": "f16", "batch": 7, "chunk": 301, "length": 9973,
         "ragged": True, "heads": 28, "kv_heads": 4, "dim": 64, "page": 16, "lse": True},
        # Sparse decoding: the indexer's 2048 keys of each of 16 sequences of 32K.
        {"name": "selected_decode_32k", "kind": "selected", "dtype": "bf16", "batch": 16, "chunk": 1, "length": 32768,
         "k": 2048, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # The same on long quantised caches, lists of no round length.
        {"name": "selected_decode_fp8", "kind": "selected", "dtype": "fp8", "batch": 4, "chunk": 1, "length": 131072,
         "k": 2011, "heads": 64, "kv_heads": 8, "dim": 128, "page": 32, "lse": False},
        # Sparse prefill: every token of a 4K prompt over its own top-512 (early tokens have fewer: padded lists).
        {"name": "selected_prefill_4k", "kind": "selected", "dtype": "bf16", "batch": 1, "chunk": 4096, "length": 4096,
         "k": 512, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": True},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A size between low and high, even over its logarithm; most are odd or ragged."""

    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.3:
        value = value // 16 * 16
    return max(low, min(high, value))


def draw(rng) -> dict:
    kind = rng.choice(["append"] * 2 + ["attention"] * 4 + ["selected"] * 3)
    dim = rng.choice([64, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 4, 4, 6, 8, 16])
    dtype = rng.choice(["bf16", "bf16", "f16", "fp8"])
    page = rng.choice([16, 32, 64, 128, 256])
    shared = {"kind": kind, "dtype": dtype, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    if kind == "append":
        tokens = _spread(rng, 1, min(8192, MOST_APPEND * 128 // (dim * (heads + 2 * kv_heads))))
        return {**shared, "tokens": tokens, "rope_dim": rng.choice([dim, dim, dim // 2]),
                "pages": -(-tokens // page) + rng.randint(1, 64), "queries": rng.random() < 0.5}
    if kind == "attention":
        batch = _spread(rng, 1, 32)
        length = _spread(rng, 512, max(512, min(131072, MOST_CACHED // (batch * kv_heads * dim))))
        most = MOST_PAIRS * 128 // (dim * batch * length * heads)
        chunk = 1 if rng.random() < 0.4 else _spread(rng, 1, max(1, min(length, 4096, most)))
        return {**shared, "batch": batch, "chunk": chunk, "length": length, "ragged": rng.random() < 0.5,
                "lse": rng.random() < 0.5}
    batch = _spread(rng, 1, 16)
    length = _spread(rng, 512, max(512, min(131072, MOST_CACHED // (batch * kv_heads * dim))))
    k = min(length, _spread(rng, 64, 2048))
    most = min(MOST_GATHERED // (batch * k * kv_heads * dim), MOST_DRAWS // (batch * length))
    chunk = 1 if rng.random() < 0.5 else _spread(rng, 1, max(1, min(length, 4096, most)))
    return {**shared, "batch": batch, "chunk": chunk, "length": length, "k": k, "lse": rng.random() < 0.5}


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Keys and new tokens of each sequence: a ragged batch falls from the stated sizes to a quarter of the keys and to
    one token."""

    batch, length, chunk = case["batch"], case["length"], case["chunk"]
    if not case.get("ragged"):
        return [length] * batch, [chunk] * batch
    lengths = [max(1, length - 3 * length * b // (4 * batch)) for b in range(batch)]
    chunks = [max(1, chunk - chunk * b // max(1, batch - 1)) for b in range(batch)]
    return lengths, [min(c, n) for c, n in zip(chunks, lengths)]


def _quantised(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    scale = (x.abs().amax(-1) / E4M3_MOST).clamp(min=LEAST_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _cache(case: dict, pages: int, gen: torch.Generator) -> dict:
    """A filled cache; one key in a hundred is hot, four times the others' size."""

    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    keys = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    hot = torch.rand(shape[:3], generator=gen, device="cuda") < 0.01
    keys *= 1.0 + 3.0 * hot[..., None]
    values = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
    if case["dtype"] == "fp8":
        keys, key_scales = _quantised(keys)
        values, value_scales = _quantised(values)
        return {"keys": keys, "values": values, "key_scales": key_scales, "value_scales": value_scales}
    dtype = DTYPES[case["dtype"]]
    return {"keys": keys.to(dtype), "values": values.to(dtype), "key_scales": None, "value_scales": None}


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = DTYPES[case["dtype"]]
    heads, kv_heads, dim, page = case["heads"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    if case["kind"] == "append":
        tokens, pages = case["tokens"], case["pages"]
        state = {**case, **_cache(case, pages, gen), "new_keys": normal(tokens, kv_heads, dim),
                 "new_values": normal(tokens, kv_heads, dim),
                 "new_queries": normal(tokens, heads, dim) if case["queries"] else None}
        # consecutive positions from somewhere in a long context, in pages that are scattered over the pool
        start = int(torch.randint(0, 65536, (1,), generator=gen, device="cuda"))
        state["positions"] = torch.arange(start, start + tokens, device="cuda")
        order = torch.randperm(pages, generator=gen, device="cuda")
        at = torch.arange(tokens, device="cuda")
        state["rows"] = order[at // page] * page + at % page
    else:
        lengths, chunks = _lengths(case)
        per = [-(-n // page) for n in lengths]
        state = {**case, **_cache(case, sum(per), gen)}
        batch, columns = len(lengths), max(per)
        order = torch.randperm(sum(per), generator=gen, device="cuda").to(torch.int32)
        table = torch.zeros((batch, columns), device="cuda", dtype=torch.int32)
        first = 0
        for b, n in enumerate(per):
            table[b, :n] = order[first:first + n]
            first += n
        total = sum(chunks)
        state.update(page_table=table, lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32),
                     starts=None if total == batch and not case.get("ragged") else torch.tensor(
                         [sum(chunks[:b]) for b in range(batch + 1)], device="cuda", dtype=torch.int32),
                     new_queries=normal(total, heads, dim), longest=max(chunks))
        if case["kind"] == "selected":
            # distinct positions of each token's visible keys, ascending, as the indexer lists them; short rows padded
            visible = torch.cat([torch.arange(n - c + 1, n + 1, device="cuda") for n, c in zip(lengths, chunks)])
            draws = torch.rand((total, max(lengths)), generator=gen, device="cuda")
            draws.masked_fill_(torch.arange(max(lengths), device="cuda")[None] >= visible[:, None], -1.0)
            best, at = draws.topk(case["k"], dim=1)
            at = at.masked_fill(best < 0, max(lengths)).sort(dim=1).values
            state["indices"] = at.masked_fill(at == max(lengths), -1)
    if own:  # the handle of the cache that a program keeps
        from dsa_amd import paged

        state["cache"] = paged.PagedCache(state["keys"], state["values"], state["key_scales"], state["value_scales"])
    return state


def run(state: dict):
    if own:
        return _run_own(state)
    if state["kind"] == "append":
        return _append(state)
    return _attention(state) if state["kind"] == "attention" else _selected(state)


def _run_own(s: dict):
    from dsa_amd import paged

    if s["kind"] == "append":
        rotated = paged.append(s["cache"], s["new_keys"], s["new_values"], s["rows"], s["positions"],
                               queries=s["new_queries"], rope_dim=s["rope_dim"], theta=THETA)
        return _stored(s, rotated)
    if s["kind"] == "attention":
        return paged.attention(s["new_queries"], s["cache"], s["page_table"], s["lengths"], s["starts"],
                               return_lse=s["lse"])
    return paged.selected_attention(s["new_queries"], s["cache"], s["page_table"], s["lengths"], s["indices"],
                                    s["starts"], return_lse=s["lse"])


def _stored(s: dict, rotated) -> list:
    out = [s["keys"], s["values"]]
    if s["key_scales"] is not None:
        out += [s["key_scales"], s["value_scales"]]
    return out + ([rotated] if rotated is not None else [])


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = cos.shape[-1]
    x = x.float()
    first, second = x[..., :half], x[..., half:2 * half]
    return torch.cat([first * cos - second * sin, second * cos + first * sin, x[..., 2 * half:]], -1)


def _put(pages: torch.Tensor, scales, rows: torch.Tensor, x: torch.Tensor) -> None:
    if scales is None:
        pages.view(-1, *pages.shape[2:])[rows] = x.to(pages.dtype)
        return
    codes, scale = _quantised(x)
    pages.view(torch.uint8).view(-1, *pages.shape[2:])[rows] = codes.view(torch.uint8)
    scales.view(-1, scales.shape[2])[rows] = scale


def _append(s: dict) -> list:
    half = s["rope_dim"] // 2
    powers = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float32) / half)
    angles = (s["positions"].float()[:, None] * powers)[:, None]
    cos, sin = angles.cos(), angles.sin()
    _put(s["keys"], s["key_scales"], s["rows"], _rotated(s["new_keys"], cos, sin))
    _put(s["values"], s["value_scales"], s["rows"], s["new_values"].float())
    queries = s["new_queries"]
    return _stored(s, None if queries is None else _rotated(queries, cos, sin).to(queries.dtype))


def _read(pages: torch.Tensor, scales, at: torch.Tensor, by_page: bool) -> torch.Tensor:
    """The cache's pages ``at`` (or single rows of it) in 32 bits."""

    if by_page:
        x = pages.view(torch.uint8)[at].view(pages.dtype) if scales is not None else pages[at]
        return x.float() if scales is None else x.float() * scales[at][..., None]
    flat = pages.view(-1, *pages.shape[2:])
    if scales is None:
        return flat[at].float()
    return flat.view(torch.uint8)[at].view(pages.dtype).float() * scales.view(-1, scales.shape[2])[at][..., None]


def _softmax(scores: torch.Tensor, seen: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights and log sums of ``scores`` over the last axis where ``seen``; rows that see nothing have weights of 0."""

    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = weights.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    return weights / total.masked_fill(total == 0, 1.0), lse


def _attention(s: dict):
    queries, lengths, batch = s["new_queries"], s["lengths"].long(), s["batch"]
    kv_heads, dim = s["kv_heads"], s["dim"]
    group, longest, tokens = s["heads"] // kv_heads, s["longest"], s["new_queries"].shape[0]
    starts = torch.arange(batch + 1, device="cuda") if s["starts"] is None else s["starts"].long()
    count = starts[1:] - starts[:-1]
    step = torch.arange(longest, device="cuda")
    token = (starts[:-1, None] + step).clamp(max=tokens - 1)  # [B, n]
    q = queries[token].float().view(batch, longest, kv_heads, group, dim).permute(0, 2, 1, 3, 4)
    q = q.reshape(batch, kv_heads, longest * group, dim)
    at = s["page_table"].long()
    k = _read(s["keys"], s["key_scales"], at, True).view(batch, -1, kv_heads, dim).permute(0, 2, 3, 1).contiguous()
    v = _read(s["values"], s["value_scales"], at, True).view(batch, -1, kv_heads, dim).permute(0, 2, 1, 3).contiguous()
    last = (lengths - count)[:, None] + step  # the last key that each new token sees
    seen = torch.arange(k.shape[-1], device="cuda") <= torch.minimum(last, lengths[:, None] - 1)[..., None]
    seen = seen[:, None, :, None, :].expand(batch, 1, longest, group, -1).reshape(batch, 1, longest * group, -1)
    weights, lse = _softmax(torch.matmul(q, k) * dim**-0.5, seen)
    out = torch.matmul(weights, v).view(batch, kv_heads, longest, group, dim).permute(0, 2, 1, 3, 4)
    real = step < count[:, None]
    out = out.reshape(batch, longest, s["heads"], dim)[real].to(queries.dtype)
    if not s["lse"]:
        return out
    return out, lse.view(batch, kv_heads, longest, group).transpose(1, 2).reshape(batch, longest, s["heads"])[real]


def _selected(s: dict):
    queries, indices, batch = s["new_queries"], s["indices"], s["batch"]
    kv_heads, dim, page = s["kv_heads"], s["dim"], s["page"]
    tokens, group = queries.shape[0], s["heads"] // s["kv_heads"]
    starts = torch.arange(batch + 1, device="cuda") if s["starts"] is None else s["starts"].long()
    sequence = torch.searchsorted(starts, torch.arange(tokens, device="cuda"), right=True) - 1
    seen = (indices >= 0) & (indices < s["lengths"].long()[sequence, None])
    at = indices.masked_fill(~seen, 0)
    rows = s["page_table"].long()[sequence[:, None], at // page] * page + at % page
    k = _read(s["keys"], s["key_scales"], rows, False).permute(0, 2, 3, 1).contiguous()  # [T, G, D, k]
    v = _read(s["values"], s["value_scales"], rows, False).permute(0, 2, 1, 3).contiguous()
    q = queries.float().view(tokens, kv_heads, group, dim)
    weights, lse = _softmax(torch.matmul(q, k) * dim**-0.5, seen[:, None, None, :])
    out = torch.matmul(weights, v).reshape(tokens, s["heads"], dim).to(queries.dtype)
    return (out, lse.reshape(tokens, s["heads"])) if s["lse"] else out


def work(case: dict) -> dict:
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    stored = dim + 4 if case["dtype"] == "fp8" else 2 * dim  # bytes of one head's key or value
    if case["kind"] == "append":
        rotated = kv_heads + (heads if case["queries"] else 0)
        per_token = 2 * kv_heads * (2 * dim + stored) + 16 + (4 * heads * dim if case["queries"] else 0)
        return {"bytes": float(case["tokens"] * per_token), "flops": 3.0 * case["tokens"] * rotated * case["rope_dim"]}
    lengths, chunks = _lengths(case)
    tokens = sum(chunks)
    row = 4 * heads * dim + (4 * heads if case["lse"] else 0)  # a token's queries and outputs
    table = 4 * sum(-(-n // case["page"]) for n in lengths)
    if case["kind"] == "attention":
        pairs = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, chunks))
        return {"bytes": float(sum(lengths) * 2 * kv_heads * stored + tokens * row + table),
                "flops": 4.0 * heads * dim * pairs}
    named = [[min(case["k"], n - c + 1 + i) for i in range(c)] for n, c in zip(lengths, chunks)]
    read = sum(min(n, sum(x)) for n, x in zip(lengths, named))  # a key that several tokens name is read once
    return {"bytes": float(read * 2 * kv_heads * stored + tokens * (row + 8 * case["k"]) + table),
            "flops": 4.0 * heads * dim * sum(map(sum, named))}


def exact(case: dict, seed: int):
    """The operator's definition in 64 bits, one sequence (or kv head) after the other."""

    s = prepare(case, seed)
    wide = torch.float64
    page, dim, kv_heads, heads = case["page"], case["dim"], case["kv_heads"], case["heads"]

    def stored(name):
        x = s[name].to(wide)
        return x if s["key_scales"] is None else x * s[name[:-1] + "_scales"].to(wide)[..., None]

    if case["kind"] == "append":
        half = case["rope_dim"] // 2
        turn = torch.exp(-math.log(THETA) / half * torch.arange(half, device="cuda", dtype=wide))
        unit = torch.polar(torch.ones((), device="cuda", dtype=wide), s["positions"].to(wide)[:, None, None] * turn)

        def rotate(x):
            x = x.to(wide)
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * unit
            return torch.cat((z.real, z.imag, x[..., 2 * half:]), dim=-1)

        found = []
        scales = []
        for name, new in (("keys", rotate(s["new_keys"])), ("values", s["new_values"].to(wide))):
            if s["key_scales"] is not None:  # the value that a code stands for: x over its head's scale
                size = torch.clamp_min(new.abs().max(dim=-1).values / E4M3_MOST, LEAST_SCALE)
                new = new / size.unsqueeze(-1)
                kept = s[name[:-1] + "_scales"].to(wide).flatten(0, 1)
                kept[s["rows"]] = size
                scales.append(kept.view(s["keys"].shape[:3]))
            pages = s[name].to(wide).flatten(0, 1)
            pages[s["rows"]] = new
            found.append(pages.view(s["keys"].shape))
        return found + scales + ([rotate(s["new_queries"])] if case["queries"] else [])

    lengths, chunks = _lengths(case)
    queries = s["new_queries"].to(wide)
    keys, values = stored("keys").flatten(0, 1), stored("values").flatten(0, 1)
    outs, sums = [], []
    first = 0
    for b, (length, count) in enumerate(zip(lengths, chunks)):
        at = torch.arange(length, device="cuda")
        rows = s["page_table"][b].long()[at // page] * page + at % page
        q = queries[first:first + count]
        out = torch.empty_like(q)
        lse = torch.empty((count, heads), device="cuda", dtype=wide)
        if case["kind"] == "selected":
            lists = s["indices"][first:first + count]
        for h in range(heads):
            kv = h * kv_heads // heads
            if case["kind"] == "attention":
                logits = q[:, h] @ keys[rows, kv].T / math.sqrt(dim)
                hidden = at[None, :] > (length - count + torch.arange(count, device="cuda"))[:, None]
                logits[hidden] = -math.inf
                out[:, h] = torch.softmax(logits, dim=1) @ values[rows, kv]
            else:
                chosen = rows[lists.clamp(min=0)]
                logits = (keys[:, kv][chosen] * q[:, h, None, :]).sum(-1) / math.sqrt(dim)
                logits[lists < 0] = -math.inf
                out[:, h] = (torch.softmax(logits, dim=1)[..., None] * values[:, kv][chosen]).sum(1)
            lse[:, h] = torch.logsumexp(logits, dim=1)
        outs.append(out)
        sums.append(lse)
        first += count
    out = torch.cat(outs)
    return (out, torch.cat(sums)) if case["lse"] else out
