"""The operators that make a paged key/value cache smaller: its rows in 4 bits, and the eviction of keys that no query
looks at.

``listed()`` names the cases, ``draw(rng)`` draws one more from the same ranges, ``prepare`` makes on the GPU what the
program holds before the call, ``run`` is one pass, in the plain form or, with ``own``, through the framework's entry
points, ``work`` says what the pass cannot do without, and ``exact`` gives its outputs in 64 bits.

A 4-bit head is e2m1 codes, two a byte (the first in the low half), with one power of two (e8m0: the byte less 127) for
each 32 of them, the least under which the largest magnitude is 7 or less, so that no code is off by more than half a
step.  Codes and scales lie head by head within a page.

Kinds:
  append     new tokens' keys and values written to a 4-bit cache, keys (and queries) rotated to their positions; the
             cache read back as the values it stands for
  attention  a chunk of new tokens per sequence (one token in a decode step) over the sequence's whole 4-bit cache
  selected   each new token over the keys of a 4-bit cache that its index list names
  weights    what each cached key has of the new tokens' softmax weights, added to what it had
  evict      each sequence cut to its newest keys and those of largest accumulated weight, in place
"""

from __future__ import annotations

import math

import torch

own = False

THETA = 10_000.0
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
E4M3_MOST = 448.0
LEAST_SCALE = 2.0**-126
BLOCK = 32                   # codes that share a scale
LEAST_POWER, MOST_POWER = -124, 125
ROW_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "fp8": torch.bfloat16, "fp4": torch.bfloat16}  # of the queries
# Bounds of the drawn cases: tokens x heads of an append, cached key/value elements and score pairs of an attention,
# gathered key elements of a selected one, score pairs of accumulated weights, and cached elements of an eviction.  Each
# is the largest listed case's.
MOST_APPEND = 8192 * 48
MOST_CACHED = 16 * 32768 * 8 * 128
MOST_PAIRS = 2048 * 32768 * 32
MOST_GATHERED = 16 * 2048 * 8 * 128
MOST_DRAWS = 2**28  # random numbers that the lists of a selected case are made from
MOST_WEIGHED = 4096 * 2048 * 32
MOST_EVICTED = 16 * 16384 * 8 * 128


def listed() -> list[dict]:
    return [
        # One interactive sequence's new token: the smallest call, where launches and latency count.
        {"name": "append4_one", "kind": "append", "tokens": 1, "heads": 32, "kv_heads": 8, "dim": 128, "rope_dim": 128,
         "page": 64, "pages": 4, "queries": True},
        # A prefill chunk of a server that rotates its queries in the same pass.
        {"name": "append4_chunk", "kind": "append", "tokens": 8192, "heads": 32, "kv_heads": 8, "dim": 128, "rope_dim": 128,
         "page": 64, "pages": 136, "queries": True},
        # Interactive decoding: one sequence of 4K keys.
        {"name": "decode4_one_4k", "kind": "attention", "batch": 1, "chunk": 1, "length": 4096, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # A full decode batch: 16 sequences of 32K keys.
        {"name": "decode4_batch_32k", "kind": "attention", "batch": 16, "chunk": 1, "length": 32768, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # Chunked prefill: the next 2048 tokens of a prompt whose context has reached 32K.
        {"name": "chunk4_2k_of_32k", "kind": "attention", "batch": 1, "chunk": 2048, "length": 32768, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # A mixed batch: chunks from one token to some hundreds over contexts of unlike lengths, an odd group of heads.
        {"name": "chunks4_ragged", "kind": "attention", "batch": 7, "chunk": 301, "length": 9973, "ragged": True,
         "heads": 28, "kv_heads": 4, "dim": 64, "page": 16, "lse": True},
        # Sparse decoding: the indexer's 2048 keys of each of 16 sequences of 32K.
        {"name": "selected4_decode_32k", "kind": "selected", "batch": 16, "chunk": 1, "length": 32768, "k": 2048,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "lse": False},
        # Sparse decoding of a few long sequences, lists of no round length.
        {"name": "selected4_decode_long", "kind": "selected", "batch": 3, "chunk": 1, "length": 100003, "k": 1531,
         "heads": 64, "kv_heads": 8, "dim": 64, "page": 32, "lse": True},
        # A decode step's weights, each step of a server that evicts by them: 16 sequences of 32K keys.
        {"name": "weights_decode_32k", "kind": "weights", "dtype": "bf16", "batch": 16, "chunk": 1, "length": 32768,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # The weights of a whole prompt's rows, after its prefill into a 4-bit cache.
        {"name": "weights_prompt_4k", "kind": "weights", "dtype": "fp4", "batch": 1, "chunk": 4096, "length": 4096,
         "ragged": False, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64},
        # One sequence back to its budget of 4K keys after 64 more tokens, all heads alike.
        {"name": "evict_one_4k", "kind": "evict", "dtype": "bf16", "batch": 1, "length": 4160, "keep": 4096, "recent": 256,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "ragged": False, "per_head": False},
        # A batch after its prompts: each head of 16 sequences cut from 16K keys to its own 4K.
        {"name": "evict_batch_16k", "kind": "evict", "dtype": "bf16", "batch": 16, "length": 16384, "keep": 4096,
         "recent": 128, "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "ragged": True, "per_head": True},
    ]


def _spread(rng, low: int, high: int) -> int:
    """A size between low and high, even over its logarithm; most are odd or ragged."""

    value = int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))
    if rng.random() < 0.3:
        value = value // 16 * 16
    return max(low, min(high, value))


def draw(rng) -> dict:
    kind = rng.choice(["append"] * 2 + ["attention"] * 4 + ["selected"] * 2 + ["weights"] * 3 + ["evict"] * 3)
    dim = rng.choice([64, 128, 128, 128, 256])
    kv_heads = rng.choice([1, 2, 4, 8, 8])
    heads = kv_heads * rng.choice([1, 4, 4, 6, 8, 16])
    page = rng.choice([16, 32, 64, 128, 256])
    shared = {"kind": kind, "heads": heads, "kv_heads": kv_heads, "dim": dim, "page": page}
    if kind == "append":
        tokens = _spread(rng, 1, min(8192, MOST_APPEND * 128 // (dim * (heads + 2 * kv_heads))))
        return {**shared, "tokens": tokens, "rope_dim": rng.choice([dim, dim, dim // 2]),
                "pages": -(-tokens // page) + rng.randint(1, 4), "queries": rng.random() < 0.5}
    if kind == "evict":
        batch = _spread(rng, 1, 16)
        length = _spread(rng, 256, max(256, min(65536, MOST_EVICTED // (batch * kv_heads * dim))))
        keep = max(16, int(length * rng.uniform(0.1, 1.0)))
        return {**shared, "dtype": rng.choice(["bf16", "f16", "fp8", "fp4"]), "batch": batch, "length": length,
                "keep": keep, "recent": rng.randint(0, keep // 2), "ragged": rng.random() < 0.5,
                "per_head": rng.random() < 0.5}
    batch = _spread(rng, 1, 32 if kind == "attention" else 16)
    length = _spread(rng, 512, max(512, min(131072, MOST_CACHED // (batch * kv_heads * dim))))
    if kind == "selected":
        k = min(length, _spread(rng, 64, 2048))
        most = min(MOST_GATHERED // (batch * k * kv_heads * dim), MOST_DRAWS // (batch * length))
        chunk = 1 if rng.random() < 0.5 else _spread(rng, 1, max(1, min(length, 4096, most)))
        return {**shared, "batch": batch, "chunk": chunk, "length": length, "k": k, "lse": rng.random() < 0.5}
    most = (MOST_PAIRS if kind == "attention" else MOST_WEIGHED) * 128 // (dim * batch * length * heads)
    chunk = 1 if rng.random() < 0.4 else _spread(rng, 1, max(1, min(length, 4096, most)))
    shared.update(batch=batch, chunk=chunk, length=length, ragged=rng.random() < 0.5)
    if kind == "weights":
        return {**shared, "dtype": rng.choice(["bf16", "f16", "fp8", "fp4", "fp4"])}
    return {**shared, "lse": rng.random() < 0.5}


def _dtype(case: dict) -> str:
    return case.get("dtype", "fp4")


def _lengths(case: dict) -> tuple[list[int], list[int]]:
    """Keys and new tokens of each sequence: a ragged batch falls from the stated sizes to a quarter of the keys and to
    one token."""

    batch, length, chunk = case["batch"], case["length"], case.get("chunk", 1)
    if not case.get("ragged"):
        return [length] * batch, [chunk] * batch
    lengths = [max(1, length - 3 * length * b // (4 * batch)) for b in range(batch)]
    chunks = [max(1, chunk - chunk * b // max(1, batch - 1)) for b in range(batch)]
    return lengths, [min(c, n) for c, n in zip(chunks, lengths)]


def _quantised8(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    scale = (x.abs().amax(-1) / E4M3_MOST).clamp(min=LEAST_SCALE)
    return (x / scale[..., None]).to(torch.float8_e4m3fn), scale


def _power_of_two(power: torch.Tensor) -> torch.Tensor:
    """2^power in 32 bits, for -126 to 127, to the bit."""

    return (power.to(torch.int32) + 127 << 23).view(torch.float32)


def _quantised4(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Packed codes ``[..., D / 2]`` and scale bytes ``[..., D / 32]`` of ``x`` (32 or 64 bits, finite)."""

    x = x.unflatten(-1, (-1, BLOCK))
    fraction, power = torch.frexp(x.abs().amax(-1))  # the largest is fraction * 2^power, fraction in [1/2, 1)
    power = torch.where(fraction <= 7 / 8, power - 3, power - 2)
    power = power.masked_fill(fraction == 0, LEAST_POWER).clamp(LEAST_POWER, MOST_POWER)
    size = x.abs() * _power_of_two(-power)[..., None]
    # codes 0 .. 7: steps of 1/2 below 2, of 1 below 4, of 2 above
    code = torch.where(size < 2, (2 * size).round(), torch.where(size < 4, size.round() + 2, (size / 2).round() + 4))
    code = code.clamp(max=7).to(torch.uint8) | (x < 0).to(torch.uint8) << 3
    code = code.flatten(-2).unflatten(-1, (-1, 2))
    return code[..., 0] | code[..., 1] << 4, (power + 127).to(torch.uint8)


def _read4(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """What codes ``[..., D / 2]`` under scales ``[..., D / 32]`` stand for, in 32 bits."""

    values = torch.tensor([*E2M1, *(-v for v in E2M1)], device=codes.device)
    x = torch.stack([values[(codes & 15).int()], values[(codes >> 4).int()]], -1).flatten(-2)
    powers = _power_of_two(scales.to(torch.int32) - 127)
    return (x.unflatten(-1, (-1, BLOCK)) * powers[..., None]).flatten(-2)


def _paged_heads(x: torch.Tensor) -> torch.Tensor:
    """``[pages, page, heads, n]`` laid out head by head within a page."""

    return x.transpose(1, 2).contiguous().transpose(1, 2)


def _cache(case: dict, pages: int, gen: torch.Generator) -> dict:
    """A filled cache; one key in a hundred is hot, four times the others' size.  4-bit codes are uint8 here, and
    scales ``[pages, heads, page, D / 32]``."""

    shape = (pages, case["page"], case["kv_heads"], case["dim"])
    dtype = _dtype(case)
    found = {"key_scales": None, "value_scales": None}
    for name in ("key", "value"):
        x = torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32)
        if name == "key":
            x *= 1.0 + 3.0 * (torch.rand(shape[:3], generator=gen, device="cuda") < 0.01)[..., None]
        if dtype == "fp8":
            found[name + "s"], found[name + "_scales"] = _quantised8(x)
        elif dtype == "fp4":
            codes, scales = _quantised4(x)
            found[name + "s"], found[name + "_scales"] = _paged_heads(codes), scales.transpose(1, 2).contiguous()
        else:
            found[name + "s"] = x.to(ROW_TYPES[dtype])
    return found


def prepare(case: dict, seed: int) -> dict:
    gen = torch.Generator(device="cuda").manual_seed(seed)
    dtype = ROW_TYPES[_dtype(case)]
    kind, heads, kv_heads, dim, page = case["kind"], case["heads"], case["kv_heads"], case["dim"], case["page"]

    def normal(*shape):
        return torch.randn(shape, generator=gen, device="cuda", dtype=torch.float32).to(dtype)

    if kind == "append":
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
        state["every_row"] = torch.arange(pages * page, device="cuda")
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
        state.update(page_table=table, lengths=torch.tensor(lengths, device="cuda", dtype=torch.int32))
        if kind != "evict":
            state.update(starts=None if total == batch and not case.get("ragged") else torch.tensor(
                             [sum(chunks[:b]) for b in range(batch + 1)], device="cuda", dtype=torch.int32),
                         new_queries=normal(total, heads, dim), longest=max(chunks))
        if kind in ("weights", "evict"):
            # weights of a long run: most of the mass on few keys, some keys with none at all
            size = (kv_heads, sum(per) * page)
            weights = torch.exp(2.0 * torch.randn(size, generator=gen, device="cuda"))
            state["weights"] = weights * (torch.rand(size, generator=gen, device="cuda") > 0.02)
        if kind == "weights":  # counted anew a few calls ago: what one call adds is as large as what is there
            state["weights"] *= heads // kv_heads * case["chunk"] / case["length"]
            state["lse"] = _denominators(state, lengths, chunks)
        if kind == "evict":  # the rows that a sequence keeps, to read them back
            at = torch.arange(case["keep"], device="cuda")
            mine = at[None] < state["lengths"][:, None]
            at = at.clamp(max=columns * page - 1)
            state["kept_rows"] = (table.long()[:, at // page] * page + at % page)[mine]
        if kind == "selected":
            # distinct positions of each token's visible keys, ascending, as the indexer lists them; short rows padded
            visible = torch.cat([torch.arange(n - c + 1, n + 1, device="cuda") for n, c in zip(lengths, chunks)])
            draws = torch.rand((total, max(lengths)), generator=gen, device="cuda")
            draws.masked_fill_(torch.arange(max(lengths), device="cuda")[None] >= visible[:, None], -1.0)
            best, at = draws.topk(case["k"], dim=1)
            at = at.masked_fill(best < 0, max(lengths)).sort(dim=1).values
            state["indices"] = at.masked_fill(at == max(lengths), -1)
    if own:  # the handle of the cache that a program keeps
        from dsa_amd import paged

        parts = [state[n] for n in ("keys", "values", "key_scales", "value_scales")]
        if _dtype(case) == "fp4":
            parts = [x.view(t) for x, t in zip(parts, [torch.float4_e2m1fn_x2] * 2 + [torch.float8_e8m0fnu] * 2)]
        state["cache"] = paged.PagedCache(*parts)
    return state


def _denominators(s: dict, lengths: list[int], chunks: list[int]) -> torch.Tensor:
    """The log sums that the attention before has returned, sequence by sequence."""

    group = s["heads"] // s["kv_heads"]
    found, first = [], 0
    for b, (n, c) in enumerate(zip(lengths, chunks)):
        k = _stored(s, "key", s["page_table"][b:b + 1, :-(-n // s["page"])].long())[0].flatten(0, 1)[:n]
        q = s["new_queries"][first:first + c].float().unflatten(1, (-1, group)).permute(1, 0, 2, 3).flatten(1, 2)
        scores = torch.matmul(q, k.permute(1, 2, 0).contiguous()) * s["dim"]**-0.5
        last = n - c + torch.arange(c, device="cuda").repeat_interleave(group)
        scores.masked_fill_(torch.arange(n, device="cuda") > last[:, None], -math.inf)
        found.append(torch.logsumexp(scores, -1).unflatten(1, (c, group)).transpose(0, 1).flatten(1))
        first += c
    return torch.cat(found)


def run(state: dict):
    if own:
        return _run_own(state)
    return {"append": _append, "attention": _attention, "selected": _selected, "weights": _weights,
            "evict": _evict}[state["kind"]](state)


def _run_own(s: dict):
    from dsa_amd import eviction, paged

    kind = s["kind"]
    if kind == "append":
        rotated = paged.append(s["cache"], s["new_keys"], s["new_values"], s["rows"], s["positions"],
                               queries=s["new_queries"], rope_dim=s["rope_dim"], theta=THETA)
        out = list(paged.read(s["cache"], s["every_row"]))
        return out if rotated is None else [*out, rotated]
    if kind == "attention":
        return paged.attention(s["new_queries"], s["cache"], s["page_table"], s["lengths"], s["starts"],
                               return_lse=s["lse"])
    if kind == "selected":
        return paged.selected_attention(s["new_queries"], s["cache"], s["page_table"], s["lengths"], s["indices"],
                                        s["starts"], return_lse=s["lse"])
    weights = s["weights"].clone()
    if kind == "weights":
        eviction.accumulate_weights(weights, s["new_queries"], s["cache"], s["page_table"], s["lengths"], s["lse"],
                                    s["starts"])
        return weights
    lengths, kept = eviction.evict(s["cache"], s["page_table"], s["lengths"], weights, s["keep"], recent=s["recent"],
                                   per_head=s["per_head"])
    if _dtype(s) == "fp4":
        return [*paged.read(s["cache"], s["kept_rows"]), weights, lengths, kept]
    return [*_buffers(s), weights, lengths, kept]


def _buffers(s: dict) -> list:
    return [s[n] for n in ("keys", "values", "key_scales", "value_scales") if s[n] is not None]


def _rotated(x: torch.Tensor, cos: torch.Tensor, sin: torch.Tensor) -> torch.Tensor:
    half = cos.shape[-1]
    x = x.double()
    first, second = x[..., :half], x[..., half:2 * half]
    return torch.cat([first * cos - second * sin, second * cos + first * sin, x[..., 2 * half:]], -1)


def _append(s: dict) -> list:
    half, page = s["rope_dim"] // 2, s["page"]
    # in 64 bits: angles of far positions, and values next to the border between two codes
    powers = THETA ** (-torch.arange(half, device="cuda", dtype=torch.float64) / half)
    angles = (s["positions"].double()[:, None] * powers)[:, None]
    cos, sin = angles.cos(), angles.sin()
    pages, slots = s["rows"] // page, s["rows"] % page
    for name, new in (("key", _rotated(s["new_keys"], cos, sin)), ("value", s["new_values"].float())):
        codes, scales = _quantised4(new)
        s[name + "s"][pages, slots] = codes
        s[name + "_scales"][pages, :, slots] = scales
    every = torch.arange(s["pages"], device="cuda")
    out = [_stored(s, n, every).flatten(0, 1).to(torch.bfloat16) for n in ("key", "value")]
    queries = s["new_queries"]
    return out if queries is None else [*out, _rotated(queries, cos, sin).to(queries.dtype)]


def _stored(s: dict, name: str, pages: torch.Tensor) -> torch.Tensor:
    """The cache's ``pages`` in 32 bits: ``[..., page, heads, D]``."""

    x, scales = s[name + "s"], s[name + "_scales"]
    if _dtype(s) == "fp4":
        return _read4(x[pages], scales[pages].transpose(-3, -2))
    if _dtype(s) == "fp8":
        return x.view(torch.uint8)[pages].view(x.dtype).float() * scales[pages][..., None]
    return x[pages].float()


def _softmax(scores: torch.Tensor, seen: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """Weights and log sums of ``scores`` over the last axis where ``seen``; rows that see nothing have weights of 0."""

    scores = scores.masked_fill(~seen, -math.inf)
    top = scores.amax(-1, keepdim=True)
    weights = torch.exp(scores - top.masked_fill(top == -math.inf, 0.0))
    total = weights.sum(-1, keepdim=True)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    return weights / total.masked_fill(total == 0, 1.0), lse


def _chunks(s: dict):
    """The batch padded to its longest chunk: queries ``[B, G, n * group, D]`` in 32 bits, each row's token ``[B, n]``,
    whether it has one, and which keys each row sees, ``[B, 1, n * group, keys]``."""

    queries, lengths, batch = s["new_queries"], s["lengths"].long(), s["batch"]
    kv_heads, group, longest = s["kv_heads"], s["heads"] // s["kv_heads"], s["longest"]
    starts = torch.arange(batch + 1, device="cuda") if s["starts"] is None else s["starts"].long()
    count = starts[1:] - starts[:-1]
    step = torch.arange(longest, device="cuda")
    token = (starts[:-1, None] + step).clamp(max=queries.shape[0] - 1)
    q = queries[token].float().unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    last = torch.minimum((lengths - count)[:, None] + step, lengths[:, None] - 1)  # that each new token sees
    keys = torch.arange(s["page_table"].shape[1] * s["page"], device="cuda")
    seen = (keys <= last[..., None])[:, None, :, None].expand(-1, 1, longest, group, -1).flatten(2, 3)
    return q, token, step < count[:, None], seen


def _attention(s: dict):
    kv_heads, group, longest = s["kv_heads"], s["heads"] // s["kv_heads"], s["longest"]
    q, _, real, seen = _chunks(s)
    at = s["page_table"].long()
    k = _stored(s, "key", at).flatten(1, 2).permute(0, 2, 3, 1).contiguous()
    v = _stored(s, "value", at).flatten(1, 2).permute(0, 2, 1, 3).contiguous()
    weights, lse = _softmax(torch.matmul(q, k) * s["dim"]**-0.5, seen)
    out = torch.matmul(weights, v).unflatten(2, (longest, group)).permute(0, 2, 1, 3, 4).flatten(2, 3)
    out = out[real].to(s["new_queries"].dtype)
    if not s["lse"]:
        return out
    return out, lse.unflatten(2, (longest, group)).transpose(1, 2).reshape(s["batch"], longest, kv_heads * group)[real]


def _selected(s: dict):
    queries, indices, batch = s["new_queries"], s["indices"], s["batch"]
    kv_heads, dim, page = s["kv_heads"], s["dim"], s["page"]
    tokens, group = queries.shape[0], s["heads"] // s["kv_heads"]
    starts = torch.arange(batch + 1, device="cuda") if s["starts"] is None else s["starts"].long()
    sequence = torch.searchsorted(starts, torch.arange(tokens, device="cuda"), right=True) - 1
    seen = (indices >= 0) & (indices < s["lengths"].long()[sequence, None])
    at = indices.masked_fill(~seen, 0)
    pages, slots = s["page_table"].long()[sequence[:, None], at // page], at % page
    k, v = (_read4(s[n + "s"][pages, slots], s[n + "_scales"][pages, :, slots]) for n in ("key", "value"))  # [T, k, G, D]
    q = queries.float().view(tokens, kv_heads, group, dim)
    weights, lse = _softmax(torch.matmul(q, k.permute(0, 2, 3, 1).contiguous()) * dim**-0.5, seen[:, None, None, :])
    out = torch.matmul(weights, v.permute(0, 2, 1, 3).contiguous()).reshape(tokens, s["heads"], dim).to(queries.dtype)
    return (out, lse.reshape(tokens, s["heads"])) if s["lse"] else out


def _places(s: dict, columns: int) -> torch.Tensor:
    """Cache rows ``[B, n]`` of every position that the page table has."""

    at = torch.arange(columns * s["page"], device="cuda")
    return s["page_table"].long()[:, at // s["page"]] * s["page"] + at % s["page"]


def _weights(s: dict):
    kv_heads, group, longest = s["kv_heads"], s["heads"] // s["kv_heads"], s["longest"]
    q, token, real, seen = _chunks(s)
    k = _stored(s, "key", s["page_table"].long()).flatten(1, 2).permute(0, 2, 3, 1).contiguous()
    lse = s["lse"][token].unflatten(2, (kv_heads, group)).permute(0, 2, 1, 3).flatten(2, 3)  # [B, G, n * group]
    weights = torch.exp(torch.matmul(q, k) * s["dim"]**-0.5 - lse[..., None])
    seen = seen & real[:, None, :, None].expand(-1, 1, longest, group).flatten(2, 3)[..., None]
    found = weights.masked_fill(~seen, 0.0).sum(2)  # [B, G, keys]
    places = _places(s, s["page_table"].shape[1])
    mine = torch.arange(places.shape[1], device="cuda") < s["lengths"][:, None]  # what lies past is another's
    return s["weights"].clone().index_add_(1, places[mine], found.transpose(0, 1)[:, mine])


def _evict(s: dict):
    """Kept keys stay below the new length where they lie; those from there on fill, in order, the places of evicted
    ones."""

    batch, kv_heads, keep, recent = s["batch"], s["kv_heads"], s["keep"], s["recent"]
    lengths = s["lengths"].long()
    weights = s["weights"].clone()
    places = _places(s, s["page_table"].shape[1])  # [B, n]
    n = places.shape[1]
    at = torch.arange(n, device="cuda")
    new = lengths.clamp(max=keep)
    mass = weights[:, places].transpose(0, 1)  # [B, G, n]
    lists = kv_heads if s["per_head"] else 1
    if not s["per_head"]:
        mass = mass.double().sum(1, keepdim=True).float()
    inside = (at < lengths[:, None])[:, None].expand(batch, lists, n)
    newest = inside & (at >= (lengths - recent)[:, None])[:, None]
    rank = mass.masked_fill(newest, math.inf).masked_fill(~inside, -math.inf)
    order = torch.sort(rank, dim=-1, descending=True, stable=True).indices
    kept = torch.zeros_like(inside).scatter_(2, order, (at < new[:, None])[:, None].expand(batch, lists, n))
    below = (at < new[:, None])[:, None]
    holes, movers = ~kept & below, kept & ~below
    b, g, to = torch.nonzero(holes, as_tuple=True)  # as many of one as of the other in every list, in order
    source = torch.nonzero(movers, as_tuple=True)[2]
    where = at.expand(batch, lists, n).masked_fill(~below, -1).clone()
    where[b, g, to] = source
    if not s["per_head"]:  # a move is every head's
        g = torch.arange(kv_heads, device="cuda").repeat(b.numel())
        b, to, source = (x.repeat_interleave(kv_heads) for x in (b, to, source))
    dst, src = places[b, to], places[b, source]
    page = s["page"]
    for x in ("keys", "values"):
        x = s[x].view(torch.uint8) if _dtype(s) in ("fp8", "fp4") else s[x]
        x[dst // page, dst % page, g] = x[src // page, src % page, g]
    for x in ("key_scales", "value_scales"):
        if _dtype(s) == "fp4":
            s[x][dst // page, g, dst % page] = s[x][src // page, g, src % page]
        elif s[x] is not None:
            s[x][dst // page, dst % page, g] = s[x][src // page, src % page, g]
    weights[g, dst] = weights[g, src]
    freed = (at < lengths[:, None]) & (at >= new[:, None])
    weights[:, places[freed]] = 0.0
    where = torch.cat([where, where.new_full((batch, lists, max(0, keep - n)), -1)], -1)[..., :keep]
    where = where if s["per_head"] else where[:, 0]
    if _dtype(s) == "fp4":
        rows = s["kept_rows"]
        out = [_read4(s[x + "s"][rows // page, rows % page], s[x + "_scales"][rows // page, :, rows % page])
               .to(torch.bfloat16) for x in ("key", "value")]
    else:
        out = _buffers(s)
    return [*out, weights, new.to(torch.int32), where]


def work(case: dict) -> dict:
    heads, kv_heads, dim = case["heads"], case["kv_heads"], case["dim"]
    # bytes of one head's key or value
    stored = {"fp4": dim / 2 + dim / BLOCK, "fp8": dim + 4.0}.get(_dtype(case), 2.0 * dim)
    if case["kind"] == "append":
        rotated = kv_heads + (heads if case["queries"] else 0)
        per_token = 2 * kv_heads * (2 * dim + stored) + 16 + (4 * heads * dim if case["queries"] else 0)
        back = case["pages"] * case["page"] * (2 * kv_heads * (stored + 2 * dim) + 8)  # the cache as bf16
        return {"bytes": float(case["tokens"] * per_token + back), "flops": 3.0 * case["tokens"] * rotated * case["rope_dim"]}
    lengths, chunks = _lengths(case)
    tokens = sum(chunks)
    table = 4 * sum(-(-n // case["page"]) for n in lengths)
    if case["kind"] == "evict":
        # every weight is read and written once (the copy that is cut), the moved keys too: with weights that do not go
        # by position, as many as evicted keys lie below the new length
        moved = sum(min(n, case["keep"]) * (1 - min(n, case["keep"]) / n) for n in lengths)
        rows = sum(-(-n // case["page"]) for n in lengths) * case["page"]
        lists = kv_heads if case["per_head"] else 1
        back = 2 * kv_heads * (stored + 2 * dim) * sum(min(n, case["keep"]) for n in lengths) if _dtype(case) == "fp4" else 0
        return {"bytes": float(8 * rows * kv_heads + moved * kv_heads * 4 * stored + 8 * lists * case["batch"] * case["keep"]
                               + back + table), "flops": float(sum(lengths) * lists)}
    row = 4 * heads * dim + (4 * heads if case.get("lse") else 0)  # a token's queries and outputs
    pairs = sum(c * n - c * (c - 1) // 2 for n, c in zip(lengths, chunks))
    if case["kind"] == "weights":
        rows = sum(-(-n // case["page"]) for n in lengths) * case["page"]
        return {"bytes": float(sum(lengths) * kv_heads * stored + 8 * rows * kv_heads + tokens * heads * (2 * dim + 4) + table),
                "flops": 2.0 * heads * dim * pairs}
    if case["kind"] == "attention":
        return {"bytes": float(sum(lengths) * 2 * kv_heads * stored + tokens * row + table),
                "flops": 4.0 * heads * dim * pairs}
    named = [[min(case["k"], n - c + 1 + i) for i in range(c)] for n, c in zip(lengths, chunks)]
    read = sum(min(n, sum(x)) for n, x in zip(lengths, named))  # a key that several tokens name is read once
    return {"bytes": float(read * 2 * kv_heads * stored + tokens * (row + 8 * case["k"]) + table),
            "flops": 4.0 * heads * dim * sum(map(sum, named))}


def _exact_power(power: torch.Tensor) -> torch.Tensor:
    """2^power for whole powers from -160 to 160."""

    table = torch.tensor([2.0**p for p in range(-160, 161)], device=power.device, dtype=torch.float64)
    return table[power.long() + 160]


def _exact_code(x: torch.Tensor) -> torch.Tensor:
    """The value nearest to each of ``x`` (64 bits, finite) that a 4-bit head can hold, ties to the even code."""

    blocks = x.reshape(*x.shape[:-1], -1, BLOCK)
    top = blocks.abs().max(-1, keepdim=True).values
    power = torch.full_like(top, float(LEAST_POWER))
    for bits in (128, 64, 32, 16, 8, 4, 2, 1):  # the least power under which the largest is 7 or less
        smaller = power + bits
        power = torch.where(7 * _exact_power(smaller - 1) < top, smaller, power)
    unit = _exact_power(power.clamp(max=float(MOST_POWER)))
    grid = torch.tensor(E2M1, device=x.device, dtype=x.dtype)
    middle = (grid[1:] + grid[:-1]) / 2
    size = (blocks / unit).abs()
    code = torch.bucketize(size, middle)  # the lower of the two codes at their middle
    odd = (code % 2 == 1) & (code < 7) & (size == middle[code.clamp(max=6)])
    return (torch.sign(blocks) * grid[code + odd] * unit).reshape(x.shape)


def _exact_stored(s: dict, name: str) -> torch.Tensor:
    """The whole cache in 64 bits, ``[rows, heads, D]``."""

    wide = torch.float64
    x, scales = s[name + "s"], s[name + "_scales"]
    if scales is None:
        return x.to(wide).flatten(0, 1)
    if _dtype(s) == "fp8":
        return (x.to(wide) * scales.to(wide)[..., None]).flatten(0, 1)
    x = x.contiguous()
    found = torch.empty((*x.shape[:3], 2 * x.shape[3]), device=x.device, dtype=wide)
    for place, code in ((0, x % 16), (1, x // 16)):
        power, half = (code % 8 // 2).to(wide), (code % 2).to(wide)
        size = torch.where(power == 0, half / 2, _exact_power(power - 1) * (1 + half / 2))
        found[..., place::2] = torch.where(code > 7, -size, size)
    unit = _exact_power(scales.permute(0, 2, 1, 3).long() - 127)
    return (found * unit.repeat_interleave(BLOCK, -1)).flatten(0, 1)


def exact(case: dict, seed: int):
    """The operator's definition in 64 bits, one sequence (or kv head) after the other."""

    s = prepare(case, seed)
    wide = torch.float64
    kind, page, dim, kv_heads, heads = case["kind"], case["page"], case["dim"], case["kv_heads"], case["heads"]
    if kind == "append":
        half = case["rope_dim"] // 2
        turn = torch.exp(-math.log(THETA) / half * torch.arange(half, device="cuda", dtype=wide))
        unit = torch.polar(torch.ones((), device="cuda", dtype=wide), s["positions"].to(wide)[:, None, None] * turn)

        def rotate(x):
            x = x.to(wide)
            z = torch.complex(x[..., :half], x[..., half:2 * half]) * unit
            return torch.cat((z.real, z.imag, x[..., 2 * half:]), dim=-1)

        found = []
        for name, new in (("key", rotate(s["new_keys"])), ("value", s["new_values"].to(wide))):
            rows = _exact_stored(s, name)
            rows[s["rows"]] = _exact_code(new)
            found.append(rows)
        return found + ([rotate(s["new_queries"])] if case["queries"] else [])

    lengths, chunks = _lengths(case)

    def rows_of(b):
        at = torch.arange(lengths[b], device="cuda")
        return s["page_table"][b].long()[at // page] * page + at % page

    if kind == "evict":
        keep, recent = case["keep"], case["recent"]
        weights = s["weights"].to(wide)
        lists = kv_heads if case["per_head"] else 1
        where = torch.full((len(lengths), lists, keep), -1, device="cuda")
        for b, n in enumerate(lengths):
            rows, size = rows_of(b), min(n, keep)
            for g in range(lists):
                mine = [g] if case["per_head"] else list(range(kv_heads))
                mass = s["weights"][mine][:, rows].to(wide).sum(0).to(torch.float32).cpu()
                old = max(0, n - recent)
                chosen = sorted(range(old), key=lambda j, m=mass.tolist(): (-m[j], j))[:max(0, size - (n - old))]
                chosen = set(chosen) | set(range(max(old, n - size), n))
                movers = iter(sorted(j for j in chosen if j >= size))
                now = [j if j in chosen else next(movers) for j in range(size)]
                now = torch.tensor(now, device="cuda")
                where[b, g, :size] = now
                for h in mine:
                    taken = weights[h, rows[now]].clone()
                    weights[h, rows] = 0.0
                    weights[h, rows[:size]] = taken
        out = [None] * (2 if _dtype(case) == "fp4" else len(_buffers(s)))
        return [*out, weights, torch.tensor([min(n, keep) for n in lengths], device="cuda"),
                where if case["per_head"] else where[:, 0]]

    queries = s["new_queries"].to(wide)
    keys = _exact_stored(s, "key")
    if kind == "weights":
        total, first = s["weights"].to(wide), 0
        for b, (length, count) in enumerate(zip(lengths, chunks)):
            rows = rows_of(b)
            hidden = torch.arange(length, device="cuda") > (length - count + torch.arange(count, device="cuda"))[:, None]
            for h in range(heads):
                kv = h * kv_heads // heads
                logits = queries[first:first + count, h] @ keys[rows, kv].T / math.sqrt(dim)
                share = torch.exp(logits - s["lse"][first:first + count, h].to(wide)[:, None])
                total[kv, rows] += torch.where(hidden, 0.0, share).sum(0)
            first += count
        return total

    values = _exact_stored(s, "value")
    outs, sums = [], []
    first = 0
    for b, (length, count) in enumerate(zip(lengths, chunks)):
        at, rows = torch.arange(length, device="cuda"), rows_of(b)
        q = queries[first:first + count]
        out = torch.empty_like(q)
        lse = torch.empty((count, heads), device="cuda", dtype=wide)
        if kind == "selected":
            lists = s["indices"][first:first + count]
        for h in range(heads):
            kv = h * kv_heads // heads
            if kind == "attention":
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
