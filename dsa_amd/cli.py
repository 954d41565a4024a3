"""Command-line driver: collect score traces on the GPU and replay them.

Mirrors the reference's ``temporal-dsa analyze`` entry point (reference
cli.py:42-103): it finds ``.npz`` traces under ``--trace-roots``, replays each
with the sweep of the ``replay`` section of a YAML config (``k_values``,
``block_sizes``, ``gamma_sigma``, ``key_bytes``, ``metadata_bytes_per_block``,
optional ``calibrated_margins`` per layer, or a ``--margin-file``), and writes
``temporal_stats.csv``, ``block_stats.csv`` (reference cli.py:17-20,55-58,
replay.py:403-474), ``replay_rows.csv`` and the aggregated
``replay_summary.csv`` to ``--output``.  The replay and the statistics run in
the HIP kernels (:mod:`dsa_amd.replay`).  The reference's graphs, hardware
extrapolation and verdict report are analysis presentation and stay with the
reference's tools, which read the traces and CSVs written here.

``collect`` writes a synthetic decode trajectory's dense score trace (AR(1)
queries, N(0,1) keys, one key appended per step) in the reference's format:

    python -m dsa_amd.cli collect --output traces/synthetic.npz --length 16384 --steps 64
    python -m dsa_amd.cli analyze --trace-roots traces --output results --config configs.yaml

``attend`` runs the attention that the indexer is there for: a synthetic prompt is
written into a paged cache (:mod:`dsa_amd.paged`) and attended to, then each
decode step appends its token, attends to the positions the indexer's top-k
names and to every position, and writes what of the softmax's mass the selection
kept, how far its output is from the dense one's, and both times:

    python -m dsa_amd.cli attend --output results --length 32768 --steps 8 --k 2048 --cache-dtype fp8
"""

from __future__ import annotations

import argparse
import json
import math
from pathlib import Path

import numpy as np
import yaml


def _trace_paths(roots: list[Path]) -> list[Path]:
    paths: list[Path] = []
    for root in roots:
        paths.extend([root] if root.is_file() and root.suffix == ".npz" else sorted(root.rglob("*.npz")))
    if not paths:
        raise FileNotFoundError("no .npz traces found")
    return paths


def analyze(args: argparse.Namespace) -> None:
    import pandas as pd

    from .replay import aggregate_rows, block_temporal_stats, replay_trace_rows, temporal_stats
    from .trace import load_trace

    config = yaml.safe_load(args.config.read_text(encoding="utf-8")) if args.config else {}
    replay = dict(config.get("replay", {}))
    if args.margin_file:
        payload = json.loads(args.margin_file.read_text(encoding="utf-8"))
        replay["calibrated_margins"] = {
            str(layer): {int(block): value for block, value in blocks.items()}
            for layer, blocks in payload["margins"].items()
        }
    k_values = replay.get("k_values", [2048])
    block_sizes = replay.get("block_sizes", [16, 32, 64, 128])
    gammas = replay.get("gamma_sigma", [0.0, 0.25, 0.5, 1.0])
    rows: list[dict] = []
    temporal_frames, block_frames = [], []
    for path in _trace_paths(args.trace_roots):
        trace = load_trace(path)
        temporal_frames.append(temporal_stats(trace, k_values))
        block_frames.append(block_temporal_stats(trace, block_sizes, k_values))
        margins = replay.get("calibrated_margins", {}).get(str(trace.layer))
        if margins:
            margins = {int(b): float(v) for b, v in margins.items()}
        rows.extend(replay_trace_rows(
            trace, k_values=k_values, block_sizes=block_sizes, gamma_sigma_values=gammas,
            key_bytes=replay.get("key_bytes", 256), metadata_bytes_per_block=replay.get("metadata_bytes_per_block", 8),
            absolute_margins=margins, wave=args.wave,
        ))
        print(f"replayed {path} ({trace.scores.shape[0] - 1} transitions)", flush=True)
    args.output.mkdir(parents=True, exist_ok=True)
    pd.concat(temporal_frames, ignore_index=True).to_csv(args.output / "temporal_stats.csv", index=False)
    pd.concat(block_frames, ignore_index=True).to_csv(args.output / "block_stats.csv", index=False)
    frame = pd.DataFrame(rows)
    frame.to_csv(args.output / "replay_rows.csv", index=False)
    aggregate_rows(frame).to_csv(args.output / "replay_summary.csv", index=False)
    print(f"wrote {len(frame)} rows to {args.output}", flush=True)


def collect(args: argparse.Namespace) -> None:
    import torch

    from .trace import collect_trace, save_trace

    gen = torch.Generator().manual_seed(args.seed)
    steps, length = args.steps, args.length
    device = torch.device("cuda", 0)
    keys = torch.randn(length + steps - 1, 128, generator=gen).to(torch.bfloat16).to(device)
    w = (torch.randn(64, generator=gen) / 8).to(device)
    q = torch.randn(64, 128, generator=gen) / math.sqrt(128)
    qs = []
    for _ in range(steps):
        qs.append(q.to(torch.bfloat16))
        q = args.rho * q + math.sqrt(1 - args.rho * args.rho) * torch.randn(64, 128, generator=gen) / math.sqrt(128)
    queries = torch.stack(qs).to(device)
    lengths = np.arange(length, length + steps)
    trace = collect_trace(queries, w, keys, lengths, layer=args.layer, workload="synthetic", prompt_id=str(args.seed),
                          metadata={"rho": args.rho, "seed": args.seed})
    save_trace(args.output, trace)
    print(f"wrote {args.output}: {steps} steps, lengths {length}..{length + steps - 1}", flush=True)


def attend(args: argparse.Namespace) -> None:
    import pandas as pd
    import torch

    from . import decode, eviction, paged

    if args.budget is not None and args.budget < 2:
        raise ValueError("the budget must be at least 2 keys")
    if args.steps < 1 or args.length < 1 or args.batch < 1 or args.k < 1:
        raise ValueError("length, steps, batch and k must be at least 1")
    if args.cache_dtype == "fp4" and paged.FP4 is None:
        raise ValueError("this torch has no 4-bit type (float4_e2m1fn_x2)")
    device = torch.device("cuda", 0)
    gen = torch.Generator(device).manual_seed(args.seed)
    batch, heads, kv_heads, dim = args.batch, args.heads, args.kv_heads, args.head_dim
    longest = args.length + args.steps
    columns = -(-longest // args.page_size)
    dtype = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp8": torch.float8_e4m3fn,
             "fp4": paged.FP4}[args.cache_dtype]
    cache = paged.new_cache(batch * columns, args.page_size, kv_heads, dim, dtype=dtype, device=device)
    table = torch.randperm(batch * columns, generator=gen, device=device).to(torch.int32).view(batch, columns)
    # A token's keys of every head share a part, which is the indexer's key and which
    # the rotation leaves alone; the queries look for the part of some earlier token.
    rope_dim = dim // 4
    shared = min(dim - rope_dim, 128)

    def normal(*shape: int) -> torch.Tensor:
        return torch.randn(shape, generator=gen, device=device)

    def tokens_of(n: int):
        part = normal(batch, n, shared)
        keys = 0.5 * normal(batch, n, kv_heads, dim)
        keys[..., rope_dim:rope_dim + shared] += part[:, :, None]
        return part, *(x.reshape(batch * n, kv_heads, dim).to(cache.row_dtype) for x in (keys, normal(*keys.shape)))

    def queries_of(parts: torch.Tensor, n: int) -> torch.Tensor:
        wanted = parts[:, torch.randint(parts.shape[1], (n,), generator=gen, device=device)]
        q = 0.5 * normal(batch, n, heads, dim)
        q[..., rope_dim:rope_dim + shared] += 1.5 * wanted[:, :, None]
        return q.reshape(batch * n, heads, dim).to(cache.row_dtype)

    index_keys = torch.zeros(batch, longest, 128, device=device, dtype=torch.bfloat16)
    index_weights = torch.full((batch, 64), 1 / 64, device=device)
    sequences = torch.arange(batch, device=device)

    def write(first: int, n: int, cached: int):
        """Appends tokens first .. first + n of every sequence behind its cached keys; their
        rotated queries."""

        part, keys, values = tokens_of(n)
        index_keys[:, cached:cached + n, :shared] = part.to(torch.bfloat16)
        places = torch.arange(cached, cached + n, device=device).repeat(batch)
        rows = paged.cache_rows(cache, table, places, sequences.repeat_interleave(n))
        positions = torch.arange(first, first + n, device=device).repeat(batch)
        queries = queries_of(index_keys[:, :cached + n, :shared].float(), n)
        plain = queries[:, :, rope_dim:rope_dim + shared]
        return paged.append(cache, keys, values, rows, positions, queries=queries, rope_dim=rope_dim), plain

    def timed(call):
        call()  # the first call of a kernel loads it
        start, stop = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        start.record()
        out = call()
        stop.record()
        stop.synchronize()
        return out, 1e3 * start.elapsed_time(stop)

    queries, _ = write(0, args.length, 0)
    lengths = torch.full((batch,), args.length, dtype=torch.int32, device=device)
    (_, prompt_lse), prompt_us = timed(lambda: paged.attention(queries, cache, table, lengths, return_lse=True))
    cached, evictions, weights = args.length, 0, None
    if args.budget is not None:  # the prompt's own rows say first what its keys are worth
        weights = eviction.new_weights(cache)
        eviction.accumulate_weights(weights, queries, cache, table, lengths, prompt_lse)
    print(f"prompt: {batch} x {args.length} tokens, {prompt_us:.0f} us of attention", flush=True)
    frames = []
    for step in range(args.steps):
        if args.budget is not None and cached >= args.budget:
            # to seven eighths of the budget, so that not every step evicts
            cached = max(1, args.budget - args.budget // 8 - 1)
            lengths, kept = eviction.evict(cache, table, lengths, weights, cached, recent=cached // 8)
            index_keys[:, :cached] = index_keys.gather(1, kept[..., None].expand(-1, -1, 128))
            evictions += 1
        queries, plain = write(args.length + step, 1, cached)
        cached += 1
        lengths = lengths + 1
        index_queries = torch.zeros(batch, 64, 128, device=device, dtype=torch.bfloat16)
        index_queries[..., :shared] = plain[:, torch.arange(64, device=device) * heads // 64].to(torch.bfloat16)
        chosen = decode.indexer_topk(index_queries, index_weights, index_keys[:, :cached].contiguous(), args.k)
        (few, few_lse), few_us = timed(
            lambda: paged.selected_attention(queries, cache, table, lengths, chosen, return_lse=True))
        (full, full_lse), full_us = timed(
            lambda: paged.attention(queries, cache, table, lengths, return_lse=True))
        if weights is not None:
            eviction.accumulate_weights(weights, queries, cache, table, lengths, full_lse)
        mass = torch.exp(few_lse - full_lse)
        off = torch.linalg.vector_norm(few.float() - full.float(), dim=(1, 2)) / torch.linalg.vector_norm(full.float(), dim=(1, 2))
        frames.append(pd.DataFrame({
            "step": step, "sequence": range(batch), "keys": cached, "selected": (chosen >= 0).sum(1).cpu(),
            "mass_kept_mean": mass.mean(1).cpu(), "mass_kept_least": mass.amin(1).cpu(), "output_error": off.cpu(),
            "selected_us": few_us, "dense_us": full_us}))
    frame = pd.concat(frames, ignore_index=True)
    args.output.mkdir(parents=True, exist_ok=True)
    frame.to_csv(args.output / "attention_steps.csv", index=False)
    print(frame.drop(columns=["step", "sequence"]).mean().to_string(float_format=lambda x: f"{x:.4g}"), flush=True)
    if args.budget is not None:
        print(f"evicted {evictions} times to a budget of {args.budget} keys", flush=True)
    print(f"wrote {len(frame)} rows to {args.output}", flush=True)


def build_parser() -> argparse.ArgumentParser:
    parser = argparse.ArgumentParser(prog="dsa-amd")
    sub = parser.add_subparsers(dest="command", required=True)
    a = sub.add_parser("analyze", help="replay traces on the GPU and write the replay tables")
    a.add_argument("--trace-roots", type=Path, nargs="+", required=True)
    a.add_argument("--config", type=Path, default=None)
    a.add_argument("--output", type=Path, required=True)
    a.add_argument("--margin-file", type=Path)
    a.add_argument("--wave", type=int, default=1, help="blocks between dynamic threshold refreshes (1: the reference)")
    a.set_defaults(function=analyze)
    c = sub.add_parser("collect", help="write a synthetic decode trajectory's score trace")
    c.add_argument("--output", type=Path, required=True)
    c.add_argument("--length", type=int, default=16384)
    c.add_argument("--steps", type=int, default=64)
    c.add_argument("--rho", type=float, default=0.95)
    c.add_argument("--seed", type=int, default=1582)
    c.add_argument("--layer", type=int, default=0)
    c.set_defaults(function=collect)
    t = sub.add_parser("attend", help="attend to a paged cache by the indexer's selection and densely")
    t.add_argument("--output", type=Path, required=True)
    t.add_argument("--length", type=int, default=16384, help="tokens of the prompt")
    t.add_argument("--steps", type=int, default=16)
    t.add_argument("--batch", type=int, default=1)
    t.add_argument("--k", type=int, default=2048, help="positions that the indexer selects")
    t.add_argument("--heads", type=int, default=32)
    t.add_argument("--kv-heads", type=int, default=8)
    t.add_argument("--head-dim", type=int, default=128, choices=(64, 128, 256))
    t.add_argument("--page-size", type=int, default=64)
    t.add_argument("--cache-dtype", default="bf16", choices=("bf16", "fp16", "fp8", "fp4"))
    t.add_argument("--budget", type=int, default=None,
                   help="cached keys of a sequence: those of least accumulated attention weight are evicted")
    t.add_argument("--seed", type=int, default=1582)
    t.set_defaults(function=attend)
    return parser


def main(argv: list[str] | None = None) -> None:
    args = build_parser().parse_args(argv)
    args.function(args)


if __name__ == "__main__":
    main()
