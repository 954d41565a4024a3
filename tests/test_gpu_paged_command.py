"""The ``attend`` command: append, indexer, selected and dense attention together."""

from __future__ import annotations

import pandas as pd
import pytest

from dsa_amd import cli

pytestmark = pytest.mark.gpu


def _run(tmp_path, *args: str) -> pd.DataFrame:
    cli.main(["attend", "--output", str(tmp_path), *args])
    return pd.read_csv(tmp_path / "attention_steps.csv")


@pytest.mark.parametrize("args", [
    ("--head-dim", "128"),
    ("--head-dim", "64", "--cache-dtype", "fp8", "--page-size", "16", "--heads", "6", "--kv-heads", "3"),
    ("--head-dim", "256", "--cache-dtype", "fp16", "--heads", "2", "--kv-heads", "1"),
])
def test_attend(device, tmp_path, args) -> None:
    print(f"attend {args}", flush=True)
    t = _run(tmp_path, "--length", "700", "--steps", "3", "--batch", "2", "--k", "64", *args)
    assert list(t["keys"]) == [701, 701, 702, 702, 703, 703]
    assert (t["selected"] == 64).all()
    assert ((t["mass_kept_mean"] > 64 / 703) & (t["mass_kept_mean"] < 1)).all()   # better than keys at random
    assert ((t["mass_kept_least"] >= 0) & (t["mass_kept_least"] <= t["mass_kept_mean"] + 1e-6)).all()
    assert (t["output_error"] >= 0).all()            # 0 where one key has all of the mass
    every = _run(tmp_path, "--length", "700", "--steps", "2", "--k", "800", *args)
    assert (every["selected"] == every["keys"]).all()
    assert (every["mass_kept_mean"] - 1).abs().max() < 1e-4
    assert every["output_error"].max() < 2**-7       # two roundings to bf16 apart
