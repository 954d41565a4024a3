"""The ``attend`` command on a 4-bit cache, and under a budget of cached keys."""

from __future__ import annotations

import pytest

from test_gpu_paged_command import _run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("head_dim", ["64", "128", "256"])
def test_attend_to_a_4_bit_cache(device, tmp_path, head_dim) -> None:
    t = _run(tmp_path, "--length", "700", "--steps", "3", "--batch", "2", "--k", "64", "--cache-dtype", "fp4",
             "--head-dim", head_dim, "--heads", "8", "--kv-heads", "2")
    assert list(t["keys"]) == [701, 701, 702, 702, 703, 703]
    assert (t["selected"] == 64).all()
    assert ((t["mass_kept_mean"] > 64 / 703) & (t["mass_kept_mean"] < 1)).all()
    every = _run(tmp_path, "--length", "700", "--steps", "2", "--k", "800", "--cache-dtype", "fp4", "--head-dim", head_dim)
    assert (every["selected"] == every["keys"]).all()
    assert (every["mass_kept_mean"] - 1).abs().max() < 1e-4
    assert every["output_error"].max() < 2**-7       # two roundings to bf16 apart


@pytest.mark.parametrize("dtype", ["bf16", "fp8", "fp4"])
def test_attend_under_a_budget(device, tmp_path, dtype, capsys) -> None:
    """The cache never passes the budget; the selection of every key that is left equals
    the dense attention, so the index moves with the keys."""

    t = _run(tmp_path, "--length", "500", "--steps", "40", "--batch", "2", "--k", "600", "--budget", "160", "--page-size", "16",
             "--cache-dtype", dtype, "--heads", "8", "--kv-heads", "2")
    assert t["keys"].max() == 160 and t["keys"].min() == 140
    assert (t["selected"] == t["keys"]).all()
    assert (t["mass_kept_mean"] - 1).abs().max() < 1e-4
    assert t["output_error"].max() < 2**-7
    assert "evicted 2 times to a budget of 160 keys" in capsys.readouterr().out
    few = _run(tmp_path, "--length", "500", "--steps", "8", "--k", "32", "--budget", "400", "--cache-dtype", dtype)
    assert (few["selected"] == 32).all() and (few["mass_kept_mean"] > 32 / 400).all()  # better than keys at random
