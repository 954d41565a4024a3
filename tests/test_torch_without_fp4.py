"""A torch that has no 4-bit type imports the package and has everything but 4-bit
caches.  (In a process of its own, whose torch the types are taken from.)"""

from __future__ import annotations

import subprocess
import sys
from pathlib import Path

_PROGRAM = """
import torch
del torch.float4_e2m1fn_x2, torch.float8_e8m0fnu
import dsa_amd
from dsa_amd import _lib, approx, certified, cli, decode, eviction, metrics, paged, progressive_kernel, sidecar, temporal

def refuses(match, call, *args, **kw):
    try:
        call(*args, **kw)
    except ValueError as error:
        assert match in str(error), error
    else:
        raise AssertionError(match)

assert paged.FP4 is None and _lib.dtype_code(torch.bfloat16) == _lib.DTYPE_BF16
for dtype in (torch.bfloat16, torch.float16, torch.float8_e4m3fn):
    refuses("GPU", paged.new_cache, 2, 16, 2, 64, dtype=dtype, device="cpu")
refuses("BF16", paged.new_cache, 2, 16, 2, 64, dtype=torch.uint8, device="cpu")
refuses("BF16", paged.new_cache, 2, 16, 2, 64, dtype=None, device="cpu")
args = cli.build_parser().parse_args(["attend", "--output", "nowhere", "--cache-dtype", "fp4"])
refuses("4-bit type", args.function, args)
print("whole")
"""


def test_everything_else_is_there() -> None:
    done = subprocess.run([sys.executable, "-c", _PROGRAM], capture_output=True, text=True, timeout=300,
                          cwd=Path(__file__).resolve().parents[1])
    assert done.returncode == 0 and done.stdout.strip() == "whole", done.stderr
