"""Refusals of the token and AdamW entry points at the borders of their arguments' types; no GPU."""
import ctypes as C
import subprocess
import sys

import pytest

from illumina import _lib
from tests.conftest import PKG_DIR
from tests.test_tokens_host import refused


def rotary_args(**over):
    a = _lib.RotaryArgs(precision=0, batch=1, tokens=4, head_dim=16, pairs=8, axes=2, positions=0x1000, turns=0x1000, axis=0x1000)
    a.first.x = a.first.y = 0x1000
    a.first.heads = 2
    for k, v in over.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("pairs", [2 ** 30, 2 ** 30 + 1, 2 ** 31 - 1, -1, -2 ** 31])
def test_rotary_pairs_whose_double_leaves_the_type(pairs):
    # in a process of its own: a count that passed the check would divide by zero in the launch's sizes
    code = f"""
import ctypes as C, sys
sys.path[:0] = [{PKG_DIR!r}]
from illumina import _lib
a = _lib.RotaryArgs(precision=0, batch=1, tokens=4, head_dim=16, pairs={pairs}, axes=2, positions=0x1000, turns=0x1000, axis=0x1000)
a.first.x = a.first.y = 0x1000
a.first.heads = 2
print(_lib.lib().illumina_op_rotary(C.byref(a), None), _lib.lib().illumina_last_error().decode())
"""
    run = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True)
    assert run.returncode == 0 and run.stdout.startswith(f"{_lib.INVALID_ARG} ") and "pairs" in run.stdout
