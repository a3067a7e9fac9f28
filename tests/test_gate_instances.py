"""The gate's kernels in the built library are those that a call can reach."""

import os
import re

from gpu_ragged_dot_amd import _capi

BYTES = {"f": 4, "DF16_": 2, "t": 2}  # float, float16, bfloat16 as 16 bits


def test_rows_in_whole_pieces_have_registers_for_one():
    path = os.path.join(os.path.dirname(_capi.__file__), "csrc", "libragged_dot_hip.so")
    with open(path, "rb") as f:
        names = re.findall(rb"moe_gate_rows_kernelI(f|DF16_|t)Li(\d+)ELb([01])E", f.read())
    found = {(t.decode(), int(per), vec == b"1") for t, per, vec in names}
    # every number of registers by element; by pieces of 16 bytes where they hold one
    assert found == {(t, per, vec) for t, size in BYTES.items() for per in (1, 4, 8, 16, 32) for vec in (False, True) if not vec or per * size >= 16}
