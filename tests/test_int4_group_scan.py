"""Sums over the group sizes of a product on 4-bit weights: their arithmetic on the CPU (tests/host_checks/group_scan.hip), and a call
of the largest number of rows whose groups all claim them."""

import os
import subprocess

import pytest
import torch

import gpu_ragged_dot_amd as rd
from gpu_ragged_dot_amd import _capi
from gpu_ragged_dot_amd.int4 import _ragged_dot_int4

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "gpu_ragged_dot_amd", "csrc")
EXE = os.path.join(ROOT, "tests", "host_checks", "group_scan")


def test_sums_of_group_sizes_stay_within_32_bits():
    r = subprocess.run(["make", "-C", CSRC, os.path.relpath(EXE, CSRC)], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    r = subprocess.run([EXE], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout + r.stderr
    assert r.stdout.startswith("group_scan ok ") and int(r.stdout.split()[2]) > 1_000_000


@pytest.mark.gpu
@pytest.mark.parametrize("kernel", [_capi.RD_INT4_STREAM, _capi.RD_INT4_TILES], ids=["stream", "tiles"])
def test_the_most_rows_in_groups_that_each_claim_them_all(kernel):
    m, g, k, n = (1 << 25) - 1, 200, 8, 8
    print(f"int4 m {m} g {g} kernel {kernel}", flush=True)
    gen = torch.Generator(device="cuda").manual_seed(0)
    q = torch.randint(0, 16, (g, k, n), generator=gen, dtype=torch.uint8, device="cuda")
    w = rd.pack_int4(q, torch.ones((g, 1, n), device="cuda").bfloat16())
    x = torch.randint(-2, 3, (m, k), generator=gen, dtype=torch.int8, device="cuda").bfloat16()  # products of small integers: exact
    sizes = torch.full((g,), m, dtype=torch.int32, device="cuda")
    sizes[0] = m - 1000
    sizes[150:] = 2 ** 31 - 1
    y = _ragged_dot_int4(x, w, sizes, kernel=kernel)
    for first, end, e in ((0, 5000, 0), (m // 2, m // 2 + 5000, 0), (m - 6000, m - 1000, 0), (m - 1000, m, 1)):
        assert torch.equal(y[first:end].float(), x[first:end].float() @ (q[e].float() - 8))
