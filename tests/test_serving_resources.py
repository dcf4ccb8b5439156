"""CPU tests of the compiler's resource report of the serving kernels (the "serving" part of fa2/kernel_resources.json, written
by csrc/build.py): every instance is there, as many workgroups fit a CU as the kernels are compiled for and the grids count on, and
the instances that spill registers to scratch are the known ones.
"""

import json
import os

import pytest

from fa2 import _lib

RESOURCES = os.path.join(os.path.dirname(_lib.LIB_PATH), "kernel_resources.json")
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libfa2_fwd.so not built")


def serving():
    return list(json.load(open(RESOURCES))["serving"].values())


def workgroups_per_cu(head_dim, source, row_waves):
    """ragged_waves() of csrc/serve_launch.hpp"""
    if row_waves == 1:
        return 3 if head_dim <= 32 else 2
    return 2 if head_dim == 128 or source == 2 else 3 if source == 1 else 4


def test_every_instance_is_recorded():
    count = {}
    for r in serving():
        count[r["kernel"]] = count.get(r["kernel"], 0) + 1
    # fp16 and bf16, four head dims; sources (packed, 16-bit pages, e4m3 pages) and forms (32 rows, 128, 128 with the log-sum-exp)
    assert count == {"attn_ragged_kernel": 8 * 3 * 3, "attn_ragged_combine_kernel": 8 * 2, "rotary_kernel": 8,
                     "cache_write_kernel": 8 * 2, "cache_read_kernel": 8 * 2}


def test_as_many_workgroups_fit_a_cu_as_the_grids_count_on():
    for r in serving():
        if r["kernel"] == "attn_ragged_kernel":
            fit = workgroups_per_cu(r["head_dim"], r["source"], r["row_waves"])
            assert r["waves_per_simd"] >= fit and r["lds_bytes"] * fit <= 160 * 1024, r


def test_the_instances_that_spill():
    """128-row ones held to three and four workgroups a CU, and e4m3 pages at head_dim 128, whose raw rows wait in registers:
    a lane's spills are at most 20 registers. tests/test_gpu_serving_determinism.py runs each of them."""
    for r in serving():
        if r["vgpr_spills"]:
            assert r["kernel"] == "attn_ragged_kernel" and r["vgpr_spills"] <= 20, r
            known = (r["row_waves"] == 4 and r["source"] < 2 and r["head_dim"] in (16, 64)) or (
                r["source"] == 2 and r["head_dim"] == 128)
            assert known, r
