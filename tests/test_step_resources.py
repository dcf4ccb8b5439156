"""CPU tests of the compiler's resource report of the kernels of windows, common prefixes, normalised rotations and pages (the "step"
part of fa2/kernel_resources.json, written by csrc/build.py)."""

import json
import os

import pytest

from fa2 import _lib
from test_serving_resources import workgroups_per_cu

RESOURCES = os.path.join(os.path.dirname(_lib.LIB_PATH), "kernel_resources.json")
pytestmark = pytest.mark.skipif(not os.path.exists(_lib.LIB_PATH), reason="libfa2_fwd.so not built")


def kernels():
    return list(json.load(open(RESOURCES))["step"].values())


def test_every_instance_is_recorded():
    count = {}
    for r in kernels():
        count[r["kernel"], r.get("mode")] = count.get((r["kernel"], r.get("mode")), 0) + 1
    # fp16 and bf16, four head dims; of a window three sources, of a prefix and what is behind it the two of pages, and three forms each (32
    # rows, 128, 128 with the log-sum-exp); a window's pieces merge as all keys' do
    assert count == {("attn_ragged_kernel", 1): 8 * 3 * 3, ("attn_ragged_kernel", 2): 8 * 2 * 3, ("attn_ragged_kernel", 3): 8 * 2 * 3,
                     ("attn_ragged_combine_kernel", 2): 8 * 2, ("attn_ragged_combine_kernel", 3): 8 * 2, ("rotary_qk_kernel", None): 8,
                     ("cache_write_kernel", None): 8 * 2, ("pages_extend_kernel", None): 1, ("pages_count_kernel", None): 1,
                     ("pages_release_kernel", None): 1}


def test_as_many_workgroups_fit_a_cu_as_the_grids_count_on():
    for r in kernels():
        if r["kernel"] == "attn_ragged_kernel":
            fit = workgroups_per_cu(r["head_dim"], r["source"], r["row_waves"])
            assert r["waves_per_simd"] >= fit and r["lds_bytes"] * fit <= 160 * 1024, r


def test_the_instances_that_spill():
    """As with all keys: 128-row ones held to three and four workgroups a CU, and e4m3 pages at head_dim 128."""
    for r in kernels():
        if r.get("vgpr_spills"):
            assert r["kernel"] == "attn_ragged_kernel" and r["vgpr_spills"] <= 40, r
            known = (r["row_waves"] == 4 and r["source"] < 2 and r["head_dim"] in (16, 64)) or (
                r["source"] == 2 and r["head_dim"] == 128)
            assert known, r
