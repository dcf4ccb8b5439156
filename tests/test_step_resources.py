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
        count[r["kernel"]] = count.get(r["kernel"], 0) + 1
    # fp16 and bf16, four head dims; of a window three sources and three forms (32 rows, 128, 128 with the log-sum-exp); of a prefix
    # the two of pages, and 32 rows for both passes, or 128 and 32, or 128, these with and without the log-sum-exp
    assert count == {"attn_ragged_kernel": 8 * 3 * 3, "attn_window_mixed_kernel": 8 * 2 * 2, "attn_shared_kernel": 8 * 2 * 5, "attn_shared_join_kernel": 8 * 3,
                     "rotary_qk_kernel": 8, "cache_write_kernel": 8 * 2, "pages_extend_kernel": 1, "pages_count_kernel": 1,
                     "pages_release_kernel": 1, "pages_release_once_kernel": 1}


def test_as_many_workgroups_fit_a_cu_as_the_grids_count_on():
    for r in kernels():
        if r["kernel"] in ("attn_ragged_kernel", "attn_window_mixed_kernel", "attn_shared_kernel"):
            fit = 2 if r["kernel"] != "attn_ragged_kernel" else workgroups_per_cu(r["head_dim"], r["source"], r["row_waves"])
            assert r["waves_per_simd"] >= fit and r["lds_bytes"] * fit <= 160 * 1024, r


def test_the_instances_that_spill():
    """Windows as with all keys: 128-row ones held to three and four workgroups a CU, and e4m3 pages at head_dim 128; two forms
    in one kernel at head_dim 128."""
    for r in kernels():
        if r.get("vgpr_spills"):
            if r["kernel"] in ("attn_window_mixed_kernel", "attn_shared_kernel"):
                assert r["head_dim"] == 128 and r["vgpr_spills"] <= (80 if r["source"] == 2 else 8), r
                continue
            assert r["kernel"] == "attn_ragged_kernel" and r["vgpr_spills"] <= 20, r
            known = (r["row_waves"] == 4 and r["source"] < 2 and r["head_dim"] in (16, 64)) or (
                r["source"] == 2 and r["head_dim"] == 128)
            assert known, r
