"""Registers of the attention over packed sequences, from the metadata of the built library: 2 waves per SIMD up to head_dim 128, and an instance that
begins to spill in its loop gets slower with every result unchanged."""
import os
import re

import pytest

import lvar_amd.build as build
from test_registers import _code_objects, _kernels


@pytest.fixture(scope="module")
def kernels():
    if not os.path.exists(build.LIB_PATH):
        build.build_library()
    found = {}
    for elf in _code_objects(open(build.LIB_PATH, "rb").read()):
        for k in _kernels(elf):
            m = re.match(r"_ZN4lvar\d+(packed_fwd_kernel|packed_dq_kernel|packed_dkv_kernel|packed_fwd_join_kernel|packed_dq_join_kernel|packed_dkv_join_kernel|pages_\w+_kernel|norm_axes_bwd_kernel|axis_tables_kernel)(?:I((?:L[ib]\d+E)+)E)?",
                         k[".name"])
            if m:
                found[(m[1],) + tuple(int(x) for x in re.findall(r"L[ib](\d+)E", m[2] or ""))] = k
    return found


def test_every_instance_is_built(kernels):
    count = lambda name: sum(k[0] == name for k in kernels)  # noqa: E731
    assert count("packed_fwd_kernel") == count("packed_dq_kernel") == 6 and count("packed_dkv_kernel") == 3
    assert count("packed_fwd_join_kernel") == count("packed_dq_join_kernel") == count("packed_dkv_join_kernel") == 3
    assert count("pages_alloc_kernel") == count("pages_fork_find_kernel") == 3 and count("norm_axes_bwd_kernel") >= 5


def test_spilled_registers(kernels):
    # packed_fwd_kernel<D, waves, SPLIT>: 256 columns, a few per tile
    may = {("packed_fwd_kernel", 256, 4, 0): 4, ("packed_fwd_kernel", 256, 4, 1): 18}
    spilled = {n: k[".vgpr_spill_count"] for n, k in kernels.items() if k.get(".vgpr_spill_count", 0) > may.get(n, 0)}
    assert not spilled, spilled


def test_waves_per_simd(kernels):
    for n, k in kernels.items():
        if n[0] in ("packed_fwd_kernel", "packed_dq_kernel", "packed_dkv_kernel") and n[1] <= 128:
            assert k[".vgpr_count"] <= 256, n
