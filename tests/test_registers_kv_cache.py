"""Registers of the kernels around the paged cache, from the metadata of the built library: the key loops of the attention kernels are laid
out for 2 or 3 waves per SIMD, and an instance that spills there gets slower with every result unchanged."""
import os
import re

import pytest

import lvar_amd.build as build
from test_registers import _code_objects, _kernels


@pytest.fixture(scope="module")
def kernels():
    """{(kernel, template arguments): metadata}"""
    if not os.path.exists(build.LIB_PATH):
        build.build_library()
    found = {}
    for elf in _code_objects(open(build.LIB_PATH, "rb").read()):
        for k in _kernels(elf):
            m = re.match(r"_ZN4lvar\d+(paged_attn_kernel|paged_tile_kernel|paged_join_kernel|norm_rope_kernel|norm_rope_bwd_kernel|kv_read_kernel)I((?:L[ib]\d+E)+)E", k[".name"])
            if m:
                found[(m[1],) + tuple(int(x) for x in re.findall(r"L[ib](\d+)E", m[2]))] = k
    return found


def test_every_instance_is_built(kernels):
    count = lambda name: sum(k[0] == name for k in kernels)  # noqa: E731
    assert count("paged_attn_kernel") == 10 and count("paged_tile_kernel") == 10 and count("paged_join_kernel") == 6
    assert count("norm_rope_bwd_kernel") == 10 and count("kv_read_kernel") == 6


def test_spilled_registers(kernels):
    # paged_attn_kernel<D, NT, F8, waves per SIMD>: 256 columns of bf16 keep 64 registers each of keys, values and outputs
    may = {("paged_attn_kernel", 256, 1, 0, 2): 8}
    spilled = {n: k[".vgpr_spill_count"] for n, k in kernels.items() if k.get(".vgpr_spill_count", 0) > may.get(n, 0)}
    assert not spilled, spilled


def test_waves_per_simd(kernels):
    for n, k in kernels.items():
        if n[0] == "paged_attn_kernel":
            assert k[".vgpr_count"] <= 512 // n[4] // 8 * 8, n
        if n[0] == "paged_tile_kernel":
            assert k[".vgpr_count"] <= 256 and k[".group_segment_fixed_size"] <= 2048, n
