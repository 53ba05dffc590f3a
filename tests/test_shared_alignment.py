"""Shared arrays of the routing and 4-bit kernels that are accessed through a
wider type say so: their element type or an alignas is as wide as the access
(a static check; a misplaced array faults on the GPU only when the linker
happens to put it off the boundary)."""
from __future__ import annotations

import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "megacu_b200", "csrc", "kernels")
SIZES = {"uint2": 8, "uint4": 16, "float4": 16, "bytes32": 32, "float2": 8, "int4": 16}


def narrow_arrays(text):
    """(array, bytes of an access, its alignment) of each array accessed wider than it is aligned."""
    found = []
    for body in re.split(r"\n__global__ ", text)[1:]:
        body = body.split("\n}\n", 1)[0]
        for align, kind, name in re.findall(
                r"__shared__ (?:alignas\((\d+)\) )?([\w:]+) (\w+)\[", body):
            have = max(int(align or 0), SIZES.get(kind.split("::")[-1], 4))
            for wide in re.findall(
                    r"reinterpret_cast<(\w+)(?: const)? \*>\(&?" + name + r"\b", body):
                if SIZES.get(wide, 0) > have:
                    found.append((name, SIZES[wide], have))
    return found


@pytest.mark.parametrize("path", ["fp4_quant_kernel.cuh", "fp4_gemm_kernel.cuh",
                                  "moe_kernels.cuh"])
def test_wide_accesses_are_aligned(path):
    assert narrow_arrays(open(os.path.join(KERNELS, path)).read()) == []


def test_a_narrow_array_is_found():
    text = ("\n__global__ void k() {\n  __shared__ std::uint32_t a[4][2];\n"
            "  x = *reinterpret_cast<uint2 const *>(a[i]);\n}\n")
    assert narrow_arrays(text) == [("a", 8, 4)]
    assert narrow_arrays(text.replace("__shared__ ", "__shared__ alignas(8) ")) == []
