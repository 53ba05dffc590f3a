"""Every kernel that may start while the kernel before it still runs
(csrc/kernels/chained.cuh) waits for it before it touches global memory: a
start signal alone does not make earlier writes visible. A static check of the
kernels' sources: nothing that a pointer parameter or `p.<pointer>` names is
read or written above the kernel's own grid_wait()."""
from __future__ import annotations

import os
import re

import pytest

KERNELS = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                       "megacu_b200", "csrc", "kernels")
# Functions that access global memory through the parameters, and its pointers.
ACCESS = (r"local_expert<Id>\(|clear_rows\(|load16<|row_at\(|load_vec<|store_vec<|locate_rows\(|"
          r"\bload\(|tma_load|p\.(?:ids|histogram|counts|offsets|row_of_slot|slot_of_row|data|scales|"
          r"alphas|out)\b\s*\[")


def kernels(text):
    """(name, body) of each __global__ function."""
    for part in re.split(r"__global__ ", text)[1:]:
        body = part.split("\n}\n", 1)[0]
        name = re.search(r"(\w+_kernel)\(", body)
        if name:
            yield name.group(1), body


def early_accesses(body):
    """Accesses above the last grid_wait of the body, lambdas' bodies aside."""
    body = re.sub(r"//[^\n]*", "", body)
    assert "grid_wait();" in body
    head = body[:body.rindex("grid_wait();")]
    return re.findall(ACCESS, head)


@pytest.mark.parametrize("path", ["moe_kernels.cuh", "fp4_quant_kernel.cuh",
                                  "fp4_gemm_kernel.cuh"])
def test_kernels_wait_before_their_first_access(path):
    found = dict(kernels(open(os.path.join(KERNELS, path)).read()))
    assert found
    for name, body in found.items():
        assert early_accesses(body) == [], name


def test_an_early_access_is_found():
    assert early_accesses("k_kernel(p) {\n  x = p.ids[0];\n  grid_wait();") != []
    assert early_accesses("k_kernel(p) {\n  grid_wait();\n  x = p.ids[0];") == []
