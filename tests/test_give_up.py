"""CPU check of the kernels' source: a kernel whose waits gave up leaves what it has started (copies into shared memory, products into tensor
memory) time to end before it gives the memory back."""
import re

import pytest

from test_launch_order import KERNELS

OWNERS = [(p, n, b) for p, n, b in KERNELS if "tcgen05.dealloc" in b]


def test_the_kernels_with_tensor_memory_are_found():
    names = {n for _, n, _ in OWNERS}
    assert {"k_grouped_mma", "k_gateup_wide", "k_down_resident", "k_ffn_fused_small", "k_attn_prefill", "k_linear_tc"} <= names


@pytest.mark.parametrize("path,name,body", OWNERS, ids=[n for _, n, _ in OWNERS])
def test_given_up_work_may_land_before_its_memory_goes(path, name, body):
    end = body[body.rindex("__syncthreads()"):body.index("tcgen05.dealloc")]
    wait = re.search(r"if \([^\n]*abort_flag\)[^}]*for \(int i = 0; i < (\d+); i\+\+\) __nanosleep\((\d+)\);", end)
    assert wait and int(wait.group(1)) * int(wait.group(2)) >= 100_000
