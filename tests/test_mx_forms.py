"""Which kernels the products of microscaled numbers launch: tests/cpp/mx_forms.cpp, built by __graft_entry__.build(), stands in for the runtime,
so no device is needed."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "mx_forms.bin")


def launches(*lines):
    """each call's kernels and workgroups, as one text"""
    assert os.path.exists(BIN), "build it with __graft_entry__.build()"
    res = subprocess.run([BIN], input="".join(line + "\n" for line in lines), stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, "%d %s" % (res.returncode, res.stderr)
    return res.stdout.splitlines()


# a few rows in one launch, rows that are quantised before, sums in one part
@pytest.mark.parametrize("first", ["product 1 4096 1000 0 0", "linear 1 4096 1000 0 0", "linear 300 4096 5000 1 0", "product 300 512 5000 2 1"])
def test_a_context_has_memory_for_parts_from_its_first_product_on(first):
    """sums that are recorded then are shared by as many workgroups as those of the same call by itself: the same bits"""
    shared = "product 40 16384 1000 0 0"
    alone, = launches(shared)
    assert alone == "mx_tile_kernel<32,64,1,2,4> 128"          # 16 x 2 tiles in four parts
    assert launches("context", first, "capture 1", shared, "capture 0", shared)[3::2] == [alone, alone]
