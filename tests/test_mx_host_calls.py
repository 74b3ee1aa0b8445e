"""What the calls on microscaled numbers and on a batch's pages ask of the runtime, and refuse: tests/cpp/mx_host_calls.cpp, built by
__graft_entry__.build(), stands in for it, so no device is needed."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "mx_host_calls.bin")


@pytest.mark.parametrize("case", ["refusals", "launches", "devices", "recording"])
def test_what_calls_ask_of_the_runtime(case):
    assert os.path.exists(BIN), "build it with __graft_entry__.build()"
    res = subprocess.run([BIN, case], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, "%d %s" % (res.returncode, res.stderr)
