"""What the key/value cache's calls ask of the runtime: tests/cpp/kv_host_calls.cpp, built by __graft_entry__.build(), stands in for it, so
no device is needed."""
import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "kv_host_calls.bin")


@pytest.mark.parametrize("case", ["no_tokens", "workspace_device", "pages_are_clear", "many_rows", "recording"])
def test_what_calls_ask_of_the_runtime(case):
    assert os.path.exists(BIN), "build it with __graft_entry__.build()"
    res = subprocess.run([BIN, case], stdout=subprocess.PIPE, stderr=subprocess.PIPE, text=True, timeout=100)
    assert res.returncode == 0, "%d %s" % (res.returncode, res.stderr)
