"""Products of torch's tensors that are views of one memory."""
import os
import subprocess
import sys

import pytest


@pytest.mark.gpu
def test_views_of_one_memory():
    """in a process of its own, with torch imported first"""
    run = subprocess.run([sys.executable, "-u", os.path.join(os.path.dirname(os.path.abspath(__file__)), "mx_torch_views.py")], stdout=subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True, timeout=110)
    assert run.returncode == 0 and "fine" in run.stdout, run.stdout[-2000:]
