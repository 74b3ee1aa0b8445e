"""The oracles of microscaled numbers and of a batch's pages against torch."""
import os
import subprocess
import sys


def test_the_oracles_are_the_plain_forms():
    """in a process of its own, as torch brings a HIP runtime along"""
    run = subprocess.run([sys.executable, "-u", os.path.join(os.path.dirname(os.path.abspath(__file__)), "mx_oracle_torch.py")], stdout=subprocess.PIPE,
                         stderr=subprocess.STDOUT, text=True, timeout=110)
    assert run.returncode == 0 and "fine" in run.stdout, run.stdout[-2000:]
