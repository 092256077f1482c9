"""bench.py refuses flags that the run it is asked for would ignore."""
import os
import subprocess
import sys


def test_kv_bits_belong_to_the_decode_bench():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "bench.py")
    done = subprocess.run([sys.executable, path, "--kv-bits", "4"], capture_output=True, text=True, timeout=120)
    assert done.returncode == 2 and "give --decode" in done.stderr
