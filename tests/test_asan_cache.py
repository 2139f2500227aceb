"""The argument validation of the cache's C entry points under the address and undefined-behaviour sanitizers (tests/asan/cache/Makefile,
target `asan`).  Needs no GPU; any finding aborts the program."""
import os
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_make_asan(tmp_path):
    out = subprocess.run(["make", "-C", os.path.join(ROOT, "tests", "asan", "cache"), "asan", "OUT=" + str(tmp_path)], capture_output=True, text=True)
    assert out.returncode == 0, out.stdout[-3000:] + out.stderr[-3000:]
    assert "\nok" in out.stdout
