"""Which row tile each workgroup of paged attention's kernel for many rows takes, on the CPU: the rule's own code
(csrc/kernels/prompt_tiles.h) in a host program that asks for every tile of ragged batches, sequences with more queries
than keys among them (tests/sanitize/prompt_tiles_check.cc)."""
import os
import subprocess

HERE = os.path.join(os.path.dirname(os.path.abspath(__file__)), "sanitize")


def test_every_tile_is_found_once():
    build = subprocess.run(["make", "-C", HERE, "_build/prompt_tiles_check"], capture_output=True, text=True, timeout=300)
    assert build.returncode == 0, build.stdout[-3000:] + build.stderr[-3000:]
    run = subprocess.run([os.path.join(HERE, "_build", "prompt_tiles_check")], capture_output=True, text=True, timeout=300)
    assert run.returncode == 0, run.stdout[-3000:] + run.stderr[-3000:]
    assert "prompt tiles:" in run.stdout and "runtime error" not in run.stderr
