"""A 4-bit decoder through the C++ engine and model layers, prompts to sampled tokens
(tests/engine/token_selftest.cpp, built by build())."""
from __future__ import annotations

import os
import subprocess

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "engine", "_bin", "token_selftest")


def test_token_driver_built_and_linked():
    assert os.path.exists(BIN), "token_selftest not built: run __graft_entry__.build()"
    out = subprocess.run(["ldd", BIN], capture_output=True, text=True, check=True).stdout
    assert "not found" not in out, out


@pytest.mark.gpu
def test_token_selftest():
    print("token_selftest", flush=True)
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=110)
    print(r.stdout[-6000:], r.stderr[-2000:], flush=True)
    fails = [l for l in r.stdout.splitlines() if l.startswith("FAIL")]
    assert r.returncode == 0 and not fails, "\n".join(fails) or f"exit status {r.returncode}"
    assert " checks, 0 failures" in r.stdout
