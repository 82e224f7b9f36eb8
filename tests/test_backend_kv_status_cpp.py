"""What a stream's wait() throws where its ops found several kinds of faults on the device, through the C++ test program
tests/cpp/backend_kv_status.cpp."""
import os
import subprocess
import sys

import pytest

BIN = os.path.join(os.path.dirname(os.path.abspath(__file__)), "cpp", "backend_kv_status")


def _need_binary():
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} is missing: build it with __graft_entry__.build()")


def test_binary_links_the_library():
    _need_binary()
    r = subprocess.run([BIN, "--list"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0 and "backend_kv_status" in r.stdout, r.stdout + r.stderr


@pytest.mark.gpu
def test_every_kind_is_thrown():
    _need_binary()
    print("[case] backend_kv_status (C++ adapter)", flush=True)
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=120)
    sys.stdout.write(r.stdout[-4000:])
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
