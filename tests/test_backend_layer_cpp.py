"""The C++ Backend adapter's head norms, 8-bit products and linear attention (include/halo_mi355x_backend.hpp,
MiBackend::norm_rope, quantize_rows, gemm_i8 and linear_attention) through their C++ test program, tests/cpp/backend_layer.cpp."""
import os
import subprocess
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
BIN = os.path.join(ROOT, "tests", "cpp", "backend_layer")


def _need_binary():
    if not os.path.exists(BIN):
        pytest.fail(f"{BIN} is missing: build it with __graft_entry__.build()")


def test_binary_links_the_library():
    """Loads without a GPU: every symbol the adapter and the test use resolves."""
    _need_binary()
    r = subprocess.run([BIN, "--list"], capture_output=True, text=True, timeout=60)
    assert r.returncode == 0, r.stdout + r.stderr
    assert "backend_layer" in r.stdout


@pytest.mark.gpu
def test_layer_of_the_adapter_on_the_gpu():
    _need_binary()
    print("[case] backend_layer (C++ adapter)", flush=True)
    r = subprocess.run([BIN], capture_output=True, text=True, timeout=240)
    sys.stdout.write(r.stdout[-4000:])
    assert r.returncode == 0, r.stdout[-4000:] + r.stderr[-2000:]
