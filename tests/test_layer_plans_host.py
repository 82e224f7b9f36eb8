"""What the tests of the layers' kernels on the GPU rest on, without one: the sizes of test_gpu_gemm_i8_tiles.py make the product take every
shape of tiles that it has, and the recurrence in torch is the one in numpy."""
import re
from pathlib import Path

import numpy as np
import pytest

from kv_helpers import BF16, F16, F32
from layer_helpers import linear_ref, linear_ref_on, tile_plan
from test_gpu_gemm_i8_tiles import BATCHES, BESIDE, SHAPES


def shapes():
    """The shapes as the kernel's source lists them."""
    source = (Path(__file__).resolve().parent.parent / "halo_amd" / "csrc" / "k_gemm_i8.hip").read_text()
    listed = re.search(r"kShapes\[\] = \{(.*)\};", source).group(1)
    return [tuple(map(int, s)) for s in re.findall(r"\{(\d+), (\d+), (\d+)\}", listed)]


def test_every_shape_of_tiles_is_tested():
    """Each over more steps than two rounds of its stages, the last one ragged, and with ragged last tiles."""
    had = {}
    for want, rows, cols, n_vec in SHAPES:
        shape, tiles_n, tiles_t, each_n, each_t = tile_plan(shapes(), rows, cols, n_vec)
        assert shape[:2] == want, (rows, cols, n_vec, shape)
        had.setdefault(shape, []).append((rows % each_n, tiles_t == 1 or n_vec % each_t))
        assert -(-cols // 128) >= 2 * shape[2] + 1 and cols % 128 and cols % 16, (rows, cols, n_vec)
    assert sorted(had) == sorted(shapes())
    for shape, ends in had.items():
        assert any(n for n, _ in ends), f"{shape}: no last tile with fewer channels"
        assert any(t for _, t in ends), f"{shape}: no last tile with fewer vectors"
    # the rows that are compared between calls meet many shapes
    rows, cols = BESIDE
    assert len({tile_plan(shapes(), rows, cols, n)[0] for n in BATCHES if n > 16}) >= 6


@pytest.mark.parametrize("t", [F32, F16, BF16])
def test_recurrence_in_torch_is_the_one_in_numpy(t):
    import torch

    rng = np.random.default_rng(t)
    q, k, v = rng.standard_normal((9, 3, 5)), rng.standard_normal((9, 3, 5)), rng.standard_normal((9, 3, 4))
    decay = (-3 * rng.uniform(0, 1, (9, 3))).astype(np.float32)
    decay[4, 1], decay[6, 2], v[7, 0, 1] = -np.inf, 0.25, np.nan
    state = rng.standard_normal((3, 5, 4)).astype(np.float32)
    want = linear_ref(t, q, k, v, decay, state, 0.5)
    got = linear_ref_on(t, *(torch.from_numpy(x).double() for x in (q, k, v, decay, state)), 0.5)
    for w, g in zip(want, got):
        assert np.allclose(w, g.numpy(), rtol=1e-13, atol=1e-300, equal_nan=True)
