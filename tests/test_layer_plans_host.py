"""What the tests of the layers' kernels on the GPU rest on, without one: the sizes of test_gpu_gemm_i8_tiles.py make the product take every
shape of tiles that it has."""
import re
from pathlib import Path

from layer_helpers import tile_plan
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
