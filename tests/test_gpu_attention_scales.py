"""ATTENTION where the blocks of V differ by more than fp32's range of exponents: the weights carry V's scale in their
exponent, the sum that divides does not, so each has to keep what the other would lose."""
import numpy as np
import pytest

from kv_helpers import BF16, F32, TYPE_NAMES, U, attention_bound, attention_ref, batch, to_type
from test_gpu_attention import setup
from test_gpu_kv_cache import OnGpu

pytestmark = pytest.mark.gpu


def far_bound(t, cache, tokens, want, weight, reach):
    """attention_bound takes exponents under 2^5 (64 U for the four roundings of one); here score, log2 of the scale and
    reference stay under 2^8, so that the four are off by 4 * 2^8 U at most, and a weight enters both sums."""
    vmax = float(cache.scales[:, 0, 1].max()) * 127
    return attention_bound(t, cache.dim, tokens, want, weight, reach, vmax) + weight * 2 * 4 * 256 * U


@pytest.mark.parametrize("t", [F32, BF16], ids=lambda t: TYPE_NAMES[t])
@pytest.mark.parametrize("dim,rows", [(64, 1), (64, 33), (64, 200), (128, 1), (128, 12), (192, 9), (256, 1), (256, 150)])
@pytest.mark.parametrize("top", [2.0 ** 9, 2.0 ** 11, 1.3e16 / 127, 2.0 ** 110])
def test_far_scales(hl, dev, t, dim, rows, top):
    """Blocks of zeros and of ordinary values before and behind blocks of a large scale, inside a step, steps apart and in
    parts of a sequence that different workgroups have; scores that are all equal (heads 0 and 1) and that spread."""
    import torch

    print("[case] attention far scales", TYPE_NAMES[t], dim, rows, top, flush=True)
    rng = np.random.default_rng(dim + rows)
    block, heads = 16, 4
    lens = np.array([32, 47, 64, 4000, 4000, 700])
    counts = np.minimum(rows, lens)
    cache, tables, _ = setup(hl, dev, rng, lens, 2, dim, block, clean=True)
    scales = cache.scales.copy()
    kinds = {  # per page of a sequence: z zeros, h the large scale, o ordinary values
        0: "zh", 1: "hzo", 2: "ohzo", 3: "z" * 125 + "h" + "z" * 124, 4: "h" + "z" * 100 + "o" * 149, 5: "o" * 20 + "z" * 20 + "oooh"}
    for s, kind in kinds.items():
        for page, what in zip(tables[s], kind):
            if what == "z":
                scales[page, 0, 1], cache.codes[page, 0, 1] = 0, 0
            elif what == "h":
                scales[page, 0, 1] = top
    cache.set_scales(scales)
    gpu = OnGpu(hl, dev, cache)
    q = rng.standard_normal((int(counts.sum()), heads, dim)) * 2
    q[:, :2] = 0
    starts = batch(counts)
    qd, qx = to_type(q, t, dev)
    want, weight, reach = attention_ref(cache, 0, tables, lens, starts, qx)
    tol = far_bound(t, cache, 4000, want, weight, reach)
    for hint in (dict(), dict(max_rows=rows, max_kv=4000)):
        out = torch.full_like(qd, 5.0)
        hl.attention(t, gpu.cache, 0, gpu.batch(tables, lens, starts, len(q), **hint), qd, out, heads)
        err = np.abs(out.double().cpu().numpy() - want)
        assert np.all(err <= tol), f"{(err / tol).max()} times the bound, {np.isnan(err).sum()} NaN"
