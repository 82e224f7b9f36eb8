"""F16 attention over few rows: the softmax weights are carried in two pieces, so that what is off is the output's rounding."""
import numpy as np
import pytest

from kv_helpers import F16, F32, HALF_LEAST, HALF_STEP, attention_bound, attention_ref, batch, to_type
from test_gpu_attention import setup
from test_gpu_kv_cache import OnGpu

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,kv,group,rows,window,seqs", [(64, 2, 4, 1, 0, 60), (96, 1, 7, 1, 2, 60), (128, 2, 4, 1, 0, 60), (192, 1, 5, 2, 0, 60), (256, 4, 6, 1, 0, 60),
                                                           (256, 4, 6, 4, 3, 8), (128, 1, 8, 4, 0, 60)])
def test_as_exact_as_the_type(hl, dev, dim, kv, group, rows, window, seqs):
    """Within fp32's bound, whose weights are two pieces, and one rounding to F16; one piece would add up to half that rounding. Few
    tokens, values of V of one sign and small scores, so that neither averages nor the scores' own errors hide it.
    24 rows a kv head at head_dim 256 are few for up to 32 pairs of sequence and kv head."""
    import torch

    print("[case] attention f16", dim, kv, group, rows, window, flush=True)
    rng = np.random.default_rng(dim + rows)
    lens = np.resize(np.array([2, 3, 5, 9, 17]), seqs) + rows - 1
    cache, tables, _ = setup(hl, dev, rng, lens, kv, dim, 16)
    for page in range(cache.n_pages):
        v = cache.v_codes(page, 0)
        v[:] = np.abs(v.astype(np.int32)).clip(90, 127)
    gpu = OnGpu(hl, dev, cache)
    starts = batch(np.full(len(lens), rows))
    q, qx = to_type(rng.standard_normal((len(lens) * rows, kv * group, dim)) * 0.1, F16, dev)
    out = torch.full_like(q, 5.0)
    hl.attention(F16, gpu.cache, 0, gpu.batch(tables, lens, starts, max_rows=rows), q, out, kv * group, window=window)
    want, weight, reach = attention_ref(cache, 0, tables, lens, starts, qx, window)
    vmax = float(np.nan_to_num(cache.scales[:, 0, 1]).max()) * 127
    tol = attention_bound(F32, dim, int(lens.max()), want, weight, reach, vmax) + HALF_STEP[F16] * np.abs(want) * 1.01 + HALF_LEAST[F16]
    err = np.abs(out.double().cpu().numpy() - want)
    assert np.all(err <= tol), f"{(err / tol).max()} times the bound, {(err > tol).mean()} of the values"
