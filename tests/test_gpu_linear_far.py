"""Linear attention over rows whose elements pass 32 bits."""
import pytest

from kv_helpers import BF16

pytestmark = pytest.mark.gpu


def test_rows_past_32_bits_of_elements_in_a_bad_slot(hl, dev):
    """Every row of a sequence whose slot is out of range is NaN, also where its rows' elements pass 2^32."""
    import torch

    n, dim = (1 << 27) + 3, 64
    x = torch.zeros(n, 1, dim, dtype=torch.bfloat16, device=dev)
    out = torch.zeros_like(x)
    s, ints = torch.zeros(1, 1, dim, dim, device=dev), lambda v: torch.tensor(v, dtype=torch.int32, device=dev)
    batch = hl.LinearBatch(ints([1]), ints([0, n]), 1, n, 1)
    status = torch.zeros(1, dtype=torch.int32, device=dev)
    hl.linear_attention(BF16, hl.LinearState(s, 1, 1, dim, dim), batch, x, x, x, out, torch.zeros(1, device=dev), 1, decay_per_head=True, status=status)
    assert int(status) == hl.STATUS_BAD_INDEX
    for at in range(0, n, 1 << 24):
        assert bool(torch.isnan(out[at:at + (1 << 24)]).all()), at
