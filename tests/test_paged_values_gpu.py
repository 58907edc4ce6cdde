"""GPU: the paged cache's attention where scores, weights or values are not ordinary numbers."""
import math

import pytest
import torch

from blockedattention_b200 import blockPagedAttention
from test_paged_gpu import BF16, F16, F32, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 4, 12])
@pytest.mark.parametrize("n", [3, 40, 700, 30000])
def test_logarithm_of_scores_of_minus_infinity(cuda_device, dtype, d, group, n):
    """ln sum exp of scores that are all -inf is -inf (the softmax is 0 / 0); a single other score is the logarithm then."""
    q, k, v, table, lengths = make([n] * 3 + [0], 1, group, d, 16, dtype)
    q[:] = 0.5
    k[table[:2, : -(-n // 16)].long()] = -math.inf
    k[table[1, (n - 1) // 16].long(), 0, (n - 1) % 16] = 0.0
    out, lse = blockPagedAttention(q, k, v, table, lengths, 0.125, return_lse=True)
    assert (lse[0] == -math.inf).all() and torch.isnan(out[0]).all()
    assert (lse[1] == 0).all() and torch.equal(out[1], v[table[1, (n - 1) // 16].long(), 0, (n - 1) % 16].expand(group, -1))
    assert torch.isfinite(lse[2]).all() and (lse[3] == -math.inf).all() and (out[3] == 0).all()
    k[table[0, 0].long(), 0, 1] = math.nan
    _, lse = blockPagedAttention(q, k, v, table, lengths, 0.125, return_lse=True)
    assert torch.isnan(lse[0]).all()
