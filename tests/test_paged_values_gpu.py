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


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 64), (F16, 128), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("n", [16, 700, 30000])
@pytest.mark.parametrize("low", [-math.inf, -1000.0])
def test_tokens_without_weight_add_nothing(cuda_device, dtype, d, group, n, low):
    """One token of value zero among tokens whose weight is zero (a score of -inf, or e^-1000 of the largest, which no type here holds):
    zero exactly, however large their values and however many they are."""
    q, k, v, table, lengths = make([n], 1, group, d, 16, dtype)
    q[:] = 1.0
    k[:] = low / d
    v[:] = 60000.0
    page = table[0, n // 32].long()
    k[page, 0, 5] = 0.0
    v[page, 0, 5] = 0.0
    out, lse = blockPagedAttention(q, k, v, table, lengths, 1.0, return_lse=True)
    assert (out == 0).all() and (lse == 0).all()


@pytest.mark.parametrize("dtype,weight", [(F16, 2.0 ** -37), (BF16, 2.0 ** -100)])
def test_an_infinite_value_stays_one(cuda_device, dtype, weight):
    """Infinite values of tokens with small weights, also weights that the first of the two 16-bit numbers holds exactly."""
    for w in (weight, 2.0 ** -8, 0.7):
        q, k, v, table, lengths = make([700], 1, 2, 64, 16, dtype)
        q[:] = 0.0
        q[:, :, 0] = 1.0
        k[:] = 0.0
        v[:] = 1.0
        page = table[0, 20].long()
        k[page, 0, 5, 0] = math.log(w)
        v[page, 0, 5, 3], v[page, 0, 5, 4] = math.inf, -math.inf
        out = blockPagedAttention(q, k, v, table, lengths, 1.0)
        assert (out[..., 3] == math.inf).all() and (out[..., 4] == -math.inf).all()
        assert torch.isfinite(out[..., 5:]).all()


@pytest.mark.parametrize("group", [1, 12])
@pytest.mark.parametrize("every", [False, True])
def test_weights_too_small_for_halves_are_rounded(cuda_device, group, every):
    """fp16: a weight is off by at most 2^-39 of the largest, in both directions: tokens of 2^-40.4 do not count as more than they may,
    be it behind one large score or with one in every tile, which all of them are relative to."""
    n = 30000
    q, k, v, table, lengths = make([n], 1, group, 64, 16, F16)
    q[:] = 1.0
    k[:] = -28.0 / 64
    v[:] = 60000.0
    large = table[0].long() if every else table[0, 900:901].long()
    k[large, 0, 5] = 0.0
    v[large, 0, 5] = 0.0
    out = blockPagedAttention(q, k, v, table, lengths, 1.0).double()
    small = (n - len(large)) / len(large)
    want = small * math.exp(-28.0) * 60000.0
    assert ((out - want).abs() <= (small + 1) * 2.0 ** -39 * 60000.0 + 2.0 ** -11 * want + 2.0 ** -25).all()


@pytest.mark.parametrize("dtype,d", [(F16, 64), (BF16, 128), (F32, 64), (F32, 128)])
@pytest.mark.parametrize("group", [1, 4, 12])
@pytest.mark.parametrize("n", [3, 40, 700, 30000])
def test_logarithm_of_a_score_of_infinity(cuda_device, dtype, d, group, n):
    """ln sum exp with a score of +inf is +inf (the softmax is inf / inf: NaN), wherever the others stand, above or below zero; a NaN
    among them stays one."""
    q, k, v, table, lengths = make([n] * 4, 1, group, d, 16, dtype)
    q[:] = 8.0
    k[table[:, : -(-n // 16)].long()] = 3.0
    k[table[1].long()] = -3.0
    last = (table[:, (n - 1) // 16].long(), 0, (n - 1) % 16)
    k[last[0][:2], 0, last[2]] = math.inf
    k[table[2, 0].long(), 0, 0] = math.inf
    k[last[0][2], 0, last[2]] = -math.inf
    k[table[3, 0].long(), 0, 1] = math.inf
    k[table[3, 0].long(), 0, 2] = math.nan
    out, lse = blockPagedAttention(q, k, v, table, lengths, 1.0, return_lse=True)
    assert (lse[:3] == math.inf).all() and torch.isnan(lse[3]).all() and torch.isnan(out).all()
