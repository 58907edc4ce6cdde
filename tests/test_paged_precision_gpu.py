"""GPU: how near single-token attention over a paged cache is to 64 bits, request by request in the 2-norm.

16-bit results are to be as good as the exact ones rounded once.  With r the rounding's relative error in the 2-norm and e the error before it,
independent of it, the result is off by sqrt(r^2 + e^2).  r is a uniform error of up to half a step, between eps / 2 sqrt(3) and half of that:
at least 2^-10.8 of the values for bf16, 2^-13.8 for fp16.  e: the weights' pair of 16-bit numbers (2^-17 for bf16, 2^-22 for fp16), scores,
exponentials and sums in 32 bits as below (10^-6 = 2^-20): together below 2^-16.8 and 2^-19.8, a sixty-fourth of r, which is 1.0002.
Allowed is 1.02 (e = r / 5); weights rounded once to the type have e of about r, 1.4.

32 bits: a score is a sum of d products, each off by 2^-24 of itself and added with errors of 2^-24 of sums no larger than sqrt(d) products
(here of one each, times scale d^-0.5): about 2^-24 log2(d) <= 2^-21 as a weight's relative error; its exponent, up to 2^3 here, 2^-24 of
itself: 2^-21; the exponential 2^-22.  Sums over the tokens: chains of up to 300 terms here (tokens of a warp, or parts), which random errors
leave off by sqrt(300 / 6) 2^-24 = 4.2e-7 for values of both signs and sqrt(300) / 3 2^-24 = 3.4e-7 for weights.  Squares added: 0.9e-6;
2e-6 is allowed.  A tensor core's 10 or 11 bits for q, k or v give 1.5e-4 or more, weights rounded to bf16 8e-4.

Logarithms (up to 12): half a step of 2^-20 for the sum, a step for the logarithm's function, 2^-23 for the maximum's product, 3.4e-7 and 2^-22
for the sum's relative error, and a score's of 5e-7: 2.6e-6, 4e-6 is allowed."""
import pytest
import torch

from blockedattention_b200 import blockPagedAttention
from test_paged_gpu import BF16, F16, F32, exact, make

pytestmark = pytest.mark.gpu
LENGTHS = [17, 64, 100, 333, 1000, 2500, 20000]


def ratios(out, want):
    """Of every request: the error of 16-bit results against that of the exact ones rounded; for 32 bits relative to the values."""
    error = (out.double() - want).flatten(1).norm(dim=1)
    return error / ((want.to(out.dtype).double() - want) if out.dtype != F32 else want).flatten(1).norm(dim=1)


@pytest.mark.parametrize("dtype,d", [(t, d) for t in (F16, BF16) for d in (8, 64, 72, 96, 128, 192, 256)] + [(F32, d) for d in (4, 64, 80, 128, 200, 256)])
@pytest.mark.parametrize("kv,group,page,layout", [(8, 1, 16, "heads"), (3, 6, 24, "tokens"), (1, 32, 1, "heads")])
def test_error_in_the_norm(cuda_device, dtype, d, kv, group, page, layout):
    q, k, v, table, n = make(LENGTHS, kv, group, d, page, dtype, d + kv, layout)
    out, lse = blockPagedAttention(q, k, v, table, n, d ** -0.5, return_lse=True)
    want, log, _, _ = exact(q, k, v, table, n, d ** -0.5)
    assert ratios(out, want).max().item() <= (2e-6 if dtype == F32 else 1.02)
    assert (lse.double() - log).abs().max().item() <= 4e-6
