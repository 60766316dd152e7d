"""GPU: the likelihoods' sums over long rows of equal terms, where every addition
rounds the same way, against the closed form in 64 bits.

A row has logits 0 at every eighth place of its first 65,536 (so that every
thread has the maximum from its first chunk on) and -c everywhere else:
S = h + r e^-c, log p = x - log S, entropy = log S + c r e^-c / S.
Tolerance, of S relative (u = 2^-24): a term's exponent is rounded at a magnitude
of 16 at most, 2^-21 ln 2, and its exponential is good to 2^-22; a chunk's sum is
16 additions, chunks are added with their rounding errors carried along (2 u), and
eleven joins of equal maxima are an addition each: 2^-21 ln 2 + 2^-22 + 30 u =
2^-18.8, below the 2^-18 that test_gpu_logprobs allows a term, whatever the
row's length is.  The entropy has that of S and, times 2 sum p |x|, of its numerator."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
HIGH = 1 << 16


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("V,M", [(151936, 297), (151936, 2), (1 << 20, 297), (1 << 20, 1), (1 << 24, 1), (1 << 24, 297),
                                 ((1 << 28) + 13, 2)])
def test_equal_terms(V, M, dtype):
    """297 rows and more have a CTA each, fewer a cluster."""
    from r4q import ops
    if M * V * dtype.itemsize > 12 << 30:
        M = 40                                        # a cluster of 8 for each
    x = torch.empty(M, V, dtype=dtype, device="cuda")
    tokens = torch.full((M,), V - 1, device="cuda")
    tokens[0] = 0
    for c in (1.2, 2.88, 5.65):
        x.fill_(-c)
        x[:, :HIGH:8] = 0
        c = -x[0, 1].double().item()
        h, r = HIGH // 8, V - HIGH // 8
        S = h + r * math.exp(-c)
        spread = c * r * math.exp(-c) / S
        lp = torch.full((M,), -c - math.log(S), dtype=torch.float64, device="cuda")
        lp[0] = -math.log(S)
        got = ops.token_logprobs(x, tokens, 1)
        tol = 2.0 ** -18 + 2 * U * (c + math.log(S))
        over = lambda a, b: (a.double() - b).abs().max().item() / tol
        assert over(got.logprob, lp) <= 1
        assert over(got.top_logprobs, -math.log(S)) <= 1 and not got.top_ids.any().item()
        H = math.log(S) + spread
        tol = 2.0 ** -18 * (1 + 2 * spread) + 4 * U * H
        assert over(got.entropy, H) <= 1
        assert got.rank.tolist() == [1] + [V] * (M - 1)          # the last of all that are equal
    ops.check_status()
