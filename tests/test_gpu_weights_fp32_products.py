"""Accumulated weights of fp32 prompts: a product of an fp32 query and key is taken in three bf16 parts each, of whose nine products
six are summed.

A part is its value's remainder rounded to nearest, so the second is at most 2^-8 of the value and the third 2^-16: the three products
left out are below 2^-23 of |q| |k|.  To see them a second head dim takes the largest product away (q = (x, 1), k = (y, -1) with x and y
in [1, 1 + 2^-6)), which is exact: the score x y - 1 is below 2^-5, and the five products that follow, all below 2^-5, leave no
more than 5 steps of 2^-28, below 2^-25.  A scale of 2^13 turns the score's error into one of the weight's logarithm; beside it the lse
times log2(e) is rounded (2^-24 of it), the fma (2^-24 of its result), the exponential and a sum of L terms ((L + 8) 2^-24); a term below 2^-126 may count as 0."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("D", [4, 64, 128])
@pytest.mark.parametrize("L,S,causal", [(90, 150, False), (140, 140, True)])
def test_products_left_out(D, L, S, causal):
    import dtorch_amd.nn.functional as F
    rng = np.random.default_rng(D + L)
    scale = 2.0 ** 13
    # remainders of one sign and as large as they get where parts are cut off, and any others
    near = lambda n: 1 + 2.0 ** -7 - 2.0 ** -23 * rng.integers(1, 40, n)
    any_ = lambda n: 1 + 2.0 ** -6 * rng.random(n)
    x, y = (np.where(rng.random(n) < 0.5, near(n), any_(n)).astype(np.float32) for n in (L, S))
    q, k = np.zeros((1, 1, L, D), np.float32), np.zeros((1, 1, S, D), np.float32)
    q[0, 0, :, 0], q[0, 0, :, 1], k[0, 0, :, 0], k[0, 0, :, 1] = x, 1, y, -1
    s = scale * (x.astype(np.float64)[:, None] * y.astype(np.float64) - 1)
    if causal:
        s = np.where(np.arange(S) <= np.arange(L)[:, None], s, -np.inf)
    m = s.max(1, keepdims=True)
    lse = (m + np.log(np.exp(s - m).sum(1, keepdims=True))).astype(np.float32)
    terms = np.exp(s - lse.astype(np.float64))
    # every term's relative error: the score's, the lse's and the argument's rounding; exp2's argument is log2(e) times the exponent
    arg = np.where(terms > 0, np.abs(s - lse), 0)
    rel = scale * (2.0 ** -23 * (1 + 2.0 ** -6) ** 2 + 2.0 ** -25) + 2.0 ** -24 * (np.abs(lse) + 2 * arg) + (L + 8) * 2.0 ** -24
    want, tol = terms.sum(0), (terms * np.expm1(rel)).sum(0)
    w = torch.zeros(1, 1, S, device="cuda")
    F.attention_weight_accumulate(w, torch.from_numpy(q).cuda(), torch.from_numpy(k).cuda(), torch.from_numpy(lse[None, None, :, 0]).cuda(),
                                  is_causal=causal, scale=scale)
    off = np.abs(w.double().cpu().numpy()[0, 0] - want)
    tol += L * 2.0 ** -126
    assert np.all(off <= tol), float((off / tol).max())


def test_values_at_the_ends_of_the_range():
    """The largest fp32 values, whose first part rounded to nearest would be infinite, and small ones."""
    import dtorch_amd.nn.functional as F
    L, D = 80, 64
    big = np.float32(np.finfo(np.float32).max)
    for a, b in ((big, 2.0 ** -126), (-big, 2.0 ** -125), (np.nextafter(big, np.float32(0)), -2.0 ** -126), (1.99 * 2.0 ** -100, 2.0 ** 99)):
        q, k = torch.zeros(1, 1, L, D), torch.zeros(1, 1, L, D)
        q[..., 3], k[..., 3] = float(a), float(b)
        s = float(np.float32(a)) * b
        w = torch.zeros(1, 1, L, device="cuda")
        lse = torch.full((1, 1, L), s + np.log(L), dtype=torch.float32)
        F.attention_weight_accumulate(w, q.cuda(), k.cuda(), lse.cuda(), scale=1.0)
        # parts, sums and the lse's rounding: 2^-20 of scores of at most 8 is ample; the sum is L equal terms
        want = L * np.exp(s - lse[0, 0, 0].double().item())
        assert (w.double() - want).abs().max().item() <= want * 2.0 ** -16, (a, b)
