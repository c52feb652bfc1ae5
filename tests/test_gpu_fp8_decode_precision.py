"""Decode over codes with 16-bit queries: fp32 all the way to the output, which is rounded once.

With u the half step of the output type (2^-8 bf16, 2^-11 fp16), e = 2^-24, A = softmax |V| and n keys: scores are off by
ds = (D + 8) e M, M = max sum |q_d k_d| scale, so P relatively by 2 ds + 64 e (its exponential and the merge); P enters its product as
two parts of the type, which leave u^2 of it; sums over the 2 n products add 2 n e; all that is relative to A, and O's own rounding
is u |O|.  In fp16 a part that is subnormal is off by 2^-25 whatever its value; the kernel puts the largest P of 32 tokens at 2^15, so
that is 2^-40 of it per token, at most n 2^-40 max |V|; a subnormal O is off by 2^-25."""
import numpy as np
import pytest
import torch

from oracle import cache as orc
from tests.test_gpu_fp8_cache import E, U, _decode_case, _run_decode

pytestmark = pytest.mark.gpu


def _check(c):
    dtype, D = c["q"].dtype, c["q"].shape[-1]
    o, _ = _run_decode(c)
    want, _, a, mag = orc.decode_fp8(c["q"].double().numpy()[:, :, 0], c["k"], c["v"], c["ks"], c["vs"], c["lengths"], c["table"])
    n = np.maximum(np.asarray(c["lengths"], dtype=np.float64), 1)[:, None]
    u = U[dtype]
    tol = a * (2 * (D + 8) * E * mag + (2 * n + 64) * E + u * u)[..., None]
    if dtype == torch.float16:
        tol = tol + (n * 2.0 ** -40)[..., None] * np.nanmax(np.abs(orc.values(c["v"], c["vs"]))) + 2.0 ** -25
    tol = tol * (1 + u) + np.abs(want) * u + np.finfo(np.float32).tiny
    off = np.abs(o.double().cpu().numpy()[:, :, 0] - want)
    assert (off <= tol).all(), float((off / tol).max())


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("lengths,Hq,Hkv,D,block,page", [
    ([4000], 32, 8, 128, 32, 0), ([1, 33, 700, 5, 0, 699], 8, 2, 64, 16, 16), ([3, 64, 17], 40, 2, 80, 64, 64), ([2500, 31, 900], 20, 20, 128, 128, 0),
    ([70] * 65, 12, 12, 64, 32, 32)])
def test_output_is_rounded_once(dtype, lengths, Hq, Hkv, D, block, page):
    rng = np.random.default_rng(Hq + D)
    cap = -(-max(lengths) // max(block, page)) * max(block, page)
    _check(_decode_case(rng, lengths, Hq, Hkv, D, block, page, dtype, cap))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_output_is_rounded_once_with_scales_apart(dtype):
    # V blocks up to 2^10 apart, and peaked rows
    rng = np.random.default_rng(21)
    c = _decode_case(rng, [500, 260, 18], 8, 4, 128, 16, 0, dtype, 512, scales=lambda r, s: np.exp2(r.integers(-9, 2, s)).astype(np.float32), junk=False)
    c["q"] = c["q"] * 2
    _check(c)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_same_call_same_bits(dtype):
    rng = np.random.default_rng(22)
    c = _decode_case(rng, [3000, 1, 64, 0, 1777], 32, 8, 128, 16, 16, dtype, 3008)
    first = _run_decode(c)
    for _ in range(5):
        again = _run_decode(c)
        assert torch.equal(first[0].view(torch.uint8), again[0].view(torch.uint8)) and torch.equal(first[1], again[1])


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("exponents", [(-126,), (-128,), (-130, -127), (-149,), (-140, -100), (118, 119)])
@pytest.mark.parametrize("lengths,Hq,Hkv,page", [([100, 17, 1], 8, 2, 0), ([3000], 4, 4, 16)])
def test_value_scales_at_the_ends_of_the_range(dtype, exponents, lengths, Hq, Hkv, page):
    """Any positive finite scale: subnormal ones and the largest, in one share and in records that merge.

    Outputs near the smallest normal: half a step of the type's subnormals more, 2^-134 in bf16 and 2^-150 in fp32, and one of fp32
    for each product that brings the accumulators there (three) and each record that is added (a share has 128 tokens at least)."""
    rng = np.random.default_rng(23 + len(lengths))
    D, cap = 64, -(-max(lengths) // 16) * 16
    c = _decode_case(rng, lengths, Hq, Hkv, D, 16, page, dtype, cap, scales=lambda r, s: np.exp2(r.choice(exponents, s).astype(np.float64)).astype(np.float32), junk=False)
    for name in "kv":  # every finite code, up to 448
        bits = rng.integers(0, 256, c[name].shape).astype(np.uint8)
        c[name] = np.where((bits & 0x7F) == 0x7F, np.uint8(0x18), bits)
    c["ks"][:] = 2.0 ** -8
    if max(exponents) > 0:  # outputs within the range
        c["v"] = np.where((c["v"] & 0x78) > 0x50, (c["v"] & 0x87) | 0x50, c["v"]).astype(np.uint8)
    o, _ = _run_decode(c)
    want, _, a, mag = orc.decode_fp8(c["q"].double().numpy()[:, :, 0], c["k"], c["v"], c["ks"], c["vs"], c["lengths"], c["table"])
    n = np.maximum(np.asarray(lengths, dtype=np.float64), 1)[:, None]
    u, parts = (U[dtype], 2) if dtype == torch.bfloat16 else (0.0, 3)
    tol = a * (2 * (parts * D + 8) * E * mag + (3 * n + 64) * E + u * u)[..., None]
    tol = tol * (1 + u) + np.abs(want) * max(u, E) + (2.0 ** -134 if dtype == torch.bfloat16 else 2.0 ** -150) + ((4 + n / 128) * 2.0 ** -150)[..., None]
    off = np.abs(o.double().cpu().numpy()[:, :, 0] - want)
    assert np.all(off <= tol), float((off / tol).max())
