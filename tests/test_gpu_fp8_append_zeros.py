"""Quantised append of tokens that need no scale (all zeros, or no finite value): the scale of their block stays what its other
tokens need.

A code is half a step off: 2^-4 of the value, or 2^-10 of the scale where it is subnormal.  Scales are powers of two, so re-encoding at
a larger one rounds subnormal codes alone; the values here are within 2^9 of their block's largest, so none is."""
import numpy as np
import pytest
import torch

from oracle import cache as orc
from tests.test_gpu_fp8_cache import _F, _codes

pytestmark = pytest.mark.gpu


def _append(x, sizes, cap, block, page=0):
    """x [B, H, n, D] in calls of the given sizes -> (codes, scales) as a padded cache holds them."""
    B, H, _, D = x.shape
    slots, rows = (B * cap // page, page) if page else (B, cap)
    k = torch.zeros(slots, H, rows, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
    v, ks = torch.zeros_like(k), torch.ones(slots, H, rows // block, device="cuda")
    vs, ln, at = torch.ones_like(ks), torch.zeros(B, dtype=torch.int32, device="cuda"), 0
    table = torch.arange(slots, dtype=torch.int32, device="cuda").view(B, -1) if page else None
    for n in sizes:
        new = x[:, :, at:at + n]
        if page:
            _F().kv_cache_append_fp8_paged(k, v, ks, vs, table, ln, new, -new)
        else:
            _F().kv_cache_append_fp8(k, v, ks, vs, ln, new, -new)
        at += n
    torch.cuda.synchronize()
    out = []
    for c, s in ((k, ks), (v, vs)):
        c, s = _codes(c), s.cpu().numpy()
        if page:
            c = c.reshape(B, cap // page, H, page, D).transpose(0, 2, 1, 3, 4).reshape(B, H, cap, D)
            s = s.reshape(B, cap // page, H, page // block).transpose(0, 2, 1, 3).reshape(B, H, cap // block)
        out.append((c, s))
    assert ln.tolist() == [at] * B
    return out


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("what", ["zero", "-zero", "nan", "inf", "-inf"])
@pytest.mark.parametrize("where", ["before", "inside", "after", "alone"])
@pytest.mark.parametrize("page", [0, 32])
def test_tokens_that_need_no_scale(dtype, what, where, page):
    rng = np.random.default_rng(31)
    B, H, n, D, block, cap = 2, 3, 40, 64, 32, 64
    x = (rng.choice([-1.0, 1.0], (B, H, n, D)) * np.exp2(rng.uniform(-14, -8, (B, H, n, D)))).astype(np.float32)
    rows = {"before": [0, 1, 32], "inside": [7, 13, 35], "after": [31, 38, 39], "alone": list(range(32))}[where]
    x[:, :, rows] = {"zero": 0.0, "-zero": -0.0, "nan": np.nan, "inf": np.inf, "-inf": -np.inf}[what]
    x = torch.from_numpy(x).to(dtype).cuda()
    want = x.double().cpu().numpy()
    fin = np.isfinite(want)
    # the scale that the finite values of each block need
    top = np.abs(np.where(fin, want, 0)).reshape(B, H, n // 8, 8, D).max((3, 4))  # by eight rows
    need = np.stack([top[..., :4].max(-1), top[..., 4:].max(-1)], -1)
    need = np.vectorize(lambda m: orc.block_scale(m) if m > 0 else 2.0 ** -126)(need)
    first = None
    for sizes in ([n], [1] * n, [9, 1, 30], [1, 31, 8], [32, 1, 7]):
        got = _append(x, sizes, cap, block, page)
        for (codes, scale), sign in zip(got, (1, -1)):
            assert np.array_equal(scale, need), (sizes, scale, need)
            have = sign * orc.values(codes, scale)[:, :, :n]
            assert np.array_equal(np.isnan(have), ~fin), sizes
            step = np.repeat(need, block, 2)[:, :, :n, None]
            assert (np.abs(have - want)[fin] <= np.maximum(np.abs(want) * 2.0 ** -4, step * 2.0 ** -10)[fin]).all(), sizes
        if first is None:
            first = got
        assert all(np.array_equal(a, b) for p, q in zip(got, first) for a, b in zip(p, q)), sizes


def test_zero_blocks_weigh_nothing_in_decode():
    """A value block of zeros takes part in the row sum and adds nothing; an all-zero cache gives zeros."""
    B, H, D, block, n = 2, 2, 64, 16, 48
    g = torch.Generator(device="cuda").manual_seed(4)
    for dtype in (torch.bfloat16, torch.float16, torch.float32):
        r = lambda *s: torch.randn(*s, device="cuda", generator=g).to(dtype)
        for zero in (slice(16, 32), slice(0, 48)):
            k, v, q = r(B, H, n, D), r(B, H, n, D), r(B, 2 * H, 1, D)
            k[:, :, zero], v[:, :, zero] = 0, 0
            kc = torch.zeros(B, H, 64, D, dtype=torch.uint8, device="cuda").view(torch.float8_e4m3fn)
            vc, ks = torch.zeros_like(kc), torch.ones(B, H, 4, device="cuda")
            vs, ln = torch.ones_like(ks), torch.zeros(B, dtype=torch.int32, device="cuda")
            _F().kv_cache_append_fp8(kc, vc, ks, vs, ln, k, v)
            o, lse = _F().decode_attention_fp8(q, kc, vc, ks, vs, ln)
            torch.cuda.synchronize()
            kd, vd = (orc.values(_codes(c), s.cpu().numpy())[:, :, :n] for c, s in ((kc, ks), (vc, vs)))
            assert (kd[:, :, zero] == 0).all() and (vd[:, :, zero] == 0).all()
            if zero.start == 0:
                # scores of 0, sums of equal terms
                assert (o == 0).all() and (lse - np.log(n)).abs().max().item() <= 2.0 ** -19
                continue
            for b in range(B):
                for h in range(2 * H):
                    want, wl, a = orc.attend(q[b, h].double().cpu().numpy(), kd[b, h // 2], vd[b, h // 2], D ** -0.5)
                    mag = (np.abs(q[b, h].double().cpu().numpy()) @ np.abs(kd[b, h // 2]).T).max() * D ** -0.5
                    u = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: 2.0 ** -24}[dtype]
                    # P and O in the type, fp32 sums of up to 3 D and 3 n terms
                    tol = a * (u + (2 * (3 * D + 8) * mag + 3 * n + 64) * 2.0 ** -24) + u * np.abs(want) + 2.0 ** -24
                    assert (np.abs(o[b, h].double().cpu().numpy() - want) <= tol).all()
