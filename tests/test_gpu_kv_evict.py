"""Accumulated attention weights and eviction by them, against fp64 loops.

Weights: with e = 2^-24, a score is off by at most (t D + 8) e M (M = max sum_d |q_d k_d| scale; t = 3 where fp32 queries meet codes
as three parts, 2 where fp32 products are summed four at a time), the exponent's argument by 4 e (M + |lse|), the exponential
and the sum of n terms by (n + 8) e: relative bounds, times the weight itself, since all terms are positive.
Eviction moves and selects: everything is compared exactly."""
import numpy as np
import pytest
import torch

from oracle import cache as orc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24


def _F():
    import dtorch_amd.nn.functional as F
    return F


def _weights_case(rng, B, Hq, Hkv, L, S, D, dtype, codes=0):
    q = torch.from_numpy(rng.standard_normal((B, Hq, L, D)).astype(np.float32)).to(dtype)
    w = rng.random((B, Hkv, S)).astype(np.float32) / 64
    if codes:
        c = rng.integers(0, 256, (B, Hkv, S, D)).astype(np.uint8)
        c = np.where((c & 0x78) > 0x40, (c & 0x87) | 0x40, c).astype(np.uint8)  # up to 3.75
        ks = (0.5 + rng.random((B, Hkv, S // codes))).astype(np.float32)
        return q, torch.from_numpy(c).view(torch.float8_e4m3fn), orc.values(c, ks), torch.from_numpy(ks), w
    k = torch.from_numpy(rng.standard_normal((B, Hkv, S, D)).astype(np.float32)).to(dtype)
    return q, k, k.double().numpy(), None, w


def _lse(q, k, n, causal, q_offset, scale):
    """fp32 LSE of every row over the keys it sees (-inf: none)."""
    B, Hq, L, D = q.shape
    g = Hq // k.shape[1]
    out = np.full((B, Hq, L), -np.inf)
    for b in range(B):
        for h in range(Hq):
            s = q[b, h] @ k[b, h // g].T * scale
            for i in range(L):
                top = min(n[b], max(i + q_offset + 1, 0)) if causal else n[b]
                if top > 0:
                    m = s[i, :top].max()
                    out[b, h, i] = m + np.log(np.exp(s[i, :top] - m).sum())
    return out.astype(np.float32)


def _check_weights(rng, B, Hq, Hkv, L, S, D, dtype, codes=0, lengths=None, causal=False, q_offset=0, scale=None, flat=False, layout=None):
    q, k, kv, ks, w = _weights_case(rng, B, Hq, Hkv, L, S, D, dtype, codes)
    sc = D ** -0.5 if scale is None else scale
    n = [S] * B if lengths is None else [min(max(x, 0), S) for x in lengths]
    qd = q.double().numpy()
    lse = _lse(qd, kv, n, causal, q_offset, sc)
    want, terms = w.astype(np.float64), np.zeros_like(w, dtype=np.float64)
    orc.attention_weights(want, qd, kv, lse.astype(np.float64), lengths, causal, q_offset, scale)
    g = Hq // Hkv
    mag = max(np.abs(qd[:, h]).sum(-1).max() * np.abs(kv[:, h // g]).max() for h in range(Hq)) * abs(sc) if D < 32 else \
        max((np.abs(qd[b, h]) @ np.abs(kv[b, h // g]).T).max() for b in range(B) for h in range(Hq)) * abs(sc)
    t = 3 if dtype == torch.float32 and codes else 2
    fin = np.abs(lse[np.isfinite(lse)]).max(initial=0)
    rel = (t * D + 8) * E * mag + 4 * E * (mag + fin) + (L * g + 8) * E
    dw = torch.from_numpy(w.copy()).cuda()
    dq, dk = q.cuda(), k.cuda()
    if layout is not None:
        dq, dk = layout(dq), layout(dk)
    dl = torch.from_numpy(lse).cuda()
    r = _F().attention_weight_accumulate(dw, dq, dk, dl[:, :, 0] if flat else dl, is_causal=causal, q_offset=q_offset, scale=scale,
                                         lengths=None if lengths is None else torch.tensor(lengths, dtype=torch.int32, device="cuda"),
                                         key_scale=None if ks is None else ks.cuda())
    torch.cuda.synchronize()
    assert r is dw or r.data_ptr() == dw.data_ptr()
    got = dw.double().cpu().numpy()
    for b in range(B):  # behind the sequence: untouched
        assert np.array_equal(got[b, :, n[b]:], w[b, :, n[b]:].astype(np.float64))
    # want - w is the sum added; its rounding and that of the addition
    tol = (want - w) * rel + want * 2 * E
    assert np.all(np.abs(got - want) <= tol), float(np.max(np.abs(got - want) / tol))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("codes", [0, 16, 64])
@pytest.mark.parametrize("Hq,Hkv,D", [(32, 8, 128), (7, 1, 64), (40, 2, 80), (3, 3, 16)])
def test_one_query(dtype, codes, Hq, Hkv, D):
    rng = np.random.default_rng(Hq + D + codes)
    _check_weights(rng, 6, Hq, Hkv, 1, 320, D, dtype, codes, lengths=[0, 1, 63, 64, 65, 500], flat=True)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("L,S,Hq,Hkv,D,causal,q_offset,lengths", [
    (1, 1, 2, 2, 64, True, 0, None), (50, 50, 4, 2, 128, True, 0, None), (50, 50, 6, 2, 64, True, 0, [50, 33, 0]), (130, 130, 3, 3, 48, True, 0, [1, 130, 64]),
    (33, 200, 8, 2, 128, True, 167, [200, 180, 190]), (40, 100, 4, 1, 64, False, 0, None), (40, 100, 4, 1, 64, False, 0, [7, 100, 64]),
    (30, 90, 5, 1, 128, True, -10, None), (20, 64, 2, 1, 64, True, 500, None), (257, 257, 4, 4, 128, True, 0, None), (100, 300, 2, 2, 20, True, 200, [300, 250, 1]),
    (90, 60, 12, 4, 8, False, 0, [60, 33, 0]), (600, 600, 14, 2, 64, True, 0, [600, 599, 257])])
def test_prompt(dtype, L, S, Hq, Hkv, D, causal, q_offset, lengths):
    if D == 20 and dtype != torch.float32:
        D = 24  # rows of 16-bit elements are a multiple of 8
    rng = np.random.default_rng(L * 100 + S)
    _check_weights(rng, 3, Hq, Hkv, L, S, D, dtype, lengths=lengths, causal=causal, q_offset=q_offset)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("L,S,Hq,Hkv,D,causal,q_offset,lengths", [
    (70, 20000, 2, 1, 64, True, 19930, [20000, 17000, 300]), (66, 9000, 2, 2, 64, False, 0, None), (65, 9000, 1, 1, 128, True, 8000, [9000, 8030, 0]),
    (30, 2900, 40, 1, 64, True, 2870, [2900, 2875, 100]), (1000, 1500, 2, 2, 16, True, 250, None)])
def test_prompt_over_many_keys(dtype, L, S, Hq, Hkv, D, causal, q_offset, lengths):
    """Shares of several key blocks, blocks of several shares, and more blocks than lanes."""
    _check_weights(np.random.default_rng(S), 3, Hq, Hkv, L, S, D, dtype, lengths=lengths, causal=causal, q_offset=q_offset)


def test_prompt_over_codes():
    rng = np.random.default_rng(2)
    for dtype in (torch.bfloat16, torch.float32):
        _check_weights(rng, 2, 4, 2, 60, 96, 64, dtype, 32, lengths=[96, 70], causal=True, q_offset=36)


@pytest.mark.parametrize("scale", [0.0, -0.2, 0.5])
def test_weights_scale(scale):
    _check_weights(np.random.default_rng(4), 2, 4, 2, 20, 40, 64, torch.float16, causal=True, q_offset=20, scale=scale)


def test_weights_layouts():
    rng = np.random.default_rng(5)
    _check_weights(rng, 2, 4, 2, 70, 70, 64, torch.bfloat16, causal=True, layout=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2))


def test_weights_padding_rows_of_any_value():
    """Queries past the prompt's end and rows that see no key (LSE -inf) may hold NaN; keys behind the sequence as well."""
    B, H, L, D = 2, 2, 64, 64
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(B, H, L, D, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    ln = torch.tensor([40, 17], dtype=torch.int32, device="cuda")
    o, lse = _F().scaled_dot_product_attention_with_lse(q, k, k, is_causal=True)
    w0, w1 = torch.zeros(B, H, L, device="cuda"), torch.full((B, H, L), 0.0, device="cuda")
    _F().attention_weight_accumulate(w0, q, k, lse, lengths=ln, is_causal=True)
    q2, k2, lse2 = q.clone(), k.clone(), lse.clone()
    for b, n in enumerate([40, 17]):
        q2[b, :, n:], k2[b, :, n:], lse2[b, :, n:] = float("nan"), float("nan"), float("nan")
    _F().attention_weight_accumulate(w1, q2, k2, lse2, lengths=ln, is_causal=True)
    lse3 = lse.clone()
    lse3[:, :, 5] = float("-inf")
    w2, w3 = w0.clone().zero_(), w0.clone().zero_()
    _F().attention_weight_accumulate(w2, q, k, lse3, lengths=ln, is_causal=True)
    _F().attention_weight_accumulate(w3, q[:, :, 5:6], k, lse[:, :, 5:6].contiguous(), lengths=ln, is_causal=True, q_offset=5)
    torch.cuda.synchronize()
    assert torch.equal(w0, w1)
    assert not torch.isnan(w0).any() and float(w0.sum()) == pytest.approx(H * (40 + 17), rel=1e-4)
    assert torch.allclose(w2 + w3, w0, rtol=1e-5, atol=1e-7)


# ---- eviction -------------------------------------------------------------------------------------------------

def _evict(rng, B, H, S, D, lengths, keep, recent, block, dtype, scale_block=0, weights=None, layout=None):
    def rows():
        if dtype == torch.float8_e4m3fn:
            return torch.from_numpy(rng.integers(0, 256, (B, H, S, D)).astype(np.uint8))
        it = {2: np.int16, 4: np.int32}[torch.empty(0, dtype=dtype).element_size()]
        return torch.from_numpy(rng.integers(-30000, 30000, (B, H, S, D)).astype(it))
    k, v = rows(), rows()
    w = np.exp(rng.standard_normal((B, H, S))).astype(np.float32) if weights is None else weights
    scales = [rng.random((B, H, S // scale_block)).astype(np.float32) for _ in range(2)] if scale_block else []
    lay = layout or (lambda x: x)
    dk, dv, dw = lay(k.cuda().view(dtype)), lay(v.cuda().view(dtype)), torch.from_numpy(w.copy()).cuda()
    ds = [torch.from_numpy(s.copy()).cuda() for s in scales]
    dl = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    hk, hv, hl = k.numpy().copy(), v.numpy().copy(), list(lengths)
    kept = orc.evict([hk, hv], scales, w, hl, keep, recent, block, scale_block or 1)
    got = _F().kv_cache_evict(dk, dv, dl, dw, keep, recent, block=block, **({"k_scale": ds[0], "v_scale": ds[1]} if ds else {}))
    torch.cuda.synchronize()
    back = {1: torch.uint8, 2: torch.int16, 4: torch.int32}[k.element_size()]
    assert np.array_equal(got.cpu().numpy(), kept)
    assert dl.tolist() == hl
    assert np.array_equal(dk.contiguous().view(back).cpu().numpy(), hk) and np.array_equal(dv.contiguous().view(back).cpu().numpy(), hv)
    assert np.array_equal(dw.cpu().numpy(), w, equal_nan=True)
    for a, b in zip(ds, scales):
        assert np.array_equal(a.cpu().numpy(), b)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("keep,recent,block", [(100, 10, 1), (1, 1, 1), (50, 50, 1), (299, 1, 1), (96, 32, 16), (128, 8, 8), (400, 3, 1)])
def test_evict(dtype, keep, recent, block):
    rng = np.random.default_rng(keep * 10 + block)
    _evict(rng, 7, 3, 304, 64, [0, 1, keep, keep + 1, 300, 304, 1000], keep, recent, block, dtype)


@pytest.mark.parametrize("keep,recent,block,scale_block", [(128, 32, 16, 16), (128, 64, 64, 16), (160, 32, 32, 32), (64, 64, 64, 32)])
def test_evict_codes(keep, recent, block, scale_block):
    rng = np.random.default_rng(block + scale_block)
    _evict(rng, 6, 2, 512, 48, [0, 5, 130, 257, 500, 512], keep, recent, block, torch.float8_e4m3fn, scale_block)


def test_evict_ties_and_odd_weights():
    rng = np.random.default_rng(6)
    S = 2000
    w = rng.integers(0, 3, (5, 2, S)).astype(np.float32)
    w[1] = 1.0
    w[2, :, ::3] = np.nan
    w[2, :, 1::3] = -np.inf
    w[3, 0] = np.where(rng.random(S) < 0.5, 0.0, -0.0)
    w[3, 1] = -w[3, 1]
    w[4, 0] = np.inf
    w[4, 1] = (rng.random(S) * 1e-42).astype(np.float32)  # subnormals keep their order
    for keep, recent in ((777, 10), (1999, 1500), (3, 1)):
        _evict(np.random.default_rng(7), 5, 2, S, 16, [S] * 5, keep, recent, 1, torch.bfloat16, weights=w.copy())


def test_evict_long():
    rng = np.random.default_rng(8)
    _evict(rng, 1, 2, 70000, 16, [69999], 30001, 100, 1, torch.bfloat16)
    _evict(rng, 1, 1, 70016, 16, [70001], 4000 * 16, 160, 16, torch.float8_e4m3fn, 16)


@pytest.mark.parametrize("n", [1023, 1024, 1025, 4096, 4097, 9001, 16384, 16385])
def test_evict_candidates_around_what_a_thread_holds(n):
    rng = np.random.default_rng(n)
    w = np.round(np.exp(rng.standard_normal((1, 2, n)) * 2)).astype(np.float32)  # many ties
    _evict(rng, 1, 2, n, 16, [n], n // 2 + 3, 5, 1, torch.bfloat16, weights=w)


def test_evict_many_and_few_heads():
    # 300 workgroups of whole rows, and two whose rows' chunks are shared out, one of them with an odd number of chunks
    rng = np.random.default_rng(11)
    _evict(rng, 25, 6, 96, 16, [96 - 3 * (i % 7) for i in range(25)], 40, 4, 1, torch.bfloat16)
    _evict(rng, 1, 1, 3001, 40, [3001], 1500, 7, 1, torch.bfloat16)
    _evict(rng, 1, 1, 9000, 128, [8999], 4096, 16, 16, torch.float32)


def test_evict_layouts():
    rng = np.random.default_rng(9)
    _evict(rng, 2, 3, 200, 64, [200, 151], 64, 4, 1, torch.float16, layout=lambda x: x.transpose(1, 2).contiguous().transpose(1, 2))


def test_evict_again_changes_nothing():
    rng = np.random.default_rng(10)
    k = torch.from_numpy(rng.integers(0, 9, (2, 2, 64, 16)).astype(np.int16)).cuda().view(torch.bfloat16)
    v, w = k.clone(), torch.rand(2, 2, 64, device="cuda")
    ln = torch.tensor([64, 20], dtype=torch.int32, device="cuda")
    _F().kv_cache_evict(k, v, ln, w, 32, 4)
    before = [x.clone() for x in (k.view(torch.int16), v.view(torch.int16), w, ln)]
    kept = _F().kv_cache_evict(k, v, ln, w, 32, 4)
    torch.cuda.synchronize()
    for a, b in zip(before, (k.view(torch.int16), v.view(torch.int16), w, ln)):
        assert torch.equal(a, b)
    assert kept[0, 0].tolist() == list(range(32)) and kept[1, 1].tolist() == list(range(20)) + [-1] * 12
