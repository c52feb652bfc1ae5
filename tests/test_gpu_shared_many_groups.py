"""Shared prefixes of more groups than a wave has lanes, and the cache classes' shared and partial decodes in every type, against fp64 within
the bounds that test_gpu_decode_shared.py derives."""
import numpy as np
import pytest
import torch

from oracle import shared as orc
from test_gpu_decode_shared import TYPES, _close, _np, _shared

pytestmark = pytest.mark.gpu


def _mixed(rng, groups, per, page):
    """Prefixes of 0 to 99 tokens (whole pages of a paged cache) and own tokens of 0 to 40, empty sequences and whole empty groups among them."""
    unit = max(page, 1)
    prefixes = [int(rng.integers(0, 100)) // unit * unit if rng.random() < 0.7 else 0 for _ in range(groups)]
    owns = []
    for _ in range(groups):
        gone = rng.random() < 0.1
        owns += [(None if page else 0) if gone or rng.random() < 0.1 else int(rng.integers(0, 41)) for _ in range(per)]
    return prefixes, owns


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [0, 16, 32])
@pytest.mark.parametrize("groups,per,Hq,Hkv,D", [
    (64, 1, 2, 1, 64), (65, 1, 2, 2, 128), (65, 2, 4, 1, 64), (130, 3, 2, 1, 64), (1024, 1, 2, 2, 64), (1024, 2, 1, 1, 64),
    (70, 3, 16, 1, 64),    # 48 rows of a group
    (66, 5, 32, 1, 128),   # 160 rows
    (129, 2, 40, 1, 72),   # 80 rows, odd head dim
])
def test_many_groups(dtype, page, groups, per, Hq, Hkv, D):
    rng = np.random.default_rng(groups + per + page)
    prefixes, owns = _mixed(rng, groups, per, page)
    _shared(groups, groups * per, groups, Hq, Hkv, D, dtype, page, prefixes, owns)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [0, 16])
def test_only_late_groups(dtype, page):
    """Nothing to share, and no tokens at all, in the first 64 groups."""
    groups = 100
    prefixes = [0] * 64 + [32 * (g % 4) for g in range(36)]
    owns = [None if page else 0] * 64 + [g % 5 + (1 if page else 0) for g in range(36)]
    _shared(1, groups, groups, 4, 2, 64, dtype, page, prefixes, owns)


B, HQ, HKV, D, PAGE = 6, 8, 2, 64, 16


def _qkv(n, g, dtype, batch=B):
    return [torch.randn(batch, h, n, D, generator=g, device="cuda").to(dtype) for h in (HQ, HKV, HKV)]


def _against(out, q, ks, vs, dtype, scale=D ** -0.5):
    """out [B, Hq, 1, D] against each sequence's keys and values [Hkv, n, D], or for every kv head its own rows [n, D]."""
    go, nq = _np(out), _np(q)
    for b in range(B):
        for h in range(HKV):
            K, V = _np(ks[b][h]), _np(vs[b][h])
            heads = slice(h * HQ // HKV, (h + 1) * HQ // HKV)
            want = orc.attend(nq[b, heads, 0], K, V, scale)
            _close(go[b, heads, 0], want[1], want, len(K), D, dtype, float(np.abs(V).max()))


@pytest.mark.parametrize("dtype", TYPES)
def test_padded_prefix_in_every_type(dtype):
    from dtorch_amd.nn.kv_cache import KVCache
    g = torch.Generator(device="cuda").manual_seed(41)
    prefix, cache = KVCache(2, HKV, 300, D, dtype=dtype), KVCache(B, HKV, 100, D, dtype=dtype)
    q, k, v = _qkv(211, g, dtype, 2)
    prefix.prefill(q, k, v)
    ks, vs = ([x[b // 3] for b in range(B)] for x in (k, v))
    for i in range(20):
        step = _qkv(1, g, dtype)
        out = cache.decode(*step, prefix=prefix)
        ks, vs = ([torch.cat([x, y], 1) for x, y in zip(a, new)] for a, new in ((ks, step[1]), (vs, step[2])))
        if i % 5 == 0 or i == 19:
            _against(out, step[0], ks, vs, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shared", [False, True])
def test_beams_in_every_type(dtype, shared):
    from dtorch_amd.nn.kv_cache import PagedKVCache
    g, rng = torch.Generator(device="cuda").manual_seed(42), np.random.default_rng(42)
    cache = PagedKVCache(B, HKV, 100, PAGE, 12, D, dtype=dtype)
    q, k, v = _qkv(53, g, dtype, 2)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    if shared:
        cache.share(2)
    ks, vs = ([x[b // 3] for b in range(B)] for x in (k, v))
    for i in range(30):
        if i % 3 == 2:
            parents = rng.integers(0, 3, 3).tolist() + rng.integers(3, 6, 3).tolist()
            cache.fork(parents)
            ks, vs = ([x[p] for p in parents] for x in (ks, vs))
        step = _qkv(1, g, dtype)
        out = cache.decode(*step)
        ks, vs = ([torch.cat([x, y], 1) for x, y in zip(a, new)] for a, new in ((ks, step[1]), (vs, step[2])))
        if i % 6 == 2 or i == 29:
            if shared:  # the plain decode's own bounds are its own tests' matter
                _against(out, step[0], ks, vs, dtype)
            else:
                from dtorch_amd.nn import functional as F
                both = F.decode_attention_shared_paged(step[0], cache.k, cache.v, cache.block_table, cache.lengths, torch.zeros(2, dtype=torch.int32, device="cuda"))
                _against(both[0], step[0], ks, vs, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("paged", [False, True])
def test_partial_decode_in_every_type(dtype, paged):
    """Over the blocks that the selection names, read from what was appended."""
    from dtorch_amd.nn.kv_cache import KVCache, PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(43)
    cache = PagedKVCache(B, HKV, 150, PAGE, 24, D, dtype=dtype, bounds_block=16) if paged else KVCache(B, HKV, 333, D, dtype=dtype, bounds_block=16)
    q, k, v = _qkv(300, g, dtype)
    cache.prefill(q, k, v)
    for i in range(8):
        step = _qkv(1, g, dtype)
        out = cache.decode(*step, keep=96, recent=32)
        k, v = torch.cat([k, step[1]], 2), torch.cat([v, step[2]], 2)
        n = k.shape[2]
        pad = torch.nn.functional.pad
        lo, hi = (pad(k.float(), (0, 0, 0, -n % 16), value=fill).unflatten(2, (-1, 16)) for fill in (float("inf"), -float("inf")))
        ids = orc.select(_np(step[0])[:, :, 0], _np(lo.amin(3)), _np(hi.amax(3)), None, [n] * B, 96, 32, 16)
        rows = [[[t for j in ids[b, h] for t in range(16 * j, min(16 * j + 16, n))] for h in range(HKV)] for b in range(B)]
        ks, vs = ([[x[b, h, rows[b][h]] for h in range(HKV)] for b in range(B)] for x in (k, v))
        _against(out, step[0], ks, vs, dtype)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("batch,heads,kv,d,prefix", [(4, 32, 8, 128, 2000), (32, 8, 2, 64, 700), (40, 16, 2, 128, 900)])
def test_same_bits(dtype, batch, heads, kv, d, prefix):
    """The same call gives the same bits, whatever the workspace held before."""
    from dtorch_amd.nn import functional as F
    g = torch.Generator(device="cuda").manual_seed(44)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda").to(dtype)

    q, kp, vp, k, v = normal(batch, heads, 1, d), normal(1, kv, prefix, d), normal(1, kv, prefix, d), normal(batch, kv, 200, d), normal(batch, kv, 200, d)
    n, lengths = torch.tensor([prefix], dtype=torch.int32, device="cuda"), torch.randint(0, 201, (batch,), generator=g, device="cuda", dtype=torch.int32)
    ids = torch.randint(-1, 13, (batch, kv, 9), generator=g, device="cuda", dtype=torch.int32)
    calls = [lambda: F.decode_attention_shared(q, kp, vp, n, k, v, lengths), lambda: F.decode_attention_blocks(q, k, v, lengths, ids, 16)]
    first = [[x.clone() for x in call()] for call in calls]
    for i in range(12):
        spoil = [torch.full((size,), (float("nan"), 1e30, -3.0)[i % 3], device="cuda") for size in (1 << 10, 1 << 14, 1 << 18, 1 << 20, 1 << 22)]
        del spoil
        for call, want in zip(calls, first):
            assert all(torch.equal(a, b) for a, b in zip(call(), want))
