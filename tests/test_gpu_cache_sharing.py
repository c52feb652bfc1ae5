"""The cache classes over shared pages, a shared prefix and selected blocks: whole loops, as a program runs them, against caches that
share nothing.

Two caches hold the same keys and values, so their outputs differ by how the attention is cut alone: each is within the error of its
own sums and of one rounding of the same value, so the two lie within two half steps of the type, 2^-7 of the value for bf16, and twice
the sums' error, below 2^-12 of max |V| at these sizes (P in two 16-bit parts, or rounded to 16 bits: 2^-8 A for the plain decode)."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

B, HQ, HKV, D, PAGE = 6, 8, 2, 64, 16
BF = torch.bfloat16


def _paged(batch=B, pages=200, **kw):
    from dtorch_amd.nn.kv_cache import PagedKVCache
    return PagedKVCache(batch, HKV, pages, PAGE, 24, D, **kw)


def _qkv(batch, n, g, dtype=BF):
    return [torch.randn(batch, h, n, D, generator=g, device="cuda").to(dtype) for h in (HQ, HKV, HKV)]


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _near(a, b, top=4.0):
    # 2^-7 of the value (two roundings) and 2^-7 of A = softmax |V| <= max |V| (the plain decode's P in bf16, and its own half step)
    assert (a.double() - b.double()).abs().le(2.0 ** -7 * b.double().abs() + 2.0 ** -7 * top).all()


def _lone(cache, histories):
    """The plain decode of sequences whose tokens are listed, each in pages of its own."""
    lone = _paged(len(histories), pages=24 * len(histories))
    for b, tokens in enumerate(histories):
        k, v = (torch.cat([t[i] for t in tokens], 1)[None] for i in (0, 1))
        from dtorch_amd.nn import functional as F
        n = k.shape[2]
        pages = -(-n // PAGE)
        lone._table[b, :pages] = [lone._free.pop() for _ in range(pages)]
        lone._pages[b], lone._host_len[b] = pages, n
        lone.block_table.copy_(torch.from_numpy(lone._table))
        F.kv_cache_append_paged(lone.k, lone.v, lone.block_table[b:b + 1], lone.lengths[b:b + 1], k, v)
    return lone


def _consistent(cache):
    """The host's table, lengths and free list are the device's."""
    table = cache.block_table.cpu().numpy()
    assert np.array_equal(cache._table, table)
    assert np.array_equal(cache._host_len, cache.lengths.cpu().numpy())
    refs = np.bincount(table[table >= 0], minlength=cache.k.shape[0])
    assert np.array_equal(cache.page_refs.cpu().numpy(), refs)
    assert sorted(cache._free) == np.flatnonzero(refs == 0).tolist() and cache._free == sorted(cache._free, reverse=True)


@pytest.mark.parametrize("shared", [False, True])
@pytest.mark.parametrize("bounds", [0, 16])
def test_beam_loop(shared, bounds):
    """Two prompts, three beams each: fork, then steps with new parents; the tokens of every beam are kept on the side."""
    from dtorch_amd.nn import functional as F
    g, rng = _gen(1), np.random.default_rng(1)
    cache = _paged(bounds_block=bounds)
    q, k, v = _qkv(2, 53, g)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    if shared:
        cache.share(2)
        assert cache.prefix_lengths.tolist() == [48, 48]
    history = [[(k[i // 3], v[i // 3])] for i in range(B)]
    for step in range(40):
        if step % 3 == 2:
            parents = [0 + int(rng.integers(0, 3)) for _ in range(3)] + [3 + int(rng.integers(0, 3)) for _ in range(3)]
            cache.fork(parents)
            history = [list(history[p]) for p in parents]
        if step == 20:
            assert cache.compact().item() == (cache.page_refs > 0).sum().item() == cache.block_table.max().item() + 1
            if shared:
                assert cache.prefix_lengths.min().item() >= 48
        q1, k1, v1 = _qkv(B, 1, g)
        out = cache.decode(q1, k1, v1)
        for b in range(B):
            history[b].append((k1[b], v1[b]))
        _consistent(cache)
        if step % 8 == 0:
            lone = _lone(cache, history)
            _near(out, F.decode_attention_paged(q1, lone.k, lone.v, lone.block_table, lone.lengths)[0])
            if bounds:
                n = int(cache.lengths.max())
                kept = F.select_key_blocks_paged(q1, cache.k_min, cache.k_max, cache.block_table, cache.lengths, -(-n // 16) * 16, 16, 16)
                o = F.decode_attention_blocks_paged(q1, cache.k, cache.v, cache.block_table, cache.lengths, kept, 16)[0]
                _near(o, out)  # all blocks
                lo, hi = torch.zeros_like(cache.k_min), torch.zeros_like(cache.k_max)
                F.kv_key_bounds_paged(cache.k, lo, hi, cache.block_table, cache.lengths, n)
                for b in range(B):
                    ids = cache.block_table[b, :-(-int(cache.lengths[b]) // PAGE)].long()
                    assert torch.equal(lo[ids], cache.k_min[ids]) and torch.equal(hi[ids], cache.k_max[ids])


def test_free_and_refill():
    g = _gen(2)
    cache = _paged(pages=30)
    for _ in range(5):  # without freed pages the pool would run out
        q, k, v = _qkv(B, 60, g)
        cache.prefill(q, k, v)
        cache.free(range(B))
        _consistent(cache)
        assert len(cache._free) == 30
    q, k, v = _qkv(B, 60, g)
    cache.prefill(q, k, v)
    cache.free([1, 4])
    assert cache._host_len.tolist() == [60, 0, 60, 60, 0, 60]
    out = cache.decode(*_qkv(B, 1, g))
    _consistent(cache)
    assert torch.isfinite(out).all()
    with pytest.raises(ValueError, match="out of pages"):
        cache.append(*[x.expand(B, HKV, 100, D) for x in _qkv(B, 1, g)[1:]])
    _consistent(cache)


def test_codes_fork():
    """An 8-bit cache forks with its scales: every beam decodes as a cache that shares nothing."""
    from dtorch_amd.nn import functional as F
    g = _gen(3)
    cache = _paged(dtype=torch.float8_e4m3fn, block=16)
    q, k, v = _qkv(B, 40, g)
    cache.prefill(q, k, v)
    cache.fork([2, 2, 2, 0, 0, 5])
    twin = _paged(dtype=torch.float8_e4m3fn, block=16)
    source = torch.tensor([2, 2, 2, 0, 0, 5], device="cuda")
    twin.prefill(q[source], k[source], v[source])
    for _ in range(20):
        step = _qkv(B, 1, g)
        assert torch.equal(cache.decode(*step), twin.decode(*step))
    with pytest.raises(ValueError):
        cache.share(2)
    with pytest.raises(ValueError):
        cache.decode(*_qkv(B, 1, g), keep=16)


def test_captured_loop():
    """A beam step in a graph with its parents on the device; sync_lengths brings the host up to date."""
    g, rng = _gen(4), np.random.default_rng(4)
    held, eager = _paged(), _paged()
    q, k, v = _qkv(2, 37, g)
    for c in (held, eager):
        c.prefill(q, k, v)
        c.fork([0, 0, 0, 1, 1, 1])
        c.share(2)
    step = _qkv(B, 1, g)
    parents = torch.arange(B, dtype=torch.int32, device="cuda")
    for c in (held, eager):  # warm up on both
        c.decode(*step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.fork(parents)
        out = held.decode(*step)
    for i in range(30):
        new = np.concatenate([rng.integers(0, 3, 3), rng.integers(3, 6, 3)]).astype(np.int32)
        parents.copy_(torch.from_numpy(new))
        for x in step:
            x.normal_()
        eager.fork(new.tolist())
        want = eager.decode(*step)
        graph.replay()
        torch.cuda.synchronize()
        _near(out, want)
        assert torch.equal(held.block_table, eager.block_table) and torch.equal(held.lengths, eager.lengths)
    assert held.sync_lengths().tolist() == [68] * B
    _consistent(held)
    held.share(2)
    _near(held.decode(*step), eager.decode(*step))


def test_device_parents_and_shortage():
    g = _gen(5)
    cache = _paged(pages=12)
    cache.prefill(*_qkv(B, 20, g))
    cache.fork(torch.zeros(B, dtype=torch.int32, device="cuda"))
    with pytest.raises(RuntimeError, match="sync_lengths"):
        cache.share(2)
    cache.decode(*_qkv(B, 1, g))
    cache.sync_lengths()
    _consistent(cache)
    cache.fork(torch.arange(B, dtype=torch.int32, device="cuda"))
    for _ in range(40):  # more than twelve pages' tokens: nothing faults, and the next sync says so
        cache.decode(*_qkv(B, 1, g))
    with pytest.raises(RuntimeError, match="past the assigned pages"):
        cache.sync_lengths()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_padded_prefix(dtype):
    from dtorch_amd.nn import functional as F
    from dtorch_amd.nn.kv_cache import KVCache
    g = _gen(6)
    prefix, cache, plain = KVCache(2, HKV, 300, D, dtype=dtype), KVCache(B, HKV, 100, D, dtype=dtype), KVCache(B, HKV, 400, D, dtype=dtype)
    q, k, v = _qkv(2, 211, g, dtype)
    prefix.prefill(q, k, v)
    plain.append(k.repeat_interleave(3, 0), v.repeat_interleave(3, 0))
    for _ in range(30):
        step = _qkv(B, 1, g, dtype)
        _near(cache.decode(*step, prefix=prefix), plain.decode(*step))
    assert cache._host_len.tolist() == [30] * B
    with pytest.raises(ValueError):
        KVCache(B, HKV, 100, D, track_weights=True).decode(*_qkv(B, 1, g), prefix=prefix)


@pytest.mark.parametrize("paged", [False, True])
def test_sparse_loop(paged):
    """With room for every block the selection is the whole cache; with less, a needle far back is found."""
    from dtorch_amd.nn.kv_cache import KVCache
    g = _gen(7)
    mk = (lambda bb: _paged(pages=300, bounds_block=bb)) if paged else (lambda bb: KVCache(B, HKV, 333, D, bounds_block=bb))
    sparse, plain = mk(16), mk(0)
    q, k, v = _qkv(B, 300, g)
    k[:, :, 40] = 6.0  # a key that a query of ones finds
    v[:, :, 40] = 3.0
    for c in (sparse, plain):
        c.prefill(q, k, v)
    for i in range(20):
        q1, k1, v1 = _qkv(B, 1, g)
        if i % 2:
            q1.fill_(1.0)
        _near(sparse.decode(q1, k1, v1, keep=64 if i % 2 else 320, recent=16), plain.decode(q1, k1, v1))
    with pytest.raises(ValueError):
        plain.decode(q1, k1, v1, keep=64)


def test_evict_refreshes_bounds():
    from dtorch_amd.nn import functional as F
    from dtorch_amd.nn.kv_cache import KVCache
    g = _gen(8)
    cache = KVCache(B, HKV, 256, D, track_weights=True, bounds_block=32)
    cache.prefill(*_qkv(B, 200, g))
    cache.evict(100, 20)
    lo, hi = torch.zeros_like(cache.k_min), torch.zeros_like(cache.k_max)
    F.kv_key_bounds(cache.k, lo, hi, cache.lengths, 256)
    assert torch.equal(lo[:, :, :4], cache.k_min[:, :, :4]) and torch.equal(hi[:, :, :4], cache.k_max[:, :, :4])


def test_class_refusals():
    from dtorch_amd.nn.kv_cache import KVCache
    cache = _paged()
    for bad in ([0, 1], list(range(B + 1))):
        with pytest.raises(ValueError):
            cache.fork(bad)
    for groups in (4, -1, 7):
        with pytest.raises(ValueError):
            cache.share(groups)
    with pytest.raises(ValueError):
        cache.append(*_qkv(B + 1, 1, _gen(0))[1:])
    for kw in (dict(bounds_block=8), dict(bounds_block=32), dict(bounds_block=16, dtype=torch.float8_e4m3fn)):
        with pytest.raises(ValueError):
            _paged(**kw)
    with pytest.raises(ValueError):
        KVCache(B, HKV, 64, 256, bounds_block=16)


def _same_as_lone(cache, history, step):
    from dtorch_amd.nn import functional as F
    out = cache.decode(*step)
    for b in range(B):
        history[b].append((step[1][b].clone(), step[2][b].clone()))
    lone = _lone(cache, history)
    _near(out, F.decode_attention_paged(step[0], lone.k, lone.v, lone.block_table, lone.lengths)[0])


@pytest.mark.parametrize("device", [False, True])
def test_share_with_a_freed_sequence(device):
    """A freed sequence grows again, on pages of its own, past what its group shared."""
    g = _gen(9)
    cache = _paged()
    q, k, v = _qkv(2, 50, g)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    cache.share(2)
    held = cache.prefix_lengths
    history = [[(k[i // 3], v[i // 3])] for i in range(B)]
    parents = [0, -1, 2, 4, 4, 4]
    cache.fork(torch.tensor(parents, dtype=torch.int32, device="cuda") if device else parents)
    assert held.tolist() == [0, 48]
    history = [list(history[p]) if p >= 0 else [] for p in parents]
    for i in range(60):
        step = _qkv(B, 1, g)
        if i % 7 == 3 or i > 45:
            _same_as_lone(cache, history, step)
        else:
            cache.decode(*step)
            for b in range(B):
                history[b].append((step[1][b], step[2][b]))
    cache.sync_lengths()
    cache.share(2)
    assert cache.prefix_lengths is held and held.tolist() == [0, 48]


def test_share_across_groups():
    """Parents on the device from another group: the groups that take them share nothing, the others as before."""
    g = _gen(10)
    cache = _paged()
    q, k, v = _qkv(2, 50, g)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    cache.share(2)
    parents = [0, 5, 2, 3, 3, 4]
    cache.fork(torch.tensor(parents, dtype=torch.int32, device="cuda"))
    assert cache.prefix_lengths.tolist() == [0, 48]
    _same_as_lone(cache, [[(k[p // 3], v[p // 3])] for p in parents], _qkv(B, 1, g))


def test_captured_step_outlives_share():
    """A step captured under share(2) replays rightly after eager forks and another share."""
    g = _gen(11)
    cache = _paged()
    q, k, v = _qkv(2, 40, g)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    cache.share(2)
    history = [[(k[i // 3], v[i // 3])] for i in range(B)]
    step = _qkv(B, 1, g)
    _same_as_lone(cache, history, step)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = cache.decode(*step)
    from dtorch_amd.nn import functional as F
    for i in range(6):
        for x in step:
            x.normal_()
        graph.replay()
        for b in range(B):
            history[b].append((step[1][b].clone(), step[2][b].clone()))
        lone = _lone(cache, history)
        _near(out, F.decode_attention_paged(step[0], lone.k, lone.v, lone.block_table, lone.lengths)[0])
        cache.sync_lengths()
        parents = [3, 3, 3, 0, 0, 1] if i % 2 else [2, 1, 0, 5, 0, 4]
        cache.fork(parents)
        history = [list(history[p]) for p in parents]
        cache.share(3 if i % 2 else 1)


def test_refusals_leave_the_cache_alone():
    """What decode refuses it refuses before the append."""
    from dtorch_amd.nn.kv_cache import KVCache
    g = _gen(12)
    paged, padded = _paged(bounds_block=16), KVCache(B, HKV, 64, D, bounds_block=16)
    for c in (paged, padded):
        c.prefill(*_qkv(B, 20, g))
        for kw in (dict(keep=24), dict(keep=16, recent=32), dict(keep=32, recent=8), dict(keep=-16), dict(keep=32, recent=-16)):
            with pytest.raises(ValueError):
                c.decode(*_qkv(B, 1, g), **kw)
    for other in (KVCache(4, HKV, 64, D), KVCache(2, 2 * HKV, 64, D), KVCache(2, HKV, 64, 32), KVCache(2, HKV, 64, D, dtype=torch.float16),
                  KVCache(2, HKV, 64, D, device="cpu")):
        with pytest.raises(ValueError):
            padded.decode(*_qkv(B, 1, g), prefix=other)
    with pytest.raises(ValueError):
        paged.decode(*_qkv(2, 1, g))
    for bad in ([B], [-1], [0, 99]):
        with pytest.raises(ValueError):
            paged.free(bad)
    for c in (paged, padded):
        assert c._host_len.tolist() == c.lengths.tolist() == [20] * B


def test_capture_refusals():
    g = _gen(13)
    cache = _paged()
    cache.prefill(*_qkv(B, 20, g))
    parents = torch.arange(B, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, device="cuda")
    for attempt in (lambda: cache.fork(list(range(B))), lambda: cache.fork(parents), lambda: cache.compact(), lambda: cache.share(2)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            x.add_(1)
            with pytest.raises(RuntimeError):
                attempt()
    assert cache.page_refs is None and not cache._host_stale
