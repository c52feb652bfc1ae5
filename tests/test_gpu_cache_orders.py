"""Captured steps of a paged cache, replayed after what other calls made of the cache meanwhile, against caches that share nothing."""
import numpy as np
import pytest
import torch

from test_gpu_cache_sharing import B, _consistent, _gen, _lone, _near, _paged, _qkv

pytestmark = pytest.mark.gpu


def _beams(g, n=50, **kw):
    cache = _paged(**kw)
    q, k, v = _qkv(2, n, g)
    cache.prefill(q, k, v)
    cache.fork([0, 0, 0, 1, 1, 1])
    return cache, [[(k[i // 3], v[i // 3])] for i in range(B)]


def _captured(cache, step, parents=None):
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        if parents is not None:
            cache.fork(parents)
        out = cache.decode(*step)
    return graph, out


def _check(out, q, history):
    from dtorch_amd.nn import functional as F
    lone = _lone(None, history)
    _near(out, F.decode_attention_paged(q, lone.k, lone.v, lone.block_table, lone.lengths)[0])


def _follow(history, parents, step):
    history = [list(history[p]) for p in parents]
    for b in range(B):
        history[b].append((step[1][b].clone(), step[2][b].clone()))
    return history


def _replay(graph, step, parents, new, history):
    parents.copy_(torch.tensor(new, dtype=torch.int32))
    for x in step:
        x.normal_()
    graph.replay()
    torch.cuda.synchronize()
    return _follow(history, new, step)


HOME, FOREIGN = [2, 1, 0, 4, 4, 5], [0, 5, 2, 3, 3, 4]


def test_captured_fork_before_share():
    """share() with groups that a captured fork does not know is refused; known ones stay right under its replays, also while they are not read."""
    g = _gen(21)
    cache, history = _beams(g)
    cache.share(2)
    cache.share(0)
    parents, step = torch.arange(B, dtype=torch.int32, device="cuda"), _qkv(B, 1, g)
    graph, out = _captured(cache, step, parents)
    for new in (HOME, FOREIGN, HOME, HOME):
        history = _replay(graph, step, parents, new, history)
        _check(out, step[0], history)
    cache.sync_lengths()
    with pytest.raises(RuntimeError, match="captured"):
        cache.share(3)
    cache.share(2)
    assert cache.prefix_lengths.tolist() == [0, 48]
    for new in (HOME, [0, 0, 0, 3, 3, 3], [5, 0, 0, 0, 3, 3], HOME):
        history = _replay(graph, step, parents, new, history)
        _check(out, step[0], history)
        cache.sync_lengths()
        step = [x.normal_() for x in step]
        history = _follow(history, range(B), step)
        _check(cache.decode(*step), step[0], history)  # eager, over the prefixes
        _consistent(cache)
    assert cache.prefix_lengths.tolist() == [0, 0]


def test_two_captured_forks_under_different_shares():
    g = _gen(22)
    cache, history = _beams(g)
    cache.share(2)
    cache.share(3)
    cache.share(2)
    parents, step = torch.arange(B, dtype=torch.int32, device="cuda"), _qkv(B, 1, g)
    two = _captured(cache, step, parents)
    cache.sync_lengths()
    cache.share(3)
    three = _captured(cache, step, parents)
    rng = np.random.default_rng(22)
    for i in range(12):
        graph, out = (two, three)[i % 2]
        new = (HOME, [0, 0, 2, 2, 4, 5], rng.integers(0, B, B).tolist())[i % 3]
        history = _replay(graph, step, parents, new, history)
        _check(out, step[0], history)
        if i in (5, 8):
            cache.sync_lengths()
            cache.share(2)
            cache.share(3)


def test_step_captured_before_the_first_fork():
    """It has no copy on write, so pages cannot be shared behind it; freed and moved pages are no matter."""
    g = _gen(23)
    cache = _paged()
    q, k, v = _qkv(B, 33, g)
    cache.prefill(q, k, v)
    history, step = [[(k[b], v[b])] for b in range(B)], _qkv(B, 1, g)
    graph, out = _captured(cache, step)
    keep = torch.arange(B, dtype=torch.int32, device="cuda")

    def replay():
        for x in step:
            x.normal_()
        graph.replay()
        torch.cuda.synchronize()
        return _follow(history, range(B), step)

    for _ in range(3):
        history = replay()
        _check(out, step[0], history)
    cache.sync_lengths()
    for parents in ([0, 0, 2, 3, 4, 5], keep):
        with pytest.raises(RuntimeError, match="captured"):
            cache.fork(parents)
    cache.free([0, 1])
    assert cache.compact().item() == 3 * (B - 2)
    history[:2] = [[], []]
    cache.append(*_qkv(B, 1, g)[1:])  # eager, so that the freed rows have pages
    cache.sync_lengths()
    rows = [orc_row(cache, b) for b in range(B)]
    history = [[r] for r in rows]
    for _ in range(4):
        history = replay()
        _check(out, step[0], history)
    cache.sync_lengths()
    _consistent(cache)
    with pytest.raises(RuntimeError, match="captured"):
        cache.fork([2, 2, 2, 3, 4, 5])


def orc_row(cache, b):
    """(K, V) of sequence b, as the table has it."""
    n = int(cache.lengths[b])
    ids = cache.block_table[b, :-(-n // cache.page_size)].long()
    return tuple(x[ids].transpose(0, 1).flatten(1, 2)[:, :n].clone() for x in (cache.k, cache.v))
