"""Pages that are lacking: slots whose tokens found none stay empty, whatever is freed later, and the class says so."""
import numpy as np
import pytest
import torch

from oracle import shared as orc
from test_gpu_cache_sharing import B, D, _consistent, _gen, _paged, _qkv
from test_gpu_shared_pages import _F, _i32, _num, _pools, _state

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("b,page,columns,P,n,heads", [(1, 16, 1, 3, 1, 1), (7, 16, 8, 60, 1, 2), (7, 64, 5, 30, 70, 1), (40, 32, 6, 90, 20, 1), (600, 16, 12, 9000, 90, 1),
                                                      (3000, 16, 2, 9000, 1, 1)])
@pytest.mark.parametrize("empty", [-1, -7, 1 << 20])
def test_reserve_lost_slots(b, page, columns, P, n, heads, empty):
    rng = np.random.default_rng(b + n)
    table, lengths, refs = _state(rng, b, page, columns, P)
    lost = rng.random(b) < 0.4
    lost[0] = True
    lengths[0] = min(max(lengths[0], 1) // page * page + 1, columns * page - 1)
    for i in np.flatnonzero(lost):  # the page of its last tokens is gone
        table[i, min(lengths[i], columns * page - 1) // page] = empty
    refs = orc.references(table, P)
    pools = _pools(rng, P, heads, page, 8, torch.float32, "scales")
    want_p, want_t, want_r, short = orc.reserve([_num(x) for x in pools], table, lengths, refs, n, page)
    assert short >= 1 and want_t[0, lengths[0] // page] == empty
    dev, dt, dr = [x.cuda() for x in pools], _i32(table), _i32(refs)
    assert _F().kv_pages_reserve(dev, dt, _i32(lengths), dr, n).tolist() == [short]
    assert np.array_equal(dt.cpu().numpy(), want_t) and np.array_equal(dr.cpu().numpy(), want_r)
    for a, w in zip(dev, want_p):
        assert np.array_equal(_num(a), w)


@pytest.mark.parametrize("captured", [False, True])
def test_class_after_a_shortage(captured):
    """Six sequences on one prompt of 20 tokens, nine pages: two find a third page.  One of these takes the place of the last sequence, whose pages are then free."""
    g = _gen(31)
    cache = _paged(pages=9)
    q, k, v = _qkv(1, 20, g)
    cache.prefill(q, k, v)
    cache.fork([0] * B)
    parents, step = torch.arange(B, dtype=torch.int32, device="cuda"), _qkv(B, 1, g)
    if captured:
        cache.share(1)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            cache.fork(parents)
            cache.decode(*step)
        cache.sync_lengths()

    def run(new):
        parents.copy_(torch.tensor(new, dtype=torch.int32))
        if captured:
            graph.replay()
        else:
            cache.fork(parents)
            cache.decode(*step)
        torch.cuda.synchronize()

    for _ in range(14):
        run(range(B))
    lacking = [b for b in range(B) if cache.block_table[b, 1].item() < 0 or cache.block_table[b, 2].item() < 0]
    assert lacking == [2, 3, 4, 5]
    well = next(b for b in range(B) if b not in lacking)
    run([well if b == B - 1 else -1 if b == well else b for b in range(B)])
    for _ in range(3):
        run(range(B))
    for _ in range(2):
        with pytest.raises(RuntimeError, match="past the assigned pages"):
            cache.sync_lengths()
    cache.free([b for b in range(B) if b != B - 1])
    assert cache.sync_lengths().tolist() == [0] * (B - 1) + [38]
    _consistent(cache)
    ids = cache.block_table[B - 1, :3].long()
    rows = cache.k[ids].transpose(1, 2).flatten(0, 1)[:38]
    assert torch.equal(rows[:20], k[0].transpose(0, 1)) and torch.equal(rows[20:34], step[1][well].transpose(0, 1).expand(14, -1, D))
    assert torch.equal(rows[34:], step[1][B - 1].transpose(0, 1).expand(4, -1, D))
    cache.decode(*_qkv(B, 1, g))
    _consistent(cache)
