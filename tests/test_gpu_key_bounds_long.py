"""Key bounds of more blocks than one launch's grid has rows (65535), in every block of a call, and the refresh behind an eviction."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("block,blocks,n", [(16, 65535, 0), (16, 262140, 1), (16, 262141, 0), (16, 300007, 5), (128, 65535, 0), (128, 65536, 0), (128, 66001, 77)])
@pytest.mark.parametrize("paged", [False, True])
def test_many_blocks(block, blocks, n, paged):
    """The last n tokens are missing from the last block; values are whole numbers, so the bounds are exact."""
    from dtorch_amd.nn import functional as F
    g = torch.Generator(device="cuda").manual_seed(block + blocks)
    per = 256 // block
    tokens = -(-blocks // per) * 256
    k = torch.randint(-99, 100, (1, 1, tokens, 8), generator=g, device="cuda").to(torch.bfloat16)
    length = torch.tensor([blocks * block - n], dtype=torch.int32, device="cuda")
    k[:, :, int(length):] = float("nan")  # nothing behind a sequence's tokens is read
    rows = k.clone()
    rows[:, :, int(length):] = float("inf")
    lo = rows.unflatten(2, (-1, block))[:, :, :blocks].float().amin(3)
    rows[:, :, int(length):] = -float("inf")
    hi = rows.unflatten(2, (-1, block))[:, :, :blocks].float().amax(3)
    shape = (1, 1, tokens // block, 8)
    if paged:
        pages = k.view(-1, 1, 256, 8)
        table = torch.randperm(len(pages), generator=g, device="cuda")
        pool = torch.empty_like(pages)
        pool[table] = pages
        got = [torch.full((len(pages), 1, per, 8), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        F.kv_key_bounds_paged(pool, *got, table.to(torch.int32)[None].contiguous(), length, tokens)
        got = [x[table].reshape(shape) for x in got]
    else:
        got = [torch.full(shape, 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
        F.kv_key_bounds(k, *got, length, tokens)
    for x, want in zip(got, (lo, hi)):
        assert torch.equal(x[:, :, :blocks].float(), want)
        assert (x[:, :, blocks:] == 7.0).all()


def test_evict_of_a_large_cache():
    """A cache of 2^20 positions in blocks of 16 has more blocks than a launch's grid has rows; the bounds follow the tokens that moved."""
    from dtorch_amd.nn import functional as F
    from dtorch_amd.nn.kv_cache import KVCache
    g = torch.Generator(device="cuda").manual_seed(5)
    cache = KVCache(2, 2, 1 << 20, 64, track_weights=True, bounds_block=16)
    cache.prefill(*[torch.randn(2, h, 500, 64, generator=g, device="cuda").to(torch.bfloat16) for h in (4, 2, 2)])
    cache.evict(100, 20)
    assert cache.lengths.tolist() == [100, 100]
    lo, hi = torch.zeros_like(cache.k_min), torch.zeros_like(cache.k_max)
    F.kv_key_bounds(cache.k, lo, hi, cache.lengths, 100)
    assert torch.equal(lo[:, :, :7], cache.k_min[:, :, :7]) and torch.equal(hi[:, :, :7], cache.k_max[:, :, :7])
    rows = cache.k[:, :, :96].unflatten(2, (6, 16)).float()
    assert torch.equal(lo[:, :, :6].float(), rows.amin(3)) and torch.equal(hi[:, :, :6].float(), rows.amax(3))
