"""The bookkeeping of the cache classes on the CPU: the operators that they call are replaced by the oracle's rules, and a capture by a flag
that says that one is going on.  What a step reads is checked through the tables alone: every cached row holds the number of its token."""
import numpy as np
import pytest
import torch

import dtorch_amd  # noqa: F401
from dtorch_amd.nn import kv_cache
from oracle import sdpa
from oracle import shared as orc

B, HKV, D, PAGE = 6, 1, 16, 16


class _OnDevice(torch.Tensor):
    """Whole numbers that the class takes for a tensor on the device."""
    is_cuda = property(lambda self: True)


def _parents(x):
    return torch.tensor(x, dtype=torch.int32).as_subclass(_OnDevice)


class _Operators:
    """dtorch_amd.nn.functional by the oracle's rules, on CPU tensors in place."""

    def __init__(self):
        self.capturing = False
        self.short = []
        self.bounds = []

    @staticmethod
    def scaled_dot_product_attention(q, k, v, **_):
        return torch.zeros_like(q)

    @staticmethod
    def kv_pages_fork(table, lengths, refs, parents):
        t, n, r = orc.fork(table.numpy(), lengths.numpy(), refs.numpy(), np.asarray(parents.tolist()))
        for x, y in ((table, t), (lengths, n), (refs, r)):
            x.copy_(torch.from_numpy(y))

    def kv_pages_reserve(self, pools, table, lengths, refs, n):
        p, t, r, short = orc.reserve([x.numpy() for x in pools], table.numpy(), lengths.numpy(), refs.numpy(), n, pools[0].shape[2])
        for x, y in zip([*pools, table, refs], [*p, t, r]):
            x.copy_(torch.from_numpy(y))
        self.short.append(short)
        return torch.tensor([short], dtype=torch.int32)

    @staticmethod
    def kv_pages_compact(pools, table, refs):
        p, t, r, used = orc.compact([x.numpy() for x in pools], table.numpy(), refs.numpy())
        for x, y in zip([*pools, table, refs], [*p, t, r]):
            x.copy_(torch.from_numpy(y))
        return torch.tensor([used], dtype=torch.int32)

    @staticmethod
    def kv_cache_append_paged(k, v, table, lengths, kn, vn):
        before = lengths.clone()
        sdpa.kv_append_paged(k.numpy(), table.numpy(), before.numpy(), kn.numpy())
        sdpa.kv_append_paged(v.numpy(), table.numpy(), lengths.numpy(), vn.numpy())

    @staticmethod
    def kv_cache_append(k, v, lengths, kn, vn):
        before = lengths.clone()
        sdpa.kv_append(k.numpy(), before.numpy(), kn.numpy())
        sdpa.kv_append(v.numpy(), lengths.numpy(), vn.numpy())

    @staticmethod
    def decode_attention_paged(q, k, v, table, lengths, scale=None):
        return torch.zeros_like(q), None

    @staticmethod
    def decode_attention_shared_paged(q, k, v, table, lengths, prefix, scale=None):
        return torch.zeros_like(q), None

    @staticmethod
    def decode_attention_shared(*_, **__):
        raise AssertionError("refusals come before this")


@pytest.fixture
def ops(monkeypatch):
    fake = _Operators()
    monkeypatch.setattr(kv_cache, "F", fake)
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: fake.capturing)
    return fake


def _cache(pages=60, batch=B, columns=12):
    return kv_cache.PagedKVCache(batch, HKV, pages, PAGE, columns, D, dtype=torch.float32, device="cpu")


def _tokens(first, batch=B, n=1):
    """q, k, v of tokens numbered first, first + 1, ..., a sequence's n one after another."""
    k = (first + torch.arange(batch * n, dtype=torch.float32)).view(batch, 1, n, 1).expand(batch, HKV, n, D).contiguous()
    return torch.zeros(batch, HKV, n, D), k, k.clone()


def _held(cache, b):
    """The numbers of the tokens of sequence b."""
    return orc.rows_of(cache.k.numpy(), cache.block_table.numpy(), b, np.arange(int(cache.lengths[b])))[:, 0, 0].tolist()


def _shares_hold(cache):
    """Every prefix is pages that the whole group has."""
    table = cache.block_table.numpy()
    for groups, shared in cache._shares.items():
        per = len(table) // groups
        for g, n in enumerate(shared.tolist()):
            rows = table[g * per:(g + 1) * per, :n // PAGE]
            assert (rows == rows[:1]).all(), (groups, g, n)


def _prompts(cache, n=50):
    cache.prefill(*_tokens(0, 2, n))
    cache.fork([0, 0, 0, 1, 1, 1])


def test_share_behind_a_captured_fork(ops):
    """A captured fork updates the prefixes that are there at its capture, so a number of groups that it does not know is refused."""
    cache = _cache()
    _prompts(cache)
    cache.share(2)
    ops.capturing = True
    cache.fork(_parents(range(B)))
    cache.decode(*_tokens(1000))
    ops.capturing = False
    cache.sync_lengths()
    with pytest.raises(RuntimeError, match="captured"):
        cache.share(3)
    assert cache.prefix_lengths.tolist() == [48, 48]
    cache.share(0)
    cache.share(2)
    assert cache.prefix_lengths.tolist() == [48, 48]


def test_share_never_called_before_a_captured_fork(ops):
    cache = _cache()
    _prompts(cache)
    ops.capturing = True
    cache.fork(_parents(range(B)))
    ops.capturing = False
    cache.sync_lengths()
    with pytest.raises(RuntimeError, match="captured"):
        cache.share(2)
    assert cache.prefix_lengths is None


def test_sync_lengths_brings_prefixes_down(ops):
    """Whatever changed the table on the device, sync_lengths leaves no prefix that a group does not have in common; none grows by it."""
    cache = _cache()
    _prompts(cache)
    cache.share(3)
    cache.share(2)
    held = cache.prefix_lengths
    ops.kv_pages_fork(cache.block_table, cache.lengths, cache.page_refs, torch.tensor([0, 5, 2, 3, 3, 4]))
    cache._host_stale = True
    cache.sync_lengths()
    _shares_hold(cache)
    assert cache.prefix_lengths is held and held.tolist() == [0, 48]
    ops.kv_pages_fork(cache.block_table, cache.lengths, cache.page_refs, torch.tensor([0, 0, 0, 3, 3, 3]))
    cache.sync_lengths()
    assert held.tolist() == [0, 48]
    cache.share(2)
    assert held.tolist() == [48, 48]


@pytest.mark.parametrize("seed", range(6))
def test_shares_through_any_order(ops, seed):
    """Forks on the host and on the device, steps, frees, compactions and syncs in any order: no prefix is more than what its group has."""
    rng = np.random.default_rng(seed)
    cache = _cache(pages=150, columns=20)
    _prompts(cache)
    cache.share(int(rng.choice([1, 2, 3])))
    for step in range(60):
        what = rng.integers(0, 6)
        if what == 0:
            parents = rng.integers(-1 if step % 3 == 0 else 0, B, B).tolist()
            cache.fork(_parents(parents) if rng.random() < 0.5 else parents)
        elif what == 1:
            cache.sync_lengths()
            cache.share(int(rng.choice([1, 2, 3, 6])))
        elif what == 2:
            cache.compact()
        elif what == 3 and step % 4 == 0:
            cache.free([int(rng.integers(0, B))])
        else:
            cache.decode(*_tokens(1000 * step))
        _shares_hold(cache)
    cache.sync_lengths()
    _shares_hold(cache)
