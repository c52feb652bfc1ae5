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


def _shortage(ops):
    """Three pages: two sequences share one of 8 tokens, a third holds the others; a step with its parents on the device then lacks a page."""
    cache = _cache(pages=3, batch=3, columns=4)
    cache.append(*[x[:1] for x in _tokens(100, 3, 8)[1:]])
    cache.fork([0, 0, -1])
    rows = torch.arange(24.0).add(700).view(1, 1, 24, 1).expand(1, HKV, 24, D).contiguous()
    table, lengths = cache.block_table[2:], cache.lengths[2:]
    ops.kv_pages_reserve(cache._pools(), table, lengths, cache.page_refs, 24)
    ops.kv_cache_append_paged(cache.k, cache.v, table, lengths, rows, rows)
    cache._host_stale = True
    cache.sync_lengths()
    assert cache.lengths.tolist() == [8, 8, 24] and cache.block_table[2].tolist() == [1, 2, -1, -1] and not cache._free
    cache.fork(_parents([0, 1, 2]))
    ops.short.clear()
    cache.decode(*_tokens(800, 3))
    assert ops.short == [1] and cache.block_table[:2, 0].tolist() == [-1, 0]
    return cache


def test_a_shortage_is_not_filled_by_foreign_pages(ops):
    """A sequence whose page was lacking gets none in its middle once another ends: it would find the other's rows there."""
    cache = _shortage(ops)
    cache.fork(_parents([0, 1, -1]))
    for i in range(3):
        cache.decode(*_tokens(810 + i, 3))
    assert cache.block_table[0, 0].item() == -1
    for _ in range(2):  # as long as the sequence lives
        with pytest.raises(RuntimeError, match="past the assigned pages"):
            cache.sync_lengths()
    cache.free([0])
    assert cache.sync_lengths().tolist() == [0, 12, 3]
    assert _held(cache, 1) == [100.0 + i for i in range(8)] + [801.0, 811.0, 812.0, 813.0]
    cache.decode(*_tokens(900, 3))
    assert cache.lengths.tolist() == [1, 13, 4]


def test_a_shortage_is_reported_when_its_sequence_has_ended(ops):
    """Its steps attended to rows that were not its own, so the next sync says so, once."""
    cache = _shortage(ops)
    cache.fork(_parents([1, 1, -1]))
    cache.decode(*_tokens(820, 3))
    with pytest.raises(RuntimeError, match="past the assigned pages"):
        cache.sync_lengths()
    assert cache.sync_lengths().tolist() == [10, 10, 1]
    assert _held(cache, 0) == [100.0 + i for i in range(8)] + [801.0, 820.0]


@pytest.mark.parametrize("seed", range(8))
def test_small_pools(ops, seed):
    """Steps with parents on the device over a pool that is too small at times: what sync_lengths lets pass is whole, token by token."""
    rng = np.random.default_rng(seed)
    cache = _cache(pages=14, columns=20)
    cache.fork(list(range(B)))  # the device gives out the pages
    texts, lost = [[] for _ in range(B)], False
    for step in range(120):
        parents = rng.integers(-1 if rng.random() < 0.4 else 0, B, B).tolist()
        cache.fork(_parents(parents))
        texts = [list(texts[p]) if p >= 0 else [] for p in parents]
        ops.short.clear()
        cache.decode(*_tokens(1000 * (step + 1)))
        lost |= any(ops.short)
        for b in range(B):
            texts[b].append(1000.0 * (step + 1) + b)
        if rng.random() < 0.2:
            if lost:
                with pytest.raises(RuntimeError, match="past the assigned pages"):
                    cache.sync_lengths()
            try:
                cache.sync_lengths()
            except RuntimeError:
                lost = True
                continue
            lost = False
            for b in range(B):
                assert _held(cache, b) == texts[b]


def test_a_shortage_in_replays(ops):
    """Replays that the host does not see lack a page: until the sequence is freed the host goes by the device, not by what it knew."""
    cache = _shortage(ops)
    cache.fork(_parents([1, 1, 2]))
    with pytest.raises(RuntimeError):
        cache.sync_lengths()
    cache.free([2])
    assert cache.sync_lengths().tolist() == [9, 9, 0]
    q, k, v = _tokens(830, 3, 40)
    cache._lacking += ops.kv_pages_reserve(cache._pools(), cache.block_table, cache.lengths, cache.page_refs, 40)  # a replay
    ops.kv_cache_append_paged(cache.k, cache.v, cache.block_table, cache.lengths, k, v)
    with pytest.raises(RuntimeError, match="past the assigned pages"):
        cache.sync_lengths()
    with pytest.raises(RuntimeError, match="sync_lengths"):
        cache.share(1)
    cache.free([0, 2])
    with pytest.raises(RuntimeError, match="past the assigned pages"):
        cache.sync_lengths()
    cache.free([1])
    assert cache.sync_lengths().tolist() == [0, 0, 0] and len(cache._free) == 3


def test_fork_behind_a_step_captured_without_counts(ops):
    """A step captured before the first fork gives out no pages: its replays would write the pages that a fork lets sequences share."""
    cache = _cache()
    cache.prefill(*_tokens(0, B, 20))
    ops.capturing = True
    cache.decode(*_tokens(500))
    ops.capturing = False
    cache.sync_lengths()
    before = cache.block_table.clone()
    for parents in ([0, 0, 2, 3, 4, 5], [1, 2, 3, 4, 5, 5], _parents(range(B))):
        with pytest.raises(RuntimeError, match="captured"):
            cache.fork(parents)
    assert cache.page_refs is None and not cache._host_stale and torch.equal(cache.block_table, before)
    cache.fork([5, 4, 3, 2, 1, 0])  # no page in two sequences
    cache.free([2])
    assert cache.compact().item() == 10
    with pytest.raises(RuntimeError, match="captured"):
        cache.fork([0, 0, 2, 3, 4, 5])
    assert _held(cache, 0) == [100.0 + i for i in range(20)] + [505.0] and cache.lengths.tolist() == [21, 21, 0, 21, 21, 21]


def test_fork_behind_a_step_captured_with_counts(ops):
    cache = _cache()
    cache.prefill(*_tokens(0, B, 20))
    cache.compact()
    ops.capturing = True
    cache.decode(*_tokens(500))
    ops.capturing = False
    cache.sync_lengths()
    cache.fork([0, 0, 2, 3, 4, 5])
    cache.decode(*_tokens(600))
    assert _held(cache, 0)[20:] == [500.0, 600.0] and _held(cache, 1)[20:] == [500.0, 601.0]


def test_prefixes_of_too_many_groups(ops):
    """More groups than the shared decode takes are refused before the append."""
    cache, prefix = (kv_cache.KVCache(1025, HKV, 32, D, dtype=torch.float32, device="cpu") for _ in range(2))
    with pytest.raises(ValueError, match="1024"):
        cache.decode(*_tokens(0, 1025), prefix=prefix)
    assert not cache.lengths.any() and not cache._host_len.any()


def test_full_sequences_behind_device_parents(ops):
    """With its parents on the device the host does not know the lengths; a step that might not fit asks for them before tokens are dropped."""
    cache = _cache(columns=2)
    _prompts(cache, 20)
    for i in range(12):
        cache.fork(_parents([0, 1, 1, 3, 3, 3]))
        cache.decode(*_tokens(1000 + 10 * i))
    with pytest.raises(ValueError, match="max_pages"):
        cache.decode(*_tokens(2000))
    assert cache.sync_lengths().tolist() == [32] * B
    assert _held(cache, 5)[20:] == [1000.0 + 10 * i + (3 if i < 11 else 5) for i in range(12)]
    cache.fork(_parents([-1, 1, 2, 3, 4, 5]))
    with pytest.raises(ValueError, match="max_pages"):
        cache.decode(*_tokens(2000))
    cache.fork(_parents([-1] * 5 + [0]))  # the long ones end: the next step fits
    cache.decode(*_tokens(3000))
    assert cache.sync_lengths().tolist() == [1] * B and _held(cache, 5) == [3005.0]


def test_prefill_behind_device_parents(ops):
    """A row that was empty may have been given a parent's tokens."""
    cache = _cache()
    cache.prefill(*_tokens(0, 2, 20))
    cache.fork([-1, 1, -1, -1, -1, -1])
    cache.fork(_parents([1, 1, -1, -1, -1, -1]))
    with pytest.raises(ValueError, match="empty"):
        cache.prefill(*_tokens(500, 1, 8))
    cache.fork(_parents([-1, 1, -1, -1, -1, -1]))
    cache.sync_lengths()
    cache.prefill(*_tokens(500, 1, 8))
    assert _held(cache, 0) == [500.0 + i for i in range(8)] and _held(cache, 1) == [20.0 + i for i in range(20)]


def test_ended_sequences_follow_a_sibling(ops):
    """Samples that end at different times: a row that goes on behind a living one keeps its group's prefix."""
    cache = _cache()
    _prompts(cache)
    cache.share(2)
    for i, parents in enumerate(([0, 0, 2, 3, 4, 5], [0, 0, 0, 3, 3, 5], [0, 0, 0, 3, 3, 3])):
        for j in range(20):
            cache.decode(*_tokens(1000 * (i + 1) + 10 * j))
        cache.fork(parents)
        assert cache.prefix_lengths.min() >= 48
        _shares_hold(cache)
    assert _held(cache, 2)[50:] == [1000.0 * (i + 1) + 10 * j for i in range(3) for j in range(20)]


def test_a_prompt_for_a_freed_row(ops):
    cache = _cache()
    cache.prefill(*_tokens(0, 3, 20))
    cache.free([1])
    with pytest.raises(ValueError, match="empty"):
        cache.prefill(*_tokens(500, 2, 8))
    cache.fork([1, 0, 2, 3, 4, 5])
    cache.prefill(*_tokens(500, 1, 8))
    assert [_held(cache, b)[0] for b in range(3)] == [500.0, 0.0, 40.0] and cache.lengths.tolist() == [8, 20, 20, 0, 0, 0]
