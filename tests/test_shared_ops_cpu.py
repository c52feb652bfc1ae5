"""What the entry points over shared pages, a shared prefix and selected key blocks refuse before they touch a device, what their
parameters keep through serialisation, and the oracle's own rules.  Every pointer here is made up: a call that is not refused is an
empty one."""
import ctypes
import pickle

import numpy as np
import pytest

import dtorch_amd  # noqa: F401  (loads libtorch's libraries first)
from dtorch_amd import _lib
from oracle import shared as orc

lib = _lib.cabi()
P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
SZ = ctypes.c_size_t


def _struct(fields):
    return type("Args", (ctypes.Structure,), {"_fields_": fields})


Pool = _struct([("data", P), ("heads", I64), ("row_bytes", I64), ("row_tokens", I64), ("page_stride", I64), ("head_stride", I64), ("row_stride", I64)])
Fork = _struct([("block_table", P), ("lengths", P), ("page_refs", P), ("parents", P), ("B", I64), ("max_pages", I64), ("num_pages", I64),
                ("block_table_stride", I64)])
Reserve = _struct([("pools", Pool * 8), ("n_pools", I32), ("block_table", P), ("lengths", P), ("page_refs", P), ("short_by", P), ("B", I64),
                   ("max_pages", I64), ("num_pages", I64), ("page_size", I64), ("n_new", I64), ("block_table_stride", I64), ("workspace", P),
                   ("workspace_bytes", SZ)])
Compact = _struct([("pools", Pool * 8), ("n_pools", I32), ("block_table", P), ("page_refs", P), ("used", P), ("B", I64), ("max_pages", I64),
                   ("num_pages", I64), ("page_size", I64), ("block_table_stride", I64), ("workspace", P), ("workspace_bytes", SZ)])
Shared = _struct([("q", P), ("k_prefix", P), ("v_prefix", P), ("k_cache", P), ("v_cache", P), ("block_table", P), ("prefix_lengths", P),
                  ("lengths", P), ("o", P), ("lse", P), ("B", I64), ("groups", I64), ("Hq", I64), ("Hkv", I64), ("D", I64), ("S_prefix", I64),
                  ("S_max", I64), ("num_pages", I64), ("page_size", I64), ("max_pages", I64), ("q_stride", I64 * 2),
                  ("k_prefix_stride", I64 * 3), ("v_prefix_stride", I64 * 3), ("k_stride", I64 * 3), ("v_stride", I64 * 3),
                  ("o_stride", I64 * 2), ("lse_stride", I64 * 1), ("block_table_stride", I64), ("dtype", I32), ("scale", F), ("workspace", P),
                  ("workspace_bytes", SZ)])
Bounds = _struct([("k_cache", P), ("k_min", P), ("k_max", P), ("block_table", P), ("lengths", P), ("B", I64), ("Hkv", I64), ("D", I64),
                  ("n_new", I64), ("S_max", I64), ("num_pages", I64), ("page_size", I64), ("max_pages", I64), ("k_stride", I64 * 3),
                  ("min_stride", I64 * 3), ("max_stride", I64 * 3), ("block_table_stride", I64), ("block", I32), ("dtype", I32)])
Select = _struct([("q", P), ("k_min", P), ("k_max", P), ("block_table", P), ("lengths", P), ("blocks", P), ("B", I64), ("Hq", I64),
                  ("Hkv", I64), ("D", I64), ("keep", I64), ("recent", I64), ("S_max", I64), ("num_pages", I64), ("page_size", I64),
                  ("max_pages", I64), ("q_stride", I64 * 2), ("min_stride", I64 * 3), ("max_stride", I64 * 3), ("block_table_stride", I64),
                  ("block", I32), ("dtype", I32), ("scale", F), ("workspace", P), ("workspace_bytes", SZ)])
Blocks = _struct([("q", P), ("k_cache", P), ("v_cache", P), ("block_table", P), ("lengths", P), ("blocks", P), ("o", P), ("lse", P), ("B", I64),
                  ("Hq", I64), ("Hkv", I64), ("D", I64), ("n_blocks", I64), ("S_max", I64), ("num_pages", I64), ("page_size", I64),
                  ("max_pages", I64), ("q_stride", I64 * 2), ("k_stride", I64 * 3), ("v_stride", I64 * 3), ("blocks_stride", I64 * 2),
                  ("o_stride", I64 * 2), ("lse_stride", I64 * 1), ("block_table_stride", I64), ("block", I32), ("dtype", I32), ("scale", F),
                  ("workspace", P), ("workspace_bytes", SZ)])
KINDS = {"fork": (Fork, "dtattn_kv_pages_fork"), "reserve": (Reserve, "dtattn_kv_pages_reserve"), "compact": (Compact, "dtattn_kv_pages_compact"),
         "shared": (Shared, "dtattn_decode_shared"), "bounds": (Bounds, "dtattn_key_bounds"), "select": (Select, "dtattn_select_key_blocks"),
         "blocks": (Blocks, "dtattn_decode_blocks")}


def _args(kind, paged, kw):
    a = KINDS[kind][0]()
    for i, (name, t) in enumerate(a._fields_):
        if t is P and name not in ("workspace",) and not (name == "block_table" and kind in ("shared", "bounds", "select", "blocks")):
            setattr(a, name, 0x10000 * (i + 1))
    S, D, B, Hkv = 256, 128, 2, 4
    a.B = B
    if kind in ("fork", "reserve", "compact"):
        a.max_pages, a.num_pages, a.block_table_stride = 4, 8, 4
    if kind in ("reserve", "compact"):
        a.page_size, a.n_pools = 64, 2
        for i in range(2):
            a.pools[i] = Pool(0x770000 + 0x1000 * i, Hkv, 2 * D, 1, Hkv * 64 * 2 * D, 64 * 2 * D, 2 * D)
    if kind == "reserve":
        a.n_new = 1
    if kind in ("shared", "bounds", "select", "blocks"):
        a.Hkv, a.D, a.S_max = Hkv, D, S
        if paged:
            a.block_table, a.block_table_stride, a.num_pages, a.page_size, a.max_pages = 0x990000, 4, 8, 64, 4
        for name, _ in a._fields_:
            if name.endswith("_stride") and name not in ("block_table_stride", "blocks_stride", "lse_stride"):
                s = getattr(a, name)
                for i, x in enumerate((Hkv * S * D, S * D, D)[:len(s)]):
                    s[i] = x
    if kind == "shared":
        a.groups, a.S_prefix, a.Hq, a.scale = 1, S, 8, float("nan")
    if kind in ("bounds", "select", "blocks"):
        a.block = 32
    if kind == "bounds":
        a.n_new = 1
    if kind == "select":
        a.Hq, a.keep, a.recent, a.scale = 8, 128, 32, float("nan")
    if kind == "blocks":
        a.Hq, a.n_blocks, a.scale = 8, 4, float("nan")
    for name, v in kw.items():
        target = a
        if name.startswith("pool1_"):
            target, name = a.pools[1], name[6:]
        field = getattr(target, name)
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                field[i] = x
        else:
            setattr(target, name, v)
    return a


def _call(kind, a):
    fn = getattr(lib, KINDS[kind][1])
    fn.restype, fn.argtypes = ctypes.c_int, [P, P]
    lib.dtattn_last_error.restype = ctypes.c_char_p
    return fn(ctypes.addressof(a), None), lib.dtattn_last_error().decode()


TABLE = [(dict(B=-1), 1, "bad sizes"), (dict(max_pages=0), 1, "bad sizes"), (dict(num_pages=0), 1, "bad sizes"), (dict(num_pages=1 << 31), 1, "bad sizes"),
         (dict(block_table_stride=3), 1, "overlap"), (dict(block_table=None), 1, "null")]
POOLS = [(dict(n_pools=0), 1, "pools"), (dict(n_pools=9), 1, "pools"), (dict(page_size=8), 1, "page_size"), (dict(page_size=48), 1, "page_size"),
         (dict(max_pages=1 << 25, block_table_stride=1 << 25), 1, "too many pages"), (dict(pool1_data=None), 1, "pool 1 is NULL"),
         (dict(pool1_data=0x770000), 1, "same memory"), (dict(pool1_row_tokens=128), 1, "bad sizes"), (dict(pool1_row_tokens=0), 1, "bad sizes"),
         (dict(pool1_heads=0), 1, "bad sizes"), (dict(pool1_row_bytes=6), 2, "multiples of 4"), (dict(pool1_data=0x771002), 2, "multiples of 4"),
         (dict(pool1_head_stride=-256), 2, "negative"), (dict(page_refs=None), 1, "null")]
ROWS = [(dict(D=12), 2, "head dim"), (dict(D=136), 2, "head dim"), (dict(D=256), 2, "head dim"), (dict(dtype=2), 2, "dtype"), (dict(dtype=7), 2, "dtype"),
        (dict(B=-1), 1, "bad sizes"), (dict(Hkv=0), 1, "bad sizes"), (dict(lengths=None), 1, "null")]
HEADS = [(dict(Hq=6), 1, "multiple"), (dict(Hq=0), 1, "bad sizes"), (dict(scale=float("inf")), 1, "scale"), (dict(q=None), 1, "null"), (dict(q=0x10008), 2, "aligned"),
         (dict(q_stride=(1024, 100)), 2, "16 bytes")]
CACHES = [(dict(k_cache=None), 1, "null"), (dict(k_cache=0x10004), 2, "aligned"), (dict(v_stride=(4096, 4096, 100)), 2, "16 bytes"),
          (dict(k_stride=(4096, 4096, 64)), 2, "row stride"), (dict(k_stride=(0, 0, 1 << 24)), 2, "row stride"), (dict(o=None), 1, "null")]
BLOCK = [(dict(block=8), 1, "block 8"), (dict(block=48), 1, "block 48"), (dict(block=512), 1, "block 512"), (dict(block=0), 1, "block 0"), (dict(block=-16), 1, "block")]
PAGED = [(dict(page_size=8), 1, "page_size"), (dict(page_size=48), 1, "page_size"), (dict(num_pages=0), 1, "page counts"), (dict(max_pages=0), 1, "page counts"),
         (dict(max_pages=1 << 24), 1, "page counts")]
OWN = {
    "fork": TABLE + [(dict(B=8193), 2, "8192"), (dict(parents=None), 1, "null"), (dict(lengths=0x40000, parents=0x40000), 1, "same memory")],
    "reserve": TABLE + POOLS + [(dict(short_by=None), 1, "null"), (dict(n_new=-1), 1, "new tokens"), (dict(workspace=None), 3, "workspace"),
                                (dict(workspace=0x10080, workspace_bytes=1 << 30), 3, "256-byte")],
    "compact": TABLE + POOLS + [(dict(used=None), 1, "null"), (dict(workspace=None), 3, "workspace"), (dict(workspace=0x10080, workspace_bytes=1 << 30), 3, "256-byte")],
    "shared": ROWS + HEADS + CACHES + [(dict(groups=0), 1, "bad sizes"), (dict(groups=3), 1, "equal groups"), (dict(B=4098, groups=2049), 2, "groups"), (dict(B=1025, groups=1025), 2, "groups"),
                                       (dict(prefix_lengths=None), 1, "null"), (dict(k_prefix=None), 1, "null"), (dict(S_prefix=0), 1, "capacities"),
                                       (dict(S_max=(1 << 29) + 1), 1, "capacities"), (dict(v_prefix_stride=(0, 0, 64)), 2, "row stride")],
    "bounds": ROWS + BLOCK + [(dict(n_new=-1), 1, "bad sizes"), (dict(k_min=0x880000, k_max=0x880000), 1, "share memory"), (dict(k_min=None), 1, "null"),
                              (dict(S_max=250), 1, "S_max"), (dict(max_stride=(0, 0, 100)), 2, "16 bytes"), (dict(k_max=0x880004), 2, "aligned")],
    "select": ROWS + HEADS + BLOCK + [(dict(keep=16), 1, "keep"), (dict(keep=100), 1, "keep"), (dict(recent=0), 1, "keep"), (dict(recent=48), 1, "keep"),
                                      (dict(recent=160), 1, "keep"), (dict(blocks=None), 1, "null"), (dict(S_max=250), 1, "S_max"),
                                      (dict(S_max=1 << 28), 3, "workspace")],
    "blocks": ROWS + HEADS + CACHES + BLOCK + [(dict(n_blocks=0), 1, "bad sizes"), (dict(blocks=None), 1, "null"), (dict(S_max=0), 1, "capacity")],
}


@pytest.mark.parametrize("kind,kw,code,text", [(k, *c) for k, cs in OWN.items() for c in cs])
def test_refusals(kind, kw, code, text):
    got = _call(kind, _args(kind, False, kw))
    assert got[0] == code and text in got[1], got


@pytest.mark.parametrize("kind", ["shared", "bounds", "select", "blocks"])
@pytest.mark.parametrize("kw,code,text", PAGED)
def test_paged_refusals(kind, kw, code, text):
    got = _call(kind, _args(kind, True, kw))
    assert got[0] == code and text in got[1], got


@pytest.mark.parametrize("kind", ["bounds", "select", "blocks"])
def test_pages_hold_whole_blocks(kind):
    got = _call(kind, _args(kind, True, dict(page_size=16)))
    assert got[0] == 1 and "does not hold" in got[1], got


@pytest.mark.parametrize("kind", list(KINDS))
def test_null_and_empty(kind):
    fn = getattr(lib, KINDS[kind][1])
    fn.restype, fn.argtypes = ctypes.c_int, [P, P]
    assert fn(None, None) == 1
    if kind not in ("reserve", "compact"):  # those write a count
        assert _call(kind, _args(kind, False, dict(B=0)))[0] == 0


@pytest.mark.parametrize("name,kw", [("TokenCountParam", dict(tokens=7)), ("SdpaDecodeSharedParam", dict(scale=0.25)), ("SdpaDecodeSharedParam", dict(scale=None)),
                                     ("SelectKeyBlocksParam", dict(keep=256, recent=32, block=16, scale=-1.0)), ("SdpaDecodeBlocksParam", dict(block=64, scale=None)),
                                     ("KvPagesForkParam", {}), ("KvPagesCompactParam", {})])
def test_params(name, kw):
    host = _lib.load()
    cls = getattr(host, name)
    p = cls(**kw)
    for q in (cls.from_bytes(p.to_bytes()), pickle.loads(pickle.dumps(p))):
        assert q.to_bytes() == p.to_bytes()
        for n, v in kw.items():
            assert getattr(q, n) == v


def test_device_tensors_only():
    import torch
    from dtorch_amd.nn import functional as fn
    t = torch.zeros(2, 4, dtype=torch.int32)
    with pytest.raises(ValueError, match="device tensors"):
        fn.kv_pages_fork(t, t[:, 0].contiguous(), torch.zeros(8, dtype=torch.int32), t[:, 0].contiguous())


def test_oracle_counts_stay_in_step():
    """Through random forks, reserves and compactions the counts are those of the table, and what a sequence holds stays."""
    rng = np.random.default_rng(0)
    page, P, B, columns = 16, 60, 5, 8
    pool = np.arange(P * page, dtype=np.float64).reshape(P, 1, page, 1)
    table, lengths, refs = np.full((B, columns), -1, dtype=np.int32), np.zeros(B, dtype=np.int32), np.zeros(P, dtype=np.int32)
    texts = [[] for _ in range(B)]
    for step in range(200):
        what = rng.integers(0, 3)
        if what == 0:
            parents = rng.integers(-1, B, B)
            table, lengths, refs = orc.fork(table, lengths, refs, parents)
            texts = [list(texts[p]) if p >= 0 else [] for p in parents]
        elif what == 1:
            n = int(rng.integers(1, 20))
            if (lengths + n).max() > page * columns:
                continue
            (pool,), table, refs, short = orc.reserve([pool], table, lengths, refs, n, page)
            assert short == 0
            for b in range(B):
                for i in range(n):
                    t = lengths[b] + i
                    pool[table[b, t // page], 0, t % page] = 1e4 * step + 100 * b + i
                    texts[b].append(1e4 * step + 100 * b + i)
            lengths = lengths + n
        else:
            (pool,), table, refs, used = orc.compact([pool], table, refs)
            assert (refs[:used] > 0).all() and (refs[used:] == 0).all()
        assert np.array_equal(refs, orc.references(table, P))
        for b in range(B):
            assert orc.rows_of(pool, table, b, np.arange(lengths[b]))[:, 0, 0].tolist() == texts[b]
