"""What the entry points over the 8-bit and the bounded KV cache refuse before they touch a device, and what their
parameters keep through serialisation.  Every pointer here is made up: a call that is not refused is an empty one."""
import ctypes
import pickle
import struct

import numpy as np
import pytest
import torch

import dtorch_amd  # noqa: F401  (loads libtorch's libraries first)
from dtorch_amd import _lib
from oracle import cache as orc

lib = _lib.cabi()
P, I32, I64, F = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64, ctypes.c_float
SZ = ctypes.c_size_t


def _struct(fields):
    return type("Args", (ctypes.Structure,), {"_fields_": fields})


Append = _struct([("k_new", P), ("v_new", P), ("k_cache", P), ("v_cache", P), ("k_scale", P), ("v_scale", P), ("block_table", P),
                  ("lengths", P), ("B", I64), ("Hkv", I64), ("n_new", I64), ("D", I64), ("S_max", I64), ("num_pages", I64),
                  ("page_size", I64), ("max_pages", I64), ("k_new_stride", I64 * 3), ("v_new_stride", I64 * 3), ("k_stride", I64 * 3),
                  ("v_stride", I64 * 3), ("k_scale_stride", I64 * 2), ("v_scale_stride", I64 * 2), ("block_table_stride", I64),
                  ("block", I32), ("dtype", I32)])
Decode = _struct([("q", P), ("k_cache", P), ("v_cache", P), ("k_scale", P), ("v_scale", P), ("block_table", P), ("lengths", P), ("o", P),
                  ("lse", P), ("B", I64), ("Hq", I64), ("Hkv", I64), ("D", I64), ("S_max", I64), ("num_pages", I64), ("page_size", I64),
                  ("max_pages", I64), ("q_stride", I64 * 2), ("k_stride", I64 * 3), ("v_stride", I64 * 3), ("k_scale_stride", I64 * 2),
                  ("v_scale_stride", I64 * 2), ("o_stride", I64 * 2), ("lse_stride", I64 * 1), ("block_table_stride", I64), ("block", I32),
                  ("dtype", I32), ("scale", F), ("workspace", P), ("workspace_bytes", SZ)])
Weights = _struct([("weights", P), ("q", P), ("k", P), ("k_scale", P), ("lse", P), ("lengths", P), ("B", I64), ("Hq", I64), ("Hkv", I64),
                   ("L", I64), ("S", I64), ("D", I64), ("w_stride", I64 * 2), ("q_stride", I64 * 3), ("k_stride", I64 * 3),
                   ("k_scale_stride", I64 * 2), ("lse_stride", I64 * 2), ("q_offset", I64), ("causal", I32), ("block", I32),
                   ("q_dtype", I32), ("k_dtype", I32), ("scale", F), ("workspace", P), ("workspace_bytes", SZ)])
Evict = _struct([("k_cache", P), ("v_cache", P), ("k_scale", P), ("v_scale", P), ("weights", P), ("lengths", P), ("kept", P), ("B", I64),
                 ("Hkv", I64), ("S_max", I64), ("keep", I64), ("recent", I64), ("block", I64), ("scale_block", I64), ("row_bytes", I64),
                 ("k_stride", I64 * 3), ("v_stride", I64 * 3), ("k_scale_stride", I64 * 2), ("v_scale_stride", I64 * 2),
                 ("w_stride", I64 * 2), ("workspace", P), ("workspace_bytes", SZ)])
KINDS = {"append": (Append, "dtattn_kv_append_fp8"), "decode": (Decode, "dtattn_decode_fp8"),
         "weights": (Weights, "dtattn_attention_weights"), "evict": (Evict, "dtattn_kv_evict")}


def _args(kind, paged, kw):
    a = KINDS[kind][0]()
    for i, (name, t) in enumerate(a._fields_):
        if t is P and name not in ("block_table", "workspace"):
            setattr(a, name, 0x10000 * (i + 1))
    S, D, B, Hkv = 256, 128, 2, 4
    a.B, a.Hkv = B, Hkv
    if kind == "append":
        a.n_new = 5
        for s in (a.k_new_stride, a.v_new_stride):
            s[0], s[1], s[2] = Hkv * 5 * D, 5 * D, D
    if kind in ("decode", "weights"):
        a.Hq, a.scale = 8, float("nan")
    if kind in ("append", "decode"):
        a.D, a.S_max, a.block = D, S, 32
        if paged:
            a.block_table, a.block_table_stride = 0x990000, 4
            a.num_pages, a.page_size, a.max_pages = 8, 64, 4
    if kind == "decode":
        for s in (a.q_stride, a.o_stride):
            s[0], s[1] = 8 * D, D
    if kind == "weights":
        a.k_scale = None
        a.L, a.S, a.D = 1, S, D
        a.q_stride[0], a.q_stride[1], a.q_stride[2] = 8 * D, D, D
    if kind == "evict":
        a.k_scale = a.v_scale = None
        a.S_max, a.keep, a.recent, a.block, a.scale_block, a.row_bytes = S, 64, 16, 1, 1, 2 * D
    if kind != "weights":
        for s in (a.k_stride, a.v_stride):
            s[0], s[1], s[2] = Hkv * S * D, S * D, D
    else:
        a.k_stride[0], a.k_stride[1], a.k_stride[2] = Hkv * S * D, S * D, D
    for name, v in kw.items():
        field = getattr(a, name)
        if isinstance(v, tuple):
            for i, x in enumerate(v):
                field[i] = x
        else:
            setattr(a, name, v)
    return a


def _call(kind, a):
    fn = getattr(lib, KINDS[kind][1])
    fn.restype, fn.argtypes = ctypes.c_int, [P, P]
    lib.dtattn_last_error.restype = ctypes.c_char_p
    code = fn(ctypes.addressof(a), None)
    return code, lib.dtattn_last_error().decode()


CACHE = [
    (dict(D=8), 2, "head dim"), (dict(D=136), 2, "head dim"), (dict(D=144), 2, "head dim"), (dict(D=0), 1, "bad sizes"),
    (dict(block=8), 1, "block 8"), (dict(block=48), 1, "block 48"), (dict(block=512), 1, "block 512"), (dict(block=0), 1, "block 0"),
    (dict(block=-32), 1, "block"), (dict(S_max=0), 1, "S_max"), (dict(S_max=250), 1, "S_max"), (dict(S_max=(1 << 29) + 32), 1, "S_max"),
    (dict(k_cache=None), 1, "null"), (dict(v_scale=None), 1, "null"), (dict(lengths=None), 1, "null"), (dict(k_cache=0x10008), 2, "aligned"),
    (dict(k_stride=(4096, 4096, 120)), 2, "16 bytes"), (dict(v_stride=(4096, 4096, 112)), 2, "row stride"),
    (dict(k_stride=(0, 0, (1 << 24) + 16)), 2, "row stride"), (dict(dtype=2), 2, "dtype"), (dict(dtype=5), 2, "dtype"), (dict(B=-1), 1, "bad sizes"),
    (dict(Hkv=0), 1, "bad sizes"),
]
PAGED = [(dict(page_size=8), 1, "page_size"), (dict(page_size=48), 1, "page_size"), (dict(page_size=16), 1, "does not hold"),
         (dict(num_pages=0), 1, "page counts"), (dict(max_pages=0), 1, "page counts"), (dict(max_pages=1 << 24), 1, "page counts")]


@pytest.mark.parametrize("kind", ["append", "decode"])
@pytest.mark.parametrize("kw,code,text", CACHE)
def test_cache_refusals(kind, kw, code, text):
    got = _call(kind, _args(kind, False, kw))
    assert got[0] == code and text in got[1], got


@pytest.mark.parametrize("kind", ["append", "decode"])
@pytest.mark.parametrize("kw,code,text", PAGED)
def test_paged_refusals(kind, kw, code, text):
    got = _call(kind, _args(kind, True, kw))
    assert got[0] == code and text in got[1], got


@pytest.mark.parametrize("kind,kw,code,text", [
    ("append", dict(n_new=-1), 1, "bad sizes"), ("append", dict(n_new=1 << 30), 2, "too many"), ("append", dict(k_new=None), 1, "null"),
    ("append", dict(v_new=0x20008), 2, "aligned"), ("append", dict(k_new_stride=(8, 8, 4)), 2, "16 bytes"),
    ("append", dict(v_cache=0x30000), 1, "share memory"), ("append", dict(v_scale=0x50000), 1, "share memory"),
    ("append", dict(B=1 << 20, Hkv=1 << 15), 2, "grid too large"),
    ("decode", dict(Hq=6), 1, "multiple"), ("decode", dict(Hq=0), 1, "bad sizes"), ("decode", dict(o=None), 1, "null"),
    ("decode", dict(q=0x10008), 2, "aligned"), ("decode", dict(o_stride=(1024, 4)), 2, "16 bytes"), ("decode", dict(scale=float("inf")), 1, "finite"),
    ("decode", dict(B=1 << 20, Hq=1 << 20), 2, "grid too large"),
    ("weights", dict(Hq=6), 1, "multiple"), ("weights", dict(L=-1), 1, "bad sizes"), ("weights", dict(S=-1), 1, "bad sizes"),
    ("weights", dict(q_dtype=2), 2, "dtype"), ("weights", dict(k_dtype=1), 2, "query's dtype"), ("weights", dict(D=136), 2, "head dim"),
    ("weights", dict(D=100), 2, "head dim"), ("weights", dict(D=24, k_dtype=2, block=16), 2, "head dim"), ("weights", dict(B=70000), 2, "grid"),
    ("weights", dict(S=1 << 30), 2, "grid"), ("weights", dict(q_offset=1 << 41), 1, "q_offset"), ("weights", dict(scale=float("inf")), 1, "finite"),
    ("weights", dict(k_dtype=2, block=24), 1, "block 24"), ("weights", dict(k_dtype=2, block=32, S=250), 1, "divides S"),
    ("weights", dict(k_dtype=2, block=32), 1, "null"), ("weights", dict(lse=None), 1, "null"), ("weights", dict(q=0x10004), 2, "aligned"),
    ("weights", dict(q_stride=(1024, 4, 128)), 2, "16 bytes"),
    ("evict", dict(keep=0, recent=0), 1, "keep"), ("evict", dict(recent=0), 1, "recent"), ("evict", dict(recent=65), 1, "recent"),
    ("evict", dict(block=3), 1, "block 3"), ("evict", dict(block=512, keep=512, recent=512), 1, "block 512"), ("evict", dict(block=16, keep=72), 1, "multiples"),
    ("evict", dict(block=16, recent=24), 1, "multiples"), ("evict", dict(row_bytes=24), 2, "row"), ("evict", dict(k_scale=0x30000), 1, "scales"),
    ("evict", dict(k_scale=0x30000, v_scale=0x40000, scale_block=32, block=16), 1, "multiple"), ("evict", dict(S_max=0), 1, "bad sizes"),
    ("evict", dict(k_stride=(65536, 32768, 120)), 2, "16 bytes"), ("evict", dict(k_cache=0x10008), 2, "aligned"), ("evict", dict(weights=None), 1, "null"),
    ("evict", dict(v_cache=0x10000), 1, "share memory"), ("evict", dict(B=1 << 20, Hkv=1 << 12), 2, "grid"),
    ("evict", dict(), 3, "workspace"), ("evict", dict(workspace=0x990000, workspace_bytes=8), 3, "workspace"),
    ("evict", dict(workspace=0x990010, workspace_bytes=1 << 30), 3, "aligned"),
])
def test_refusals(kind, kw, code, text):
    got = _call(kind, _args(kind, False, kw))
    assert got[0] == code and text in got[1], got


@pytest.mark.parametrize("kind", list(KINDS))
def test_null_arguments(kind):
    fn = getattr(lib, KINDS[kind][1])
    fn.restype, fn.argtypes = ctypes.c_int, [P, P]
    assert fn(None, None) == 1


@pytest.mark.parametrize("kind,kw", [("append", dict(B=0)), ("decode", dict(B=0)), ("weights", dict(B=0)), ("weights", dict(L=0)),
                                     ("weights", dict(S=0)), ("evict", dict(B=0))])
def test_empty_calls_are_no_ops(kind, kw):
    assert _call(kind, _args(kind, False, kw))[0] == 0


def test_workspace_of_an_eviction():
    fn = lib.dtattn_kv_evict_workspace_size
    fn.restype, fn.argtypes = SZ, [P]
    assert fn(None) == 0
    sizes = [fn(ctypes.addressof(_args("evict", False, dict(S_max=s)))) for s in (1, 256, 16384, 16385, 1 << 20)]
    assert sizes == sorted(sizes) and sizes[0] > 0
    # what 1024 threads do not hold in registers is held in the workspace: a word per candidate
    assert sizes[4] >= 2 * 4 * (1 << 20) * 4


def test_params_round_trip():
    host = _lib.load()
    p = pickle.loads(pickle.dumps(host.AttentionWeightsParam(0.25, True, -7)))
    assert (p.scale, p.is_causal, p.q_offset) == (0.25, True, -7)
    p = pickle.loads(pickle.dumps(host.AttentionWeightsParam(None, False, 1 << 40)))
    assert (p.scale, p.is_causal, p.q_offset) == (None, False, 1 << 40)
    p = pickle.loads(pickle.dumps(host.KvCacheEvictParam(1 << 33, 64, 16)))
    assert (p.keep, p.recent, p.block) == (1 << 33, 64, 16)
    assert host.SdpaDecodeFp8Op(0.5).param.scale == 0.5 and host.SdpaDecodeFp8Op().param.scale is None


def test_param_bytes():
    """The fields in their order: little-endian scalars, a presence byte before the optional scale."""
    host = _lib.load()
    cases = [(host.KvCacheAppendFp8Param(), b""), (host.KvCacheAppendFp8PagedParam(), b""),
             (host.SdpaDecodeFp8Param(0.5), struct.pack("<Bd", 1, 0.5)), (host.SdpaDecodeFp8PagedParam(None), struct.pack("<B", 0)),
             (host.AttentionWeightsParam(0.25, True, -3), struct.pack("<BdBq", 1, 0.25, 1, -3)),
             (host.KvCacheEvictParam(64, 16, 8), struct.pack("<qqq", 64, 16, 8))]
    for p, want in cases:
        assert p.to_bytes() == want, type(p)
        assert type(p).from_bytes(want).to_bytes() == want and type(pickle.loads(pickle.dumps(p))) is type(p)
        with pytest.raises(ValueError, match="trailing"):
            type(p).from_bytes(want + b"x")


def test_host_operators_need_the_device():
    import dtorch_amd.nn.functional as F
    k = torch.zeros(1, 2, 32, 64, dtype=torch.uint8).view(torch.float8_e4m3fn)
    s, ln, x = torch.ones(1, 2, 1), torch.zeros(1, dtype=torch.int32), torch.zeros(1, 2, 1, 64)
    w = torch.zeros(1, 2, 32)
    for call in (lambda: F.kv_cache_append_fp8(k, k, s, s, ln, x, x), lambda: F.decode_attention_fp8(x, k, k, s, s, ln),
                 lambda: F.attention_weight_accumulate(w, x, x.expand(1, 2, 32, 64), torch.zeros(1, 2)),
                 lambda: F.kv_cache_evict(x, x, ln, w[..., :1], 1, 1)):
        with pytest.raises(ValueError, match="device tensors"):
            call()


@pytest.mark.parametrize("kw,text", [
    (dict(dtype=torch.float8_e4m3fn, block=24), "block|tokens of a scale"), (dict(dtype=torch.float8_e4m3fn, block=512), "tokens of a scale"),
    (dict(dtype=torch.float8_e4m3fn, block=0), "tokens of a scale"), (dict(dtype=torch.float8_e4m3fn, head_dim=40), "head_dim"),
    (dict(dtype=torch.float8_e4m3fn, head_dim=192), "head_dim"), (dict(track_weights=True, head_dim=192), "head_dim"),
    (dict(track_weights=True, head_dim=20), "head_dim"),
])
def test_cache_classes_refuse(kw, text):
    from dtorch_amd.nn.kv_cache import KVCache
    a = dict(batch=1, kv_heads=2, max_len=40, head_dim=64, device="cpu")
    a.update(kw)
    with pytest.raises(ValueError, match=text):
        KVCache(**a)


def test_cache_classes_lay_out_codes():
    from dtorch_amd.nn.kv_cache import KVCache, PagedKVCache
    c = KVCache(2, 3, 70, 64, dtype=torch.float8_e4m3fn, device="cpu", block=32, track_weights=True)
    assert c.k.shape == (2, 3, 96, 64) and c.k_scale.shape == (2, 3, 3) and c.weights.shape == (2, 3, 96) and c.capacity == 96
    assert KVCache(1, 1, 70, 192, device="cpu").k_scale is None  # 16-bit caches as before
    with pytest.raises(ValueError, match="track_weights"):
        KVCache(1, 1, 70, 64, device="cpu").evict(16, 8)
    p = PagedKVCache(2, 3, 8, 16, 4, 64, dtype=torch.float8_e4m3fn, device="cpu", block=64)
    assert p.k_scale.shape == (8, 3, 1)
    with pytest.raises(ValueError, match="tokens of a scale"):
        PagedKVCache(2, 3, 8, 8, 4, 64, dtype=torch.float8_e4m3fn, device="cpu")


def test_oracle_scale_is_the_smallest_power_of_two():
    assert orc.block_scale(0.0) == 1.0 and orc.block_scale(448.0) == 1.0 and orc.block_scale(np.nextafter(448.0, 449.0)) == 2.0
    assert orc.block_scale(224.0) == 0.5 and orc.block_scale(1e-45) == 2.0 ** -126


def test_oracle_append_is_the_values_to_half_a_step():
    rng = np.random.default_rng(0)
    codes, scale = np.zeros((1, 2, 64, 16), np.uint8), np.ones((1, 2, 4), np.float32)
    x = rng.standard_normal((1, 2, 64, 16)) * np.exp2(rng.integers(-3, 4, (1, 2, 64, 1)))
    orc.append_fp8(codes, scale, None, [0], x, 16)
    s = np.repeat(scale, 16, 2)[..., None].astype(np.float64)
    # half a step of a normal code is 2^-4 of the value, of a subnormal one 2^-10 of the scale
    assert (np.abs(orc.values(codes, scale) - x) <= np.maximum(np.abs(x) * 2.0 ** -4, s * 2.0 ** -10)).all()


def test_oracle_evict_by_hand():
    w = np.array([[[3, 9, 1, 9, 0, 7, 2, 0]]], np.float32)
    x = np.arange(8.0).reshape(1, 1, 8, 1)
    n = np.array([7])
    kept = orc.evict([x], [], w, n, 4, 2, 1)
    # of tokens 0..4 the two heaviest are 1 and 3, then the last two of seven
    assert kept.tolist() == [[[1, 3, 5, 6]]] and n.tolist() == [4]
    assert x[0, 0, :, 0].tolist() == [1, 3, 5, 6, 4, 5, 6, 7] and w[0, 0].tolist() == [9, 9, 7, 2, 0, 0, 0, 0]
