"""Decode attention over a shared prefix and over listed key blocks, against fp64.

Tolerances are bounds, not fits.  With u the half step of the output type (2^-8 bf16, 2^-11 fp16, 2^-24 fp32), e = 2^-24,
A = softmax |V| and M = max sum_d |q_d k_d| scale: a score is an fp32 sum of D terms, off by at most (D + 8) e M, and its exponential
by twice that of itself (with the rounding of the exponent and of the instruction within the 8); P enters the second
product to 2^-16 (bf16: two numbers of 8 bits, rounded to nearest) or 2^-22 (fp16; one step of its subnormals, 2^-39 of the largest P, per
term besides); P V and the row sum are fp32 sums of n terms and a merge, (n + 64) e A each; O is rounded once, u |O| (in fp16 at
least half a subnormal step, 2^-25).  An LSE is off by the error of a score and of the row sum's logarithm."""
import math

import numpy as np
import pytest
import torch

from oracle import shared as orc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
PARTS = {torch.bfloat16: 2.0 ** -16, torch.float16: 2.0 ** -22, torch.float32: 0.0}


def _F():
    import dtorch_amd.nn.functional as F
    return F


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _np(t):
    return t.double().cpu().numpy()


def _close(o, lse, want, n, D, dtype, vmax):
    """One kv head's rows against (O, LSE, A, M)."""
    ro, rl, A, M = want
    if n == 0:
        assert (o == 0).all() and (lse == -np.inf).all()
        return
    ds = 2 * (D + 8) * E * M
    tol = U[dtype] * np.abs(ro) * 1.001 + (PARTS[dtype] + ds + 2 * (n + 64) * E) * A * 1.01
    if dtype == torch.float16:
        tol = tol + 2.0 ** -25 + n * 2.0 ** -39 * vmax
    assert (np.abs(o - ro) <= tol).all(), float((np.abs(o - ro) / tol).max())
    assert (np.abs(lse - rl) <= ds + (n + 64) * E + 2 ** -22 * np.abs(rl) + 2 ** -21).all()


def _tensors(rng, shape, dtype, layout="natural"):
    x = torch.from_numpy(rng.standard_normal(shape).astype(np.float32)).to(dtype).cuda()
    if layout == "tokens first":
        return x.transpose(1, 2).contiguous().transpose(1, 2)
    if layout == "wide rows":
        big = torch.full((*shape[:3], shape[3] + 32), float("nan"), dtype=dtype, device="cuda")
        big[..., :shape[3]] = x
        return big[..., :shape[3]]
    return x


def _shared(seed, B, G, Hq, Hkv, D, dtype, page, prefixes, owns, scale=None, layout="natural", spoil=False):
    """A call and its reference.  owns: tokens of each sequence behind its prefix (None: a sequence of length 0, paged)."""
    F = _F()
    rng = np.random.default_rng(seed)
    q = _tensors(rng, (B, Hq, 1, D), dtype)
    per = B // G
    top = max([o or 0 for o in owns] + [1])
    c = 1 / math.sqrt(D) if scale is None else scale
    if page:
        columns = max(prefixes) // page + -(-top // page) + 1
        P = B * columns + 3
        k, v = _tensors(rng, (P, Hkv, page, D), dtype, layout), _tensors(rng, (P, Hkv, page, D), dtype, layout)
        ids = rng.permutation(P)
        table = np.full((B, columns), -1, dtype=np.int32)
        at, lengths = 0, np.zeros(B, dtype=np.int32)
        for g in range(G):
            whole = prefixes[g] // page
            shared = ids[at:at + whole]
            at += whole
            for b in range(g * per, (g + 1) * per):
                if owns[b] is None:
                    table[b] = rng.choice([-1, P + 5, -9], columns)
                    continue
                lengths[b] = whole * page + owns[b]
                need = -(-owns[b] // page)
                table[b, :whole] = shared
                table[b, whole:whole + need] = ids[at:at + need]
                at += need
        if spoil:  # whatever no sequence holds must not count
            kn, vn = k.clone(), v.clone()
            kn.fill_(float("inf")), vn.fill_(float("nan"))
            for b in range(B):
                for s in range(-(-int(lengths[b]) // page)):
                    rows = min(page, int(lengths[b]) - s * page)
                    kn[table[b, s], :, :rows], vn[table[b, s], :, :rows] = k[table[b, s], :, :rows], v[table[b, s], :, :rows]
            k.copy_(kn), v.copy_(vn)
        o, lse = F.decode_attention_shared_paged(q, k, v, _i32(table), _i32(lengths), _i32(prefixes), scale=scale)
        rows = lambda x, b: orc.rows_of(x, table, b, np.arange(lengths[b]))  # noqa: E731
    else:
        Sp, So = max(max(prefixes), 1) + 5, top + 7
        kp, vp = _tensors(rng, (G, Hkv, Sp, D), dtype, layout), _tensors(rng, (G, Hkv, Sp, D), dtype, layout)
        k, v = _tensors(rng, (B, Hkv, So, D), dtype, layout), _tensors(rng, (B, Hkv, So, D), dtype, layout)
        if spoil:
            for g in range(G):
                kp[g, :, prefixes[g]:], vp[g, :, prefixes[g]:] = float("inf"), float("nan")
            for b in range(B):
                k[b, :, owns[b]:], v[b, :, owns[b]:] = float("nan"), float("inf")
        o, lse = F.decode_attention_shared(q, kp, vp, _i32(prefixes), k, v, _i32(owns), scale=scale)
        both = {id(x): (_np(a), _np(x)) for a, x in ((kp, k), (vp, v))}
        kk, vv = both[id(k)], both[id(v)]
        rows = lambda x, b: np.concatenate([x[0][b // per][:, :prefixes[b // per]], x[1][b][:, :owns[b]]], 1).swapaxes(0, 1)  # noqa: E731
    torch.cuda.synchronize()
    nk, nv = (_np(k), _np(v)) if page else (kk, vv)
    got_o, got_l, nq = _np(o), _np(lse), _np(q)
    vmax = 1.0
    for b in range(B):
        K, V = rows(nk, b), rows(nv, b)
        n = len(K)
        if n:
            vmax = float(np.abs(V).max())
        for h in range(Hkv):
            heads = slice(h * (Hq // Hkv), (h + 1) * (Hq // Hkv))
            want = orc.attend(nq[b, heads, 0], K[:, h] if n else np.zeros((0, D)), V[:, h] if n else np.zeros((0, D)), c)
            _close(got_o[b, heads, 0], got_l[b, heads], want, n, D, dtype, vmax)


TYPES = [torch.bfloat16, torch.float16, torch.float32]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,G,Hq,Hkv,D,page,prefixes,owns", [
    (1, 1, 1, 1, 64, 0, [1], [1]),
    (1, 1, 4, 1, 128, 16, [16], [1]),
    (2, 1, 4, 2, 128, 16, [160], [0, 33]),                      # one sequence has nothing of its own
    (3, 3, 2, 2, 64, 0, [0, 70, 5], [9, 0, 1]),                 # no prefix, and none behind it
    (4, 2, 8, 8, 128, 32, [64, 992], [1, 31, 32, 100]),
    (8, 1, 32, 8, 128, 16, [512], [5, 40, 100, 0, 1, 17, 64, 300]),
    (6, 2, 28, 4, 128, 256, [256, 1024], [3, 300, 5, 1, 257, 256]),
    (5, 1, 16, 2, 80, 16, [336], [9, 10, 11, 12, 13]),           # odd head dim
    (20, 1, 12, 12, 64, 0, [777], list(range(20))),
    (24, 2, 40, 2, 64, 0, [100, 3], [7] * 24),                  # 240 rows in a group, heads over 16 of a kv head
    (7, 7, 6, 3, 72, 64, [64, 0, 128, 640, 64, 0, 64], [1, 2, 3, 4, 5, 6, 70]),
])
def test_shared(dtype, B, G, Hq, Hkv, D, page, prefixes, owns):
    _shared(B + D, B, G, Hq, Hkv, D, dtype, page, prefixes, owns)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page,D", [(16, 128), (0, 64), (64, 96)])
@pytest.mark.parametrize("rows", [16, 17, 32, 33, 64, 65, 128, 129, 193])
def test_shared_row_counts(rows, page, D, dtype):
    """Rows of a group that meet the prefix together, on either side of where its form changes."""
    whole = max(page, 1)
    _shared(rows, rows, 1, 2, 2, D, dtype, page, [300 // whole * whole], [1 + b * 7 % 50 for b in range(rows)])


@pytest.mark.parametrize("page", [0, 16, 64])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2.0])
def test_shared_scales(page, scale):
    _shared(5, 6, 2, 8, 2, 64, torch.bfloat16, page, [128, 64], [3, 4, 50, 6, 1, 8], scale=scale)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("page", [0, 16, 32])
@pytest.mark.parametrize("layout", ["tokens first", "wide rows"])
def test_shared_layouts_and_what_lies_behind(dtype, page, layout):
    """Permuted caches, rows further apart, and infinities and NaN in every row that no sequence holds."""
    _shared(6, 6, 2, 12, 3, 64, dtype, page, [96, 32], [3, 40, 17, 0, 1, 33], layout=layout, spoil=True)


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_with_empty_sequences(dtype):
    """Sequences of length 0 among a group, whose table rows hold anything, and a group of them."""
    _shared(7, 9, 3, 8, 2, 128, dtype, 16, [160, 32, 48], [None, 5, 70, 1, None, 2, None, None, None])


@pytest.mark.parametrize("dtype", TYPES)
def test_shared_long(dtype):
    _shared(8, 4, 1, 8, 2, 128, dtype, 16, [20000], [1, 700, 33, 64])


def test_shared_prefix_lengths_beyond_the_sequences():
    """prefix_lengths that are no whole pages, negative, past the capacity or past a sequence: no more than all of a group hold is shared."""
    F = _F()
    rng = np.random.default_rng(9)
    page, D, Hq, Hkv, B = 16, 64, 4, 2, 6
    k, v = _tensors(rng, (40, Hkv, page, D), torch.bfloat16), _tensors(rng, (40, Hkv, page, D), torch.bfloat16)
    q = _tensors(rng, (B, Hq, 1, D), torch.bfloat16)
    table = np.tile(rng.permutation(40)[:8].astype(np.int32), (B, 1))  # all the same pages, of different lengths
    lengths = np.array([100, 20, 128, 128, 70, 15], dtype=np.int32)
    want = F.decode_attention_shared_paged(q, k, v, _i32(table), _i32(lengths), _i32([0, 0, 0]))
    nk, nv, nq = _np(k), _np(v), _np(q)
    for prefix in ([37, 60, 15], [-4, 2 ** 31 - 1, -2 ** 31], [1000, 128, 1000]):
        o, lse = F.decode_attention_shared_paged(q, k, v, _i32(table), _i32(lengths), _i32(prefix))
        for got in ((o, lse), want):
            go, gl = _np(got[0]), _np(got[1])
            for b in range(B):
                K, V = (orc.rows_of(x, table, b, np.arange(lengths[b])) for x in (nk, nv))
                for h in range(Hkv):
                    heads = slice(2 * h, 2 * h + 2)
                    _close(go[b, heads, 0], gl[b, heads], orc.attend(nq[b, heads, 0], K[:, h], V[:, h], D ** -0.5), int(lengths[b]), D, torch.bfloat16, 5.0)


def test_shared_page_ids_outside_the_pool():
    """Ids outside the pool are read as its first or last page: nothing faults, and other sequences are right."""
    F = _F()
    rng = np.random.default_rng(10)
    k, v = _tensors(rng, (6, 1, 16, 64), torch.float32), _tensors(rng, (6, 1, 16, 64), torch.float32)
    q = _tensors(rng, (4, 2, 1, 64), torch.float32)
    table = _i32([[0, 1], [0, -7], [0, 2 ** 31 - 1], [0, 6]])
    want = F.decode_attention_shared_paged(q, k, v, _i32([[0, 1], [0, 0], [0, 5], [0, 5]]), _i32([30, 31, 32, 20]), _i32([16]))
    got = F.decode_attention_shared_paged(q, k, v, table, _i32([30, 31, 32, 20]), _i32([16]))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_shared_infinities():
    """Scores of -inf drop out; a sequence of nothing else is 0 / 0, as softmax gives it; a NaN stays in its own sequence."""
    F = _F()
    D = 64
    k = torch.zeros(2, 1, 40, D, device="cuda")
    v = torch.randn(2, 1, 40, D, device="cuda")
    kp, vp = torch.zeros(1, 1, 32, D, device="cuda"), torch.randn(1, 1, 32, D, device="cuda")
    q = torch.ones(2, 1, 1, D, device="cuda")
    kp[..., 0] = -math.inf  # every prefix score is -inf
    k[0, 0, :5, 0] = -math.inf
    k[1, 0, :, 0] = -math.inf
    o, lse = F.decode_attention_shared(q, kp, vp, _i32([32]), k, v, _i32([40, 40]))
    torch.testing.assert_close(o[0, 0, 0], v[0, 0, 5:].mean(0), rtol=0, atol=40 * E * float(v.abs().max()) * 4)
    assert abs(float(lse[0, 0]) - math.log(35)) < 1e-6 and torch.isnan(o[1]).all()
    kp.zero_()
    k[0, 0, 3, 0] = math.nan
    o, lse = F.decode_attention_shared(q, kp, vp, _i32([32]), k, v, _i32([40, 40]))
    assert torch.isnan(o[0]).all() and torch.isfinite(o[1]).all() and abs(float(lse[1, 0]) - math.log(32)) < 1e-6


# ---- key bounds, selection and the attention over the selected blocks --------------------------------------

def _blocked(rng, B, Hkv, D, dtype, page, block, lengths, layout="natural", spoil=True):
    cap = -(-max(max(lengths), 1) // max(page, block)) * max(page, block)
    table = None
    if page:
        P = B * (cap // page) + 2
        table = rng.permutation(P)[:B * (cap // page)].reshape(B, -1).astype(np.int32)
        shape = (P, Hkv, page, D)
    else:
        shape = (B, Hkv, cap, D)
    k, v = _tensors(rng, shape, dtype, layout), _tensors(rng, shape, dtype, layout)
    if spoil:
        for b, n in enumerate(lengths):
            t = np.arange(max(n, 0), cap)
            if len(t) and table is None:
                k[b, :, n:], v[b, :, n:] = math.inf, math.nan
            elif len(t):
                slot, at = torch.from_numpy(table[b, t // page].astype(np.int64)).cuda(), torch.from_numpy(t % page).cuda()
                k[slot, :, at], v[slot, :, at] = math.nan, math.inf
    lo = torch.zeros(shape[0], Hkv, shape[2] // block, D, dtype=dtype, device="cuda")
    return k, v, lo, torch.zeros_like(lo), table


BLOCKS = [
    # B, Hq, Hkv, D, page, block, lengths, keep, recent
    (1, 1, 1, 64, 0, 16, [1], 16, 16),
    (2, 4, 2, 128, 0, 16, [16, 17], 16, 16),
    (3, 8, 2, 64, 16, 16, [0, 5, 400], 112, 32),
    (2, 32, 8, 128, 64, 32, [1000, 63], 256, 64),
    (2, 28, 4, 128, 256, 64, [3000, 1024], 640, 128),
    (4, 16, 2, 80, 0, 32, [500, 33, 512, 97], 96, 32),
    (3, 12, 12, 64, 128, 128, [2000, 128, 129], 384, 128),
    (2, 20, 1, 72, 32, 16, [700, 300], 160, 16),       # 20 heads of one kv head
    (1, 8, 8, 128, 0, 256, [5000], 1024, 256),
]


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("B,Hq,Hkv,D,page,block,lengths,keep,recent", BLOCKS)
@pytest.mark.parametrize("layout", ["natural", "tokens first", "wide rows"])
def test_bounds_select_and_attention(dtype, B, Hq, Hkv, D, page, block, lengths, keep, recent, layout):
    F = _F()
    rng = np.random.default_rng(D + block + len(lengths))
    k, v, lo, hi, table = _blocked(rng, B, Hkv, D, dtype, page, block, lengths, layout)
    q = _tensors(rng, (B, Hq, 1, D), dtype)
    dl = _i32(lengths)
    t = [] if table is None else [_i32(table)]
    sfx = "" if table is None else "_paged"
    nk, nv, nq, nl, nh = _np(k), _np(v), _np(q), _np(lo), _np(hi)
    for n_new in (1, 40, 10 ** 6):
        want = orc.bounds(nk, nl, nh, table, lengths, n_new, block)
        args = [k, lo, hi] + t + [dl]
        getattr(F, "kv_key_bounds" + sfx)(*args, n_new)
        nl, nh = _np(lo), _np(hi)
        assert np.array_equal(nl, want[0]) and np.array_equal(nh, want[1])
    for sign, scale in ((1.0, None), (-1.0, -0.5), (0.0, 0.0)):
        ids = getattr(F, "select_key_blocks" + sfx)(q, lo, hi, *t, dl, keep, recent, block, scale=scale)
        assert np.array_equal(ids.cpu().numpy(), orc.select(nq[:, :, 0], nl, nh, table, lengths, keep, recent, block, sign))
    ids = getattr(F, "select_key_blocks" + sfx)(q, lo, hi, *t, dl, keep, recent, block)
    ids[:, :, -1] = torch.where(ids[:, :, -1] % 2 == 1, 2 ** 30, ids[:, :, -1])  # an index past the sequence stands for nothing
    o, lse = getattr(F, "decode_attention_blocks" + sfx)(q, k, v, *t, dl, ids, block)
    _check_blocks(o, lse, nq, nk, nv, table, lengths, ids.cpu().numpy(), block, D, dtype)


def _check_blocks(o, lse, nq, nk, nv, table, lengths, ids, block, D, dtype):
    go, gl = _np(o), _np(lse)
    group = nq.shape[1] // ids.shape[1]
    for b in range(ids.shape[0]):
        for h in range(ids.shape[1]):
            tokens = np.concatenate([np.arange(j * block, min((j + 1) * block, lengths[b])) for j in ids[b, h].tolist() if 0 <= j * block < lengths[b]] + [np.zeros(0, int)]).astype(int)
            K, V = (orc.rows_of(x, table, b, tokens)[:, h] for x in (nk, nv)) if len(tokens) else (np.zeros((0, D)),) * 2
            heads = slice(h * group, (h + 1) * group)
            _close(go[b, heads, 0], gl[b, heads], orc.attend(nq[b, heads, 0], K, V, D ** -0.5), len(tokens), D, dtype, 6.0)


@pytest.mark.parametrize("page", [0, 16, 64])
def test_listed_blocks(page):
    """Lists as a caller may make them: any order, a block twice, none at all, strided, more of them than a share holds."""
    F = _F()
    rng = np.random.default_rng(page)
    B, Hq, Hkv, D, block, lengths = 3, 8, 2, 64, 16, [5000, 0, 77]
    k, v, _, _, table = _blocked(rng, B, Hkv, D, torch.bfloat16, page, block, lengths)
    q = _tensors(rng, (B, Hq, 1, D), torch.bfloat16)
    ids = rng.integers(-3, 320, (B, Hkv, 300)).astype(np.int32)
    ids[0, 1] = -1  # a kv head without a block
    ids[2, 0, :7], ids[2, 1, :3] = 4, [0, 0, 4]
    wide = torch.zeros(B, 2 * Hkv, 310, dtype=torch.int32, device="cuda")
    wide[:, ::2, :300] = _i32(ids)
    args = [_i32(table)] if page else []
    o, lse = getattr(F, "decode_attention_blocks" + ("_paged" if page else ""))(q, k, v, *args, _i32(lengths), wide[:, ::2, :300], block)
    _check_blocks(o, lse, _np(q), _np(k), _np(v), table, lengths, ids, block, D, torch.bfloat16)


def test_blocks_of_infinite_scores():
    """All scores -inf: 0 / 0 as softmax gives it, not the 0 of a list without tokens; in one share and in several."""
    F = _F()
    for n in (16, 8192):
        k = torch.full((1, 1, n, 64), 0.0, device="cuda")
        k[..., 0] = -math.inf
        ids = torch.arange(n // 16, dtype=torch.int32, device="cuda").view(1, 1, -1)
        o, lse = F.decode_attention_blocks(torch.ones(1, 1, 1, 64, device="cuda"), k, torch.ones_like(k), _i32([n]), ids, 16)
        assert torch.isnan(o).all()
        o, lse = F.decode_attention_blocks(torch.ones(1, 1, 1, 64, device="cuda"), k, torch.ones_like(k), _i32([0]), ids, 16)
        assert (o == 0).all() and (lse == -math.inf).all()


@pytest.mark.parametrize("blocks", [100, 4096, 4097, 20000])
def test_select_many_blocks_and_ties(blocks):
    """Scores that are often equal (the first ones win), NaN and infinite bounds, and counts around what LDS holds."""
    F = _F()
    rng = np.random.default_rng(blocks)
    D, block = 16, 16
    lo = rng.integers(-3, 1, (1, 2, blocks, D)).astype(np.float32)
    hi = lo + rng.integers(0, 3, lo.shape)
    hi[0, 0, ::7, 3], lo[0, 1, 5::11, 2], hi[0, 1, 3::50, 1] = np.nan, -np.inf, np.inf
    q = np.zeros((1, 4, D))
    q[..., :4] = rng.integers(-2, 3, (1, 4, 4))
    dt = torch.float32
    dq, dlo, dhi = (torch.from_numpy(x.astype(np.float32)).to(dt).cuda() for x in (q[:, :, None], lo, hi))
    lengths = [blocks * block - 3]
    for keep, recent in ((16, 16), (block * (blocks // 2), block * 3), (block * (blocks - 1), block)):
        got = F.select_key_blocks(dq, dlo, dhi, _i32(lengths), keep, recent, block)
        assert np.array_equal(got.cpu().numpy(), orc.select(q, lo.astype(float), hi.astype(float), None, lengths, keep, recent, block))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_bounds_hold(dtype):
    """No token of a block scores above the block's bound."""
    F = _F()
    rng = np.random.default_rng(4)
    k, v, lo, hi, _ = _blocked(rng, 1, 1, 64, dtype, 0, 16, [512])
    F.kv_key_bounds(k, lo, hi, _i32([512]), 512)
    q = rng.standard_normal((50, 64))
    s = q @ _np(k)[0, 0].T
    top = q.clip(min=0) @ _np(hi)[0, 0].T + q.clip(max=0) @ _np(lo)[0, 0].T
    assert (s.reshape(50, -1, 16).max(2) <= top + 1e-9).all()


def test_bounds_of_nan_keys_and_bad_pages():
    F = _F()
    k = torch.randn(3, 1, 16, 8, device="cuda")
    k[0, 0, :, 0], k[1, 0, 3, 1] = math.nan, math.nan
    lo, hi = torch.zeros(3, 1, 1, 8, device="cuda"), torch.zeros(3, 1, 1, 8, device="cuda")
    F.kv_key_bounds_paged(k, lo, hi, _i32([[0, 1, -1], [5, -2, 2]]), _i32([48, 48]), 48)
    assert lo[0, 0, 0, 0] == math.inf and hi[0, 0, 0, 0] == -math.inf
    for x, y in ((lo, np.nanmin), (hi, np.nanmax)):
        assert np.array_equal(x[1:, 0, 0].cpu().numpy(), y(k[1:, 0].cpu().numpy(), 1))
    F.kv_key_bounds_paged(k, lo, hi, _i32([[0, 1, -1]]), _i32([48]), 0)


def test_capture_and_streams():
    """The chain in a graph, replayed with other inputs; two graphs with workspaces of their own; a call on another stream."""
    F = _F()
    rng = np.random.default_rng(11)
    B, Hq, Hkv, D, block, lengths = 2, 8, 2, 64, 32, [900, 333]
    k, v, lo, hi, _ = _blocked(rng, B, Hkv, D, torch.bfloat16, 0, block, lengths, spoil=False)
    q = _tensors(rng, (B, Hq, 1, D), torch.bfloat16)
    dl, pl = _i32(lengths), _i32([500, 100])
    kp, vp = _tensors(rng, (2, Hkv, 512, D), torch.bfloat16), _tensors(rng, (2, Hkv, 512, D), torch.bfloat16)

    def chain():
        F.kv_key_bounds(k, lo, hi, dl, 1000)
        ids = F.select_key_blocks(q, lo, hi, dl, 256, 64, block)
        return F.decode_attention_blocks(q, k, v, dl, ids, block) + (ids,)

    def shared():
        return F.decode_attention_shared(q, kp, vp, pl, k, v, dl)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        chain(), shared()
    torch.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for f in (chain, shared):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(f())
        graphs.append(g)
    for i in range(4):
        for x in (q, k, v, kp, vp):
            x.normal_()
        dl.copy_(_i32(rng.integers(1, 960, 2)))
        pl.copy_(_i32(rng.integers(0, 512, 2)))
        want = [f() for f in (chain, shared)]
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b)), i
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = [f() for f in (chain, shared)]
        side.synchronize()
        for a, b in zip(other, want):
            assert all(torch.equal(x, y) for x, y in zip(a, b))


def test_host_refusals():
    F = _F()
    z = lambda *s, dt=torch.bfloat16: torch.zeros(*s, dtype=dt, device="cuda")  # noqa: E731
    q, k, kp, l, pl = z(2, 4, 1, 64), z(2, 2, 32, 64), z(1, 2, 32, 64), _i32([3, 4]), _i32([5])
    for bad in (dict(q=z(2, 4, 2, 64)), dict(q=z(2, 3, 1, 64)), dict(q=z(2, 4, 1, 32)), dict(q=q.float()), dict(k=z(3, 2, 32, 64)),
                dict(k=z(2, 2, 32, 64, dt=torch.float16)), dict(kp=z(2, 2, 32, 64)), dict(kp=z(1, 4, 32, 64)), dict(l=l.long()), dict(l=_i32([1])),
                dict(pl=_i32([1, 2, 3])), dict(pl=pl.long()), dict(pl=pl.cpu()), dict(q=z(2, 4, 1, 12), k=z(2, 2, 32, 12), kp=z(1, 2, 32, 12)),
                dict(q=z(2, 4, 1, 256), k=z(2, 2, 32, 256), kp=z(1, 2, 32, 256)), dict(scale=math.inf)):
        a = dict(dict(q=q, k=k, kp=kp, l=l, pl=pl, scale=None), **bad)
        with pytest.raises(ValueError):
            F.decode_attention_shared(a["q"], a["kp"], a["kp"], a["pl"], a["k"], a["k"], a["l"], scale=a["scale"])
    pool, t = z(6, 2, 16, 64), _i32([[0, 1], [0, 2]])
    for bad in (dict(t=t.long()), dict(t=_i32([[0, 1]])), dict(pool=z(6, 2, 24, 64)), dict(pool=z(6, 2, 8, 64)), dict(pl=_i32([]))):
        a = dict(dict(t=t, pool=pool, pl=pl), **bad)
        with pytest.raises(ValueError):
            F.decode_attention_shared_paged(q, a["pool"], a["pool"], a["t"], l, a["pl"])
    lo = z(2, 2, 2, 64)
    for args in ((k, lo, lo), (k, lo, z(2, 2, 2, 64, dt=torch.float16)), (k, z(2, 2, 3, 64), z(2, 2, 3, 64)), (k, z(2, 2, 32, 64), z(2, 2, 32, 64)),
                 (k, lo, z(1, 2, 2, 64).expand(2, 2, 2, 64))):
        with pytest.raises(ValueError):
            F.kv_key_bounds(*args, l, 1)
    with pytest.raises(ValueError):
        F.kv_key_bounds(k, lo, z(2, 2, 2, 64), l, -1)
    hi = z(2, 2, 2, 64)
    for keep, recent, block in ((0, 16, 16), (24, 16, 16), (32, 8, 16), (16, 32, 16), (32, 16, 0), (32, 16, 24), (32, 16, 512)):
        with pytest.raises(ValueError):
            F.select_key_blocks(q, lo, hi, l, keep, recent, block)
    ids = torch.zeros(2, 2, 2, dtype=torch.int32, device="cuda")
    for bad, block in ((ids.long(), 16), (ids[:1], 16), (ids[:, :, :0], 16), (ids, 8), (ids, 24), (ids, 512)):
        with pytest.raises(ValueError):
            F.decode_attention_blocks(q, k, k, l, bad, block)
    with pytest.raises(ValueError):  # blocks larger than a page
        F.decode_attention_blocks_paged(q, pool, pool, t, l, ids, 32)
    e = F.decode_attention_shared(q[:0], kp, kp, pl, k[:0], k[:0], l[:0])
    assert e[0].shape == (0, 4, 1, 64)


def test_offsets_past_32_bits():
    """Pages past 2^31 elements of a pool (and past 2^32 bytes): the same outputs as from a small pool, bit by bit."""
    F = _F()
    P, H, page, D, B = 140000, 8, 16, 128, 3
    if torch.cuda.mem_get_info()[0] < 16 * 2 ** 30:
        pytest.skip("needs 16 GiB of device memory")
    rng = np.random.default_rng(21)
    ids = np.array([P - 1, 5, P - 2, 131073, 90000, P - 7, 65537, 1])
    small = [_tensors(rng, (8, H, page, D), torch.bfloat16) for _ in range(2)]
    k, v = (torch.empty(P, H, page, D, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    at = torch.from_numpy(ids).cuda()
    k[at], v[at] = small
    table = np.array([[0, 1, 2, 3], [0, 1, 4, 5], [0, 1, 6, 7]])
    q, lengths, prefix = _tensors(rng, (B, 32, 1, D), torch.bfloat16), _i32([64, 50, 33]), _i32([32])
    bounds = [[torch.empty(x.shape[0], H, 1, D, dtype=torch.bfloat16, device="cuda") for _ in range(2)] for x in (small[0], k)]
    outs = []
    for (kk, vv), (lo, hi), t in ((small, bounds[0], table), ((k, v), bounds[1], ids[table])):
        t = _i32(t)
        F.kv_key_bounds_paged(kk, lo, hi, t, lengths, 64)
        kept = F.select_key_blocks_paged(q, lo, hi, t, lengths, 32, 16, 16)
        outs.append([kept, *F.decode_attention_shared_paged(q, kk, vv, t, lengths, prefix), *F.decode_attention_blocks_paged(q, kk, vv, t, lengths, kept, 16)])
    assert all(torch.equal(a, b) for a, b in zip(*outs))
    # and the pages move
    refs, t = torch.zeros(P, dtype=torch.int32, device="cuda"), _i32(ids[table])
    refs[at] = _i32([3, 3, 1, 1, 1, 1, 1, 1])
    assert F.kv_pages_compact([k, v], t, refs).item() == 8 and t.max().item() == 7
    again = F.decode_attention_shared_paged(q, k, v, t, lengths, prefix)
    assert all(torch.equal(a, b) for a, b in zip(outs[0][1:3], again))
