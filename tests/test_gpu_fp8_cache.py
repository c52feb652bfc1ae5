"""The 8-bit KV cache: quantised append (bit for bit) and decode attention over codes, against fp64.

Tolerances are bounds, not fits.  With u the half step of the output type (2^-8 bf16, 2^-11 fp16), e = 2^-24 and
A = softmax |V|: P is rounded to 16 bits (u A), O is rounded (u |O|), an fp32 sum of n terms is off by at most n e times the
sum of their magnitudes, which is (D + 8) e M per score, M = max sum_d |q_d k_d| scale, and (n + 64) e A for P V and the row sum
together with the exponentials' own rounding.  fp32 queries: no 16-bit rounding, sums of three times as many terms.  In fp16 the
half step of a subnormal is 2^-25 whatever the value: for O it is added as it is; for P, whose largest value per 32 tokens the
kernel puts at 2^15, it is 2^-40 of that largest value, or at most n 2^-40 max |V| over all tokens."""
import numpy as np
import pytest
import torch

from oracle import cache as orc
from oracle.sdpa import e4m3fn_decode

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}


def _F():
    import dtorch_amd.nn.functional as F
    return F


def _codes(t):
    return t.view(torch.uint8).cpu().numpy()


def _dev8(x):
    return torch.from_numpy(x.copy()).cuda().view(torch.float8_e4m3fn)


def _same_codes(a, b):
    """Equal bytes, NaN codes of either sign alike."""
    nan = (a & 0x7F) == 0x7F
    return np.array_equal(nan, (b & 0x7F) == 0x7F) and np.array_equal(a[~nan], b[~nan])


def _pool(rng, slots, H, rows, D, block):
    """Any bytes as codes, and powers of two as scales."""
    k = rng.integers(0, 256, (slots, H, rows, D)).astype(np.uint8)
    s = np.exp2(rng.integers(-9, 3, (slots, H, rows // block))).astype(np.float32)
    return k, s


def _append(rng, lengths, H, D, cap, block, page, n, dtype, spoil=None, table=None, scales=None):
    B = len(lengths)
    if page and table is None:
        table = rng.permutation(B * (cap // page) + 2)[:B * (cap // page)].reshape(B, -1).astype(np.int32)
    slots, rows = (B * (cap // page) + 2, page) if page else (B, cap)
    k, ks = _pool(rng, slots, H, rows, D, block)
    v, vs = _pool(rng, slots, H, rows, D, block)
    if scales is not None:
        ks[:], vs[:] = scales(ks), scales(vs)
    new = [torch.from_numpy(rng.standard_normal((B, n, H, D)).astype(np.float32) * np.exp2(rng.integers(-8, 9, (1, n, H, 1))).astype(np.float32)).to(dtype)
           for _ in range(2)]
    if spoil is not None:
        for x in new:
            spoil(x)
    kn, vn = (x.cuda().transpose(1, 2) for x in new)  # the projection's natural layout
    dk, dv, dks, dvs = _dev8(k), _dev8(v), torch.from_numpy(ks.copy()).cuda(), torch.from_numpy(vs.copy()).cuda()
    dl = torch.tensor(lengths, dtype=torch.int32, device="cuda")
    for c, s, x in ((k, ks, kn), (v, vs, vn)):
        orc.append_fp8(c, s, table, lengths, x.double().cpu().numpy(), block)
    if page:
        _F().kv_cache_append_fp8_paged(dk, dv, dks, dvs, torch.from_numpy(table).cuda(), dl, kn, vn)
    else:
        _F().kv_cache_append_fp8(dk, dv, dks, dvs, dl, kn, vn)
    torch.cuda.synchronize()
    assert _same_codes(_codes(dk), k) and _same_codes(_codes(dv), v)
    assert np.array_equal(dks.cpu().numpy(), ks, equal_nan=True) and np.array_equal(dvs.cpu().numpy(), vs, equal_nan=True)
    assert dl.tolist() == [min(max(x, 0) + n, cap) for x in lengths]


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("n,block,page,D", [(1, 32, 0, 128), (1, 16, 16, 64), (3, 64, 0, 80), (16, 16, 64, 128), (17, 32, 32, 16), (70, 16, 0, 128),
                                            (200, 64, 128, 96), (300, 256, 0, 128), (300, 128, 256, 128)])
def test_append(dtype, n, block, page, D):
    rng = np.random.default_rng(1000 * n + D)
    cap = 512
    # empty, inside a block, at a block's end, running past the capacity, full, negative (counts as empty)
    _append(rng, [0, 5, block - 1, block, cap - 1, cap, -3], 3, D, cap, block, page, n, dtype)


def test_append_of_no_tokens():
    rng = np.random.default_rng(7)
    _append(rng, [0, 9, 64, -1], 2, 64, 64, 16, 0, 0, torch.bfloat16)


def test_append_many_heads():
    rng = np.random.default_rng(8)
    _append(rng, [0, 40], 70, 16, 64, 16, 0, 2, torch.float16)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append_extreme_values(dtype):
    # zeros, NaN, infinities, the type's largest and smallest values, and rows of 448 and a little more times powers of two
    rng = np.random.default_rng(9)
    info = torch.finfo(dtype)

    def spoil(x):  # [B, n, H, D]
        x[0, 0] = 0
        x[0, 1, 0, 3] = float("nan")
        x[0, 2, 1, 5] = float("inf")
        x[0, 3, 1, 6] = float("-inf")
        x[1, 0, 0, 0] = info.max
        x[1, 1, 1, :] = info.tiny
        x[2] = 0
        x[2, :, 0] = info.smallest_normal / 2  # subnormal
        x[3, :, 0] = 448.0
        x[3, :, 1] = 464.0 if dtype != torch.bfloat16 else 450.0
        x[4] = float("nan")

    for n in (1, 4, 20):
        _append(rng, [0, 3, 0, 16, 2], 2, 64, 64, 16, 0, n, dtype, spoil if n > 3 else None)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_append_behind_scales_of_any_value(dtype):
    # scales of the caller's own: kept where they hold the new values (the product with their reciprocal, rounded once to fp32, is
    # what is encoded), replaced where they do not; 0 and NaN count as none
    def scales(s):
        s = np.where(np.arange(s.size).reshape(s.shape) % 2, np.float32(4.0), s * np.float32(2.0 ** -12))
        s[0, 0], s[1, 0] = 0.0, np.nan
        return s

    rng = np.random.default_rng(12)
    for n in (1, 9):
        _append(rng, [3, 17, 40, 63], 2, 64, 128, 16, 0, n, dtype, scales=scales)


def test_append_token_by_token_is_append_at_once():
    # powers of two re-encode without rounding (subnormal codes apart: every value here is within 2^9 of its block's largest)
    rng = np.random.default_rng(10)
    B, H, D, cap, block = 2, 2, 64, 96, 32
    x = torch.from_numpy((rng.standard_normal((B, H, 70, D)) * np.exp2(rng.integers(-2, 3, (1, 1, 70, 1)))).astype(np.float32)).to(torch.bfloat16).cuda()
    x = torch.where(x.abs() < 2.0 ** -3, torch.full_like(x, 0.25), x)
    outs = []
    for sizes in ([70], [1] * 70, [33, 1, 36]):
        k = torch.zeros(B, H, cap, D, dtype=torch.float8_e4m3fn, device="cuda")
        v, ks = torch.zeros_like(k), torch.zeros(B, H, cap // block, device="cuda")
        vs, ln, at = torch.zeros_like(ks), torch.zeros(B, dtype=torch.int32, device="cuda"), 0
        for n in sizes:
            _F().kv_cache_append_fp8(k, v, ks, vs, ln, x[:, :, at:at + n], x[:, :, at:at + n])
            at += n
        torch.cuda.synchronize()
        outs.append((_codes(k), ks.cpu().numpy(), ln.tolist()))
    for o in outs[1:]:
        assert np.array_equal(o[0], outs[0][0]) and np.array_equal(o[1], outs[0][1]) and o[2] == outs[0][2]


def test_append_drops_tokens_without_a_page():
    rng = np.random.default_rng(11)
    table = np.array([[0, 5, 2, 3], [4, -1, 6, 99]], dtype=np.int32)
    for n, start in ((1, [16, 16]), (40, [0, 10]), (20, [60, 40])):
        _append(rng, start, 2, 64, 64, 16, 16, n, torch.bfloat16, table=table)


# ---- decode -------------------------------------------------------------------------------------------------

def _decode_case(rng, lengths, Hq, Hkv, D, block, page, dtype, cap, scales=None, junk=True):
    B = len(lengths)
    table = None
    if page:
        per = cap // page
        table = rng.permutation(B * per + 3)[:B * per].reshape(B, per).astype(np.int32)
    slots, rows = (B * (cap // page) + 3, page) if page else (B, cap)
    out = {"table": table, "block": block}
    for name in "kv":
        c = rng.integers(0, 256, (slots, Hkv, rows, D)).astype(np.uint8)
        c = np.where((c & 0x7F) == 0x7F, np.uint8(0x18), c)  # finite ones
        mag = (c >> 3) & 0xF
        c = np.where(mag > 9, (c & 0x87) | (9 << 3), c).astype(np.uint8)  # up to 7.5
        s = (0.5 + rng.random((slots, Hkv, rows // block))).astype(np.float32) if scales is None else scales(rng, (slots, Hkv, rows // block))
        if junk:  # NaN codes and scales where no token lies
            used = np.zeros((slots, rows), dtype=bool)
            for b in range(B):
                t = np.arange(min(max(lengths[b], 0), cap))
                used[(table[b, t // page], t % page) if page else (b, t)] = True
            c = np.where(used[:, None, :, None], c, np.uint8(0x7F))
            s = np.where(used.reshape(slots, 1, -1, block).any(-1), s, np.float32("nan"))
        out[name], out[name + "s"] = c, s
    if page:  # entries past a sequence's last page name no page
        for b in range(B):
            table[b, -(-min(max(lengths[b], 0), cap) // page):] = -1
    out["q"] = torch.from_numpy(rng.standard_normal((B, Hq, 1, D)).astype(np.float32)).to(dtype)
    out["lengths"] = lengths
    return out


def _run_decode(c, scale=None, layout=None, stream=None):
    q = c["q"].cuda()
    k, v, ks, vs = _dev8(c["k"]), _dev8(c["v"]), torch.from_numpy(c["ks"]).cuda(), torch.from_numpy(c["vs"]).cuda()
    if layout is not None:
        k, v = layout(k), layout(v)
    ln = torch.tensor(c["lengths"], dtype=torch.int32, device="cuda")
    if c["table"] is not None:
        o, l = _F().decode_attention_fp8_paged(q, k, v, ks, vs, torch.from_numpy(c["table"]).cuda(), ln, scale=scale)
    else:
        o, l = _F().decode_attention_fp8(q, k, v, ks, vs, ln, scale=scale)
    torch.cuda.synchronize()
    return o, l


def _tolerances(c, o, a, mag, ln):
    dtype, D = c["q"].dtype, c["q"].shape[-1]
    n = np.maximum(np.asarray(c["lengths"], dtype=np.float64), 1)[:, None]
    terms = 3 if dtype == torch.float32 else 1
    ds = (terms * D + 8) * E * mag  # of a score, and so relative to its exponential
    rel = 2 * ds + (terms * n + 64) * E
    u = U[dtype]
    to = a * (rel + (u if terms == 1 else 0))[..., None] + np.abs(o) * u + np.finfo(np.float32).tiny
    if dtype == torch.float16:
        to = to + 2.0 ** -25 + (n * 2.0 ** -40)[..., None] * np.nanmax(np.abs(orc.values(c["v"], c["vs"])), initial=0)
    return to, ds + (n + 64) * E + 8 * E * np.abs(np.where(np.isfinite(ln), ln, 0))


def _check(c, o, l, scale=None):
    eo, el, a, mag = orc.decode_fp8(c["q"].double().numpy()[:, :, 0], c["k"], c["v"], c["ks"], c["vs"], c["lengths"], c["table"], scale)
    to, tl = _tolerances(c, eo, a, mag, el)
    go, gl = o.double().cpu().numpy()[:, :, 0], l.double().cpu().numpy()
    assert o.dtype == c["q"].dtype and l.dtype == torch.float32
    assert np.array_equal(np.isnan(go), np.isnan(eo))
    fin = np.isfinite(eo)
    assert np.all(np.abs(go - eo)[fin] <= to[fin]), float(np.max((np.abs(go - eo) / to)[fin]))
    assert np.array_equal(np.isneginf(gl), np.isneginf(el))
    fin = np.isfinite(el)
    assert np.all(np.abs(gl[fin] - el[fin]) <= tl[fin]), float(np.max(np.abs(gl[fin] - el[fin]) / tl[fin]))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("Hq,Hkv,D,block,page", [(32, 8, 128, 32, 0), (8, 8, 64, 16, 16), (7, 1, 128, 16, 64), (40, 2, 80, 64, 0), (64, 1, 16, 256, 256),
                                                 (6, 2, 128, 32, 32), (16, 1, 112, 128, 0)])
def test_decode(dtype, Hq, Hkv, D, block, page):
    rng = np.random.default_rng(Hq * 1000 + D)
    lengths = [0, 1, 15, 16, 17, 31, 32, 33, 200, 511, 512, -4, 600]  # past the capacity: clamped
    c = _decode_case(rng, lengths, Hq, Hkv, D, block, page, dtype, 512)
    _check(c, *_run_decode(c))


@pytest.mark.parametrize("page", [0, 16])
def test_decode_more_sequences_than_lanes(page):
    rng = np.random.default_rng(5 + page)
    lengths = [int(x) for x in rng.integers(0, 130, 150)]
    c = _decode_case(rng, lengths, 4, 2, 64, 16, page, torch.bfloat16, 160)
    _check(c, *_run_decode(c))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("B,n,Hq,Hkv", [(1, 9001, 8, 2), (3, 5000, 20, 20), (1, 31, 1, 1), (2, 40000, 4, 1)])
def test_decode_long(dtype, B, n, Hq, Hkv):
    rng = np.random.default_rng(n)
    cap = -(-n // 64) * 64
    c = _decode_case(rng, [n - 7 * b for b in range(B)], Hq, Hkv, 128, 64, 0, dtype, cap)
    _check(c, *_run_decode(c))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.7])
def test_decode_scale(scale):
    rng = np.random.default_rng(3)
    c = _decode_case(rng, [5, 100, 64], 8, 2, 128, 16, 0, torch.float16, 128)
    _check(c, *_run_decode(c, scale=scale), scale=scale)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_decode_scales_of_any_size(dtype):
    # V blocks 2^-40 to 2^10 apart: what the small ones add is lost in rounding, and the row sum still counts their tokens
    rng = np.random.default_rng(13)
    c = _decode_case(rng, [500, 33, 17, 1], 8, 4, 128, 16, 0, dtype, 512)
    c["vs"] = np.exp2(rng.integers(-40, 10, c["vs"].shape)).astype(np.float32)
    c["vs"][:, 0] = np.float32(2.0 ** -100)
    c["vs"][0, 1, 3:9] = 0.0
    c["ks"] = (c["ks"] * np.exp2(rng.integers(-20, 1, c["ks"].shape))).astype(np.float32)
    c["q"] = c["q"] * 4
    if dtype == torch.float16:  # outputs within fp16's range, and steps of its subnormals
        c["vs"] = np.minimum(c["vs"], np.float32(16.0))
    eo, el, a, mag = orc.decode_fp8(c["q"].double().numpy()[:, :, 0], c["k"], c["v"], c["ks"], c["vs"], c["lengths"])
    to, tl = _tolerances(c, eo, a, mag, el)
    o, l = _run_decode(c)
    assert np.all(np.abs(o.double().cpu().numpy()[:, :, 0] - eo) <= to)
    assert np.all(np.abs(l.double().cpu().numpy() - el) <= tl)


def test_decode_nan_stays_in_its_head():
    rng = np.random.default_rng(14)
    c = _decode_case(rng, [100, 200, 300], 8, 4, 64, 16, 0, torch.bfloat16, 304)
    c["k"][1, 2, 37, 5] = 0x7F
    c["v"][2, 0, 299, 9] = 0xFF
    o, l = _run_decode(c)
    on, ln = torch.isnan(o)[:, :, 0], torch.isnan(l)
    assert on[1, 4:6].all() and ln[1, 4:6].all() and on[2, :2, 9].all()
    on[1, 4:6], ln[1, 4:6], on[2, :2, 9] = False, False, False
    assert not on.any() and not ln.any()


def test_decode_layouts():
    rng = np.random.default_rng(15)
    c = _decode_case(rng, [77, 130, 144], 8, 2, 128, 16, 0, torch.bfloat16, 144)
    want = _run_decode(c)
    for layout in (lambda x: x.view(torch.uint8).transpose(1, 2).contiguous().transpose(1, 2).view(torch.float8_e4m3fn),  # [B, S, H, D]
                   lambda x: torch.cat([x.view(torch.uint8)] * 2, 3)[..., 128:].view(torch.float8_e4m3fn)):  # rows of a wider tensor
        got = _run_decode(c, layout=layout)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize("page", [16, 64])
def test_decode_of_shared_and_of_bad_pages(page):
    """A prefix that two sequences share, a page twice in one sequence, and page ids outside the pool, which count as its ends."""
    rng = np.random.default_rng(page)
    c = _decode_case(rng, [300, 290, 256, 200], 8, 2, 128, 16, page, torch.bfloat16, 320, junk=False)
    t = c["table"]
    t[1, :2] = t[0, :2]
    t[2, 3] = t[2, 0]
    t[3, 0], t[3, 1] = -5, 1 << 30
    _check(c, *_run_decode(c))


def test_decode_of_a_longer_cache_view():
    # the same tokens in a larger cache: other shares, the same values within their rounding; and a view of its first blocks
    rng = np.random.default_rng(16)
    c = _decode_case(rng, [60, 96], 8, 2, 128, 16, 0, torch.bfloat16, 1024)
    _check(c, *_run_decode(c))
    q, ln = c["q"].cuda(), torch.tensor(c["lengths"], dtype=torch.int32, device="cuda")
    k, v, ks, vs = _dev8(c["k"]), _dev8(c["v"]), torch.from_numpy(c["ks"]).cuda(), torch.from_numpy(c["vs"]).cuda()
    o, l = _F().decode_attention_fp8(q, k[:, :, :96], v[:, :, :96], ks[:, :, :6], vs[:, :, :6], ln)
    _check(c, o, l)


@pytest.mark.parametrize("page", [0, 128])
def test_decode_past_four_gigabytes(page):
    """K and V whose last rows lie past 2^32 bytes."""
    rng = np.random.default_rng(17)
    Hkv, D, block, n = 8, 128, 32, 300
    c = _decode_case(rng, [n], 16, Hkv, D, block, page, torch.bfloat16, 384, junk=False)
    ln, q = torch.tensor([n], dtype=torch.int32, device="cuda"), c["q"].cuda()
    if page:
        pages = 34000  # of 128 KB
        big = [torch.empty(pages, Hkv, page, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
        scales = [torch.ones(pages, Hkv, page // block, device="cuda") for _ in range(2)]
        ids = torch.tensor([pages - 1, 3, pages - 2])
        for x, s, name in zip(big, scales, "kv"):
            x[ids.cuda()] = torch.from_numpy(c[name][c["table"][0, :3]]).cuda()
            s[ids.cuda()] = torch.from_numpy(c[name + "s"][c["table"][0, :3]]).cuda()
        o, l = _F().decode_attention_fp8_paged(q, big[0].view(torch.float8_e4m3fn), big[1].view(torch.float8_e4m3fn), *scales,
                                               ids[None].to(torch.int32).cuda(), ln)
    else:
        wide = 1 << 24  # bytes between tokens
        big = [torch.empty(n, wide, dtype=torch.uint8, device="cuda") for _ in range(2)]
        views = []
        for x, name in zip(big, "kv"):
            x[:, -Hkv * D:] = torch.from_numpy(c[name][0, :, :n]).cuda().transpose(0, 1).reshape(n, -1)
            views.append(x[:, -Hkv * D:].view(n, Hkv, D).transpose(0, 1)[None].view(torch.float8_e4m3fn)[:, :, :288])
        c["lengths"] = [288]
        ln.fill_(288)
        o, l = _F().decode_attention_fp8(q, *views, torch.from_numpy(c["ks"][:, :, :9]).cuda(), torch.from_numpy(c["vs"][:, :, :9]).cuda(), ln)
    torch.cuda.synchronize()
    _check(c, o, l)


def test_append_past_four_gigabytes():
    rng = np.random.default_rng(18)
    Hkv, D, block, page, pages = 8, 128, 32, 128, 34000
    big = [torch.zeros(pages, Hkv, page, D, dtype=torch.uint8, device="cuda") for _ in range(2)]
    scales = [torch.zeros(pages, Hkv, page // block, device="cuda") for _ in range(2)]
    new = torch.from_numpy(rng.standard_normal((1, Hkv, 150, D)).astype(np.float32)).cuda()
    table = torch.tensor([[pages - 1, pages - 3]], dtype=torch.int32, device="cuda")
    _F().kv_cache_append_fp8_paged(big[0].view(torch.float8_e4m3fn), big[1].view(torch.float8_e4m3fn), *scales, table,
                                   torch.zeros(1, dtype=torch.int32, device="cuda"), new, 2 * new)
    torch.cuda.synchronize()
    for i in range(2):
        k, s = np.zeros((2, Hkv, page, D), np.uint8), np.zeros((2, Hkv, page // block), np.float32)
        orc.append_fp8(k, s, np.array([[0, 1]]), [0], new.double().cpu().numpy() * (1 + i), block)
        assert np.array_equal(big[i][[pages - 1, pages - 3]].cpu().numpy(), k) and np.array_equal(scales[i][[pages - 1, pages - 3]].cpu().numpy(), s)
        big[i][[pages - 1, pages - 3]] = 0
        assert int(big[i].view(torch.int64).ne(0).sum()) == 0


def test_values_are_what_the_append_was_given():
    # a round trip: every value within half a step of its code (2^-4 of it, or of the block's subnormal step)
    rng = np.random.default_rng(19)
    x = torch.from_numpy(rng.standard_normal((2, 2, 100, 128)).astype(np.float32)).cuda()
    k = torch.zeros(2, 2, 128, 128, dtype=torch.float8_e4m3fn, device="cuda")
    v, ks = torch.zeros_like(k), torch.zeros(2, 2, 4, device="cuda")
    vs, ln = torch.zeros_like(ks), torch.zeros(2, dtype=torch.int32, device="cuda")
    _F().kv_cache_append_fp8(k, v, ks, vs, ln, x, x)
    torch.cuda.synchronize()
    got = orc.values(_codes(k), ks.cpu().numpy())[:, :, :100]
    want = x.double().cpu().numpy()
    step = np.repeat(ks.cpu().numpy(), 32, 2)[:, :, :100, None] * 2.0 ** -10
    assert np.all(np.abs(got - want) <= np.maximum(np.abs(want) * 2.0 ** -4, step))
    assert e4m3fn_decode(_codes(k)).max() > 224  # the scale is the smallest one
