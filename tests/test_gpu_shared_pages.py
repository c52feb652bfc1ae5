"""Fork, reserve (copy on write) and compact of a paged cache's tables, against plain loops: whole numbers and copied bytes, equal."""
import numpy as np
import pytest
import torch

from oracle import shared as orc

pytestmark = pytest.mark.gpu


def _F():
    import dtorch_amd.nn.functional as F
    return F


def _i32(x):
    return torch.from_numpy(np.ascontiguousarray(x, dtype=np.int32)).cuda()


def _state(rng, B, page, columns, P, most=None, share=True):
    """A table whose sequences share their first pages in part, with lengths, counts and consistent pages."""
    most = columns * page if most is None else most
    ids = list(rng.permutation(P))
    table = np.full((B, columns), -1, dtype=np.int32)
    lengths = np.zeros(B, dtype=np.int32)
    for b in range(B):
        n = int(rng.integers(0, most + 1))
        need = -(-n // page)
        if share and b and rng.random() < 0.7:  # the front of an earlier sequence
            a = int(rng.integers(0, b))
            have = int(rng.integers(0, -(-int(lengths[a]) // page) + 1))
            table[b, :have] = table[a, :have]
            if rng.random() < 0.5:
                n, need = min(n, int(lengths[a])), -(-min(n, int(lengths[a])) // page)
        while need and (table[b, :need] < 0).sum() > len(ids):
            need -= 1
        n = min(n, need * page)
        for s in range(need):
            if table[b, s] < 0:
                table[b, s] = ids.pop()
        table[b, need:] = -1
        lengths[b] = n
    return table, lengths, orc.references(table, P)


def _pools(rng, P, H, page, D, dtype, extra):
    out = [torch.from_numpy(rng.standard_normal((P, H, page, D)).astype(np.float32)).to(dtype) for _ in range(2)]
    if "scales" in extra:
        out += [torch.from_numpy(rng.standard_normal((P, H, page // 16)).astype(np.float32)) for _ in range(2)]
    if "bounds" in extra:
        out += [torch.from_numpy(rng.standard_normal((P, H, page // 16, D)).astype(np.float32)).to(dtype) for _ in range(2)]
    return out


def _num(t):
    return t.float().cpu().numpy() if t.dtype != torch.float8_e4m3fn else t.view(torch.uint8).cpu().numpy()


@pytest.mark.parametrize("B,columns,P", [(1, 1, 1), (2, 3, 5), (7, 33, 200), (64, 130, 3000), (300, 17, 2000), (8192, 2, 4000)])
def test_fork(B, columns, P):
    rng = np.random.default_rng(B + columns)
    table, lengths, refs = _state(rng, B, 16, columns, P)
    for parents in (rng.integers(-2, B + 2, B), np.zeros(B, dtype=int), np.full(B, -1), np.arange(B)[::-1].copy()):
        want = orc.fork(table, lengths, refs, parents)
        wide = torch.full((B, columns + 3), 77, dtype=torch.int32, device="cuda")  # a view of rows further apart
        wide[:, :columns] = _i32(table)
        dl, dr = _i32(lengths), _i32(refs)
        _F().kv_pages_fork(wide[:, :columns], dl, dr, _i32(parents))
        for got, w in zip((wide[:, :columns], dl, dr), want):
            assert np.array_equal(got.cpu().numpy(), w)
        assert (wide[:, columns:] == 77).all()


RESERVE = [
    # B, page, columns, P, n, heads, D, dtype, extra pools
    (1, 16, 1, 1, 1, 1, 64, torch.bfloat16, ""),
    (5, 16, 8, 60, 1, 2, 64, torch.float16, "scales"),
    (5, 32, 8, 60, 1, 3, 128, torch.float32, "bounds"),
    (9, 64, 5, 40, 70, 2, 80, torch.bfloat16, "bounds"),
    (40, 16, 20, 700, 1, 2, 128, torch.bfloat16, "scales bounds"),
    (40, 16, 20, 700, 100, 1, 8, torch.float32, "scales"),
    (3, 256, 3, 12, 300, 2, 128, torch.float16, ""),
    (600, 16, 12, 9000, 90, 1, 4, torch.float32, ""),   # more slots than LDS holds
    (1500, 16, 3, 9000, 1, 1, 4, torch.float32, ""),
    (6, 16, 6, 12, 30, 1, 64, torch.bfloat16, ""),      # not enough pages
    (4, 16, 4, 40, 1000, 1, 64, torch.bfloat16, ""),    # more tokens than a sequence holds
]


@pytest.mark.parametrize("B,page,columns,P,n,H,D,dtype,extra", RESERVE)
@pytest.mark.parametrize("layout", ["natural", "tokens first"])
def test_reserve(B, page, columns, P, n, H, D, dtype, extra, layout):
    rng = np.random.default_rng(B * 7 + n)
    table, lengths, refs = _state(rng, B, page, columns, P)
    parents = rng.integers(-1, B, B)  # as a beam search leaves them
    table, lengths, refs = orc.fork(table, lengths, refs, parents)
    lengths[rng.random(B) < 0.2] //= 2  # sequences cut short: whole pages are written then
    pools = _pools(rng, P, H, page, D, dtype, extra)
    dev = []
    for x in pools:
        if layout == "natural":
            dev.append(x.cuda())
        else:  # [P, page, H, D] behind a permuted view
            dev.append(x.transpose(1, 2).contiguous().cuda().transpose(1, 2))
    want_p, want_t, want_r, short = orc.reserve([_num(x) for x in pools], table, lengths, refs, n, page)
    dt, dl, dr = _i32(table), _i32(lengths), _i32(refs)
    got = _F().kv_pages_reserve(dev, dt, dl, dr, n)
    assert got.tolist() == [short]
    assert np.array_equal(dt.cpu().numpy(), want_t) and np.array_equal(dr.cpu().numpy(), want_r)
    assert np.array_equal(dl.cpu().numpy(), lengths)
    for a, b in zip(dev, want_p):
        assert np.array_equal(_num(a), b)


def test_reserve_lengths_outside_the_table():
    """Lengths below 0 count as 0, those at or past the capacity write nothing."""
    table = np.array([[0, 1], [0, 2], [3, -1], [0, 4]], dtype=np.int32)
    lengths = np.array([-5, 32, 16, 40], dtype=np.int32)
    refs = orc.references(table, 8)
    pools = [torch.arange(8 * 16 * 4, dtype=torch.float32).view(8, 1, 16, 4) + i for i in (0, 9)]
    want_p, want_t, want_r, short = orc.reserve([x.numpy() for x in pools], table, lengths, refs, 1, 16)
    dev, dt, dr = [x.cuda() for x in pools], _i32(table), _i32(refs)
    assert _F().kv_pages_reserve(dev, dt, _i32(lengths), dr, 1).tolist() == [short]
    assert np.array_equal(dt.cpu().numpy(), want_t) and np.array_equal(dr.cpu().numpy(), want_r)
    for a, b in zip(dev, want_p):
        assert np.array_equal(_num(a), b)


def test_reserve_nothing():
    table = _i32([[0, 1]])
    refs, k = _i32([1, 1, 0]), torch.zeros(3, 1, 16, 8, device="cuda")
    assert _F().kv_pages_reserve([k, k.clone()], table, _i32([20]), refs, 0).tolist() == [0]
    assert table.tolist() == [[0, 1]] and refs.tolist() == [1, 1, 0]


@pytest.mark.parametrize("P,B,columns,page,H,D,dtype,extra", [
    (1, 1, 1, 16, 1, 8, torch.float32, ""), (2, 1, 1, 16, 2, 64, torch.bfloat16, "scales"), (63, 4, 9, 32, 3, 80, torch.float16, "bounds"),
    (500, 9, 30, 16, 2, 64, torch.bfloat16, "scales bounds"), (40000, 100, 200, 16, 1, 4, torch.float32, ""), (17, 3, 4, 256, 2, 128, torch.float32, "")])
@pytest.mark.parametrize("layout", ["natural", "tokens first", "apart"])
def test_compact(P, B, columns, page, H, D, dtype, extra, layout):
    rng = np.random.default_rng(P)
    table, lengths, refs = _state(rng, B, page, columns, P)
    pools = _pools(rng, P, H, page, D, dtype, extra)
    dev = []
    for x in pools:
        if layout == "natural":
            dev.append(x.cuda())
        elif layout == "tokens first":
            dev.append(x.transpose(1, 2).contiguous().cuda().transpose(1, 2))
        else:  # every second page and head of a larger pool
            big = torch.full((2 * x.shape[0], 2 * x.shape[1], *x.shape[2:]), -3.0, dtype=x.dtype, device="cuda")
            big[::2, 1::2] = x.cuda()
            dev.append(big[::2, 1::2])
    want_p, want_t, want_r, used = orc.compact([_num(x) for x in pools], table, refs)
    dt, dr = _i32(table), _i32(refs)
    assert _F().kv_pages_compact(dev, dt, dr).tolist() == [used]
    assert np.array_equal(dt.cpu().numpy(), want_t) and np.array_equal(dr.cpu().numpy(), want_r)
    for a, b in zip(dev, want_p):
        assert np.array_equal(_num(a), b)
    if layout == "apart":
        for x in dev:
            assert (x._base[1::2] == -3.0).all() and (x._base[:, ::2] == -3.0).all()


def test_compact_full_and_empty():
    for refs in ([1, 1, 2], [0, 0, 0]):
        table = _i32([[0, 1, 2, 2]] if refs[0] else [[-1, -1, -1, -1]])
        before, k = table.clone(), torch.randn(3, 1, 16, 8, device="cuda")
        was = k.clone()
        dr = _i32(refs)
        assert _F().kv_pages_compact([k, was.clone()], table, dr).tolist() == [sum(r > 0 for r in refs)]
        assert torch.equal(table, before) and torch.equal(k, was) and dr.tolist() == refs


def test_captured_beam_steps():
    """Fork, reserve, append and decode of a beam search in one graph, replayed with other parents each time, against eager calls."""
    F = _F()
    rng = np.random.default_rng(3)
    B, H, page, columns, P, D = 6, 2, 16, 6, 60, 64
    table, lengths, refs = _state(rng, B, page, columns, P, most=40)
    start = dict(t=_i32(table), l=_i32(lengths), r=_i32(refs), k=torch.randn(P, H, page, D, device="cuda", dtype=torch.bfloat16),
                 v=torch.randn(P, H, page, D, device="cuda", dtype=torch.bfloat16))
    parents = _i32(np.zeros(B))
    q = torch.empty(B, 2 * H, 1, D, device="cuda", dtype=torch.bfloat16)
    kn, vn = (torch.empty(B, H, 1, D, device="cuda", dtype=torch.bfloat16) for _ in range(2))

    def step(s):
        F.kv_pages_fork(s["t"], s["l"], s["r"], parents)
        short = F.kv_pages_reserve([s["k"], s["v"]], s["t"], s["l"], s["r"], 1)
        F.kv_cache_append_paged(s["k"], s["v"], s["t"], s["l"], kn, vn)
        return F.decode_attention_paged(q, s["k"], s["v"], s["t"], s["l"])[0], short

    eager, held = ({n: x.clone() for n, x in start.items()} for _ in range(2))
    warm = {n: x.clone() for n, x in start.items()}
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(warm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, short = step(held)
    for i in range(5):
        parents.copy_(_i32(rng.integers(-1 if i == 2 else 0, B, B)))
        for x in (q, kn, vn):
            x.normal_()
        want, lack = step(eager)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and short.tolist() == lack.tolist() == [0]
        for n in "tlrkv":
            assert torch.equal(held[n], eager[n]), (i, n)


def test_host_refusals():
    F = _F()
    t, l, r, p = _i32([[0, 1]]), _i32([20]), _i32([1, 1, 0]), _i32([0])
    k = torch.zeros(3, 1, 16, 8, device="cuda")
    for bad in (dict(t=t.float()), dict(t=t[0]), dict(l=l.long()), dict(l=_i32([1, 2])), dict(r=r[::2]), dict(p=_i32([0, 0])), dict(p=p.long()),
                dict(t=_i32([[0]]).expand(1, 3)), dict(t=_i32([[0, 1, 2]])[:, ::2]), dict(p=p.cpu())):
        a = dict(dict(t=t, l=l, r=r, p=p), **bad)
        with pytest.raises(ValueError):
            F.kv_pages_fork(a["t"], a["l"], a["r"], a["p"])
    with pytest.raises(ValueError):  # one row for two sequences
        F.kv_pages_fork(_i32([[0, 1]]).expand(2, 2), _i32([1, 2]), r, _i32([0, 0]))
    for pools in ([], [k, k], [k[:2], k.clone()], [k.expand(3, 2, 16, 8)], [k[..., 0]], [k, torch.zeros(3, 1, 5, device="cuda")],
                  [torch.zeros(3, 1, 16, 3, device="cuda", dtype=torch.bfloat16)], [k[..., ::2]], [k.clone() for _ in range(9)],
                  [torch.zeros(3, 1, 24, 8, device="cuda")], [k.cpu()]):
        with pytest.raises(ValueError):
            F.kv_pages_reserve(pools, t, l, r, 1)
        with pytest.raises(ValueError):
            F.kv_pages_compact(pools, t, r)
    with pytest.raises(ValueError):
        F.kv_pages_reserve([k], t, l, r, -1)
    assert t.tolist() == [[0, 1]] and r.tolist() == [1, 1, 0]


@pytest.mark.parametrize("P", [1023, 1024, 1025, 4096, 4097, 8192, 8193, 16384, 16385, 40001])
def test_compact_page_counts(P):
    """Page counts on either side of where the plan changes; counts at an odd address; every page alike, so the table tells them apart."""
    rng = np.random.default_rng(P)
    table, lengths, refs = _state(rng, 16, 16, min(P // 24, 300), P)
    pool = torch.arange(P, dtype=torch.int32)[:, None, None, None].repeat(1, 1, 16, 1)
    want_p, want_t, want_r, used = orc.compact([_num(pool)], table, refs)
    held = torch.full((P + 1,), 7, dtype=torch.int32, device="cuda")
    dp, dt, dr = pool.cuda(), _i32(table), held[1:]
    dr.copy_(_i32(refs))
    assert _F().kv_pages_compact([dp], dt, dr).item() == used
    assert np.array_equal(dt.cpu().numpy(), want_t) and np.array_equal(dr.cpu().numpy(), want_r)
    live = want_r > 0
    assert np.array_equal(_num(dp)[live], want_p[0][live]) and held[0].item() == 7
