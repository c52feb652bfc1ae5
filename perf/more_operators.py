"""Performance cases of a KV cache whose pages are shared and which is read in part: page tables that fork, grow and are
compacted on the device, decode attention over a shared prefix, and decode attention over the key blocks that a bound
of their scores selects, through dtorch_amd.nn.functional.

A case is a dict with a "kind" (the operator or the chain of them), its sizes and its types; `listed()` holds two or more
of each, `draw()` gives more over the same ranges.  `run()` computes a case in elementary torch operations, or with
`own` set through the package's operators.  Heads and head dims are those of the models that the package names (Llama:
32 query / 8 kv heads of 128) and of generic multi-head layers.  Inputs are unit normals, which is what projections
behind a norm layer give; keys have channels of different sizes, as they do behind a projection.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4}


def listed():
    return [
        # a step of beam search over two requests: sequences continue their parents, and each gets room for a token
        dict(name="beam_step", kind="beam", G=2, beams=4, Hkv=8, lo=300, hi=1500, tail=40, D=128, page=16, n=1, dtype="bf16"),
        # the same of a serving batch: 32 requests of four beams over pages of 64 tokens
        dict(name="beam_batch", kind="beam", G=32, beams=4, Hkv=8, lo=500, hi=2000, tail=150, D=128, page=64, n=1, dtype="fp16"),
        # a small pool of full precision, half of it freed, made dense
        dict(name="compact_small", kind="compact", P=512, used=230, B=8, Hkv=12, D=64, page=16, dtype="fp32"),
        # a large pool after many requests have come and gone
        dict(name="compact_pool", kind="compact", P=8000, used=4100, B=64, Hkv=8, D=128, page=16, dtype="bf16"),
        # four samples of one prompt: a token's attention (latency)
        dict(name="shared_samples", kind="shared", G=1, B=4, Hq=32, Hkv=8, plo=2000, phi=2000, lo=1, hi=100, D=128, page=16, dtype="bf16"),
        # a serving batch behind one long system prompt, own parts of mixed lengths
        dict(name="shared_prompt", kind="shared", G=1, B=64, Hq=32, Hkv=8, plo=8192, phi=8192, lo=16, hi=1500, D=128, page=16, dtype="bf16"),
        # four prompts of eight samples each in padded full-precision caches
        dict(name="shared_fp32", kind="shared", G=4, B=32, Hq=12, Hkv=12, plo=1000, phi=4001, lo=5, hi=333, D=64, page=0, dtype="fp32"),
        # key bounds of four prompts just cached
        dict(name="bounds_prompts", kind="bounds", B=4, Hkv=8, n=4000, lo=4000, hi=4000, D=128, block=64, page=64, dtype="bf16"),
        # key bounds after a step of a serving batch
        dict(name="bounds_step", kind="bounds", B=64, Hkv=8, n=1, lo=512, hi=8191, D=128, block=32, page=32, dtype="fp16"),
        # one token of one long context reads 2048 of its 30000 tokens
        dict(name="sparse_one", kind="sparse", B=1, Hq=32, Hkv=8, lo=30000, hi=30000, keep=2048, recent=256, D=128, block=64, page=0, dtype="bf16"),
        # a serving batch of long contexts over a paged cache
        dict(name="sparse_batch", kind="sparse", B=32, Hq=32, Hkv=8, lo=3000, hi=32000, keep=4096, recent=512, D=128, block=64, page=64, dtype="bf16"),
        # a full-precision multi-head layer
        dict(name="sparse_fp32", kind="sparse", B=4, Hq=12, Hkv=12, lo=900, hi=9000, keep=1024, recent=64, D=64, block=32, page=0, dtype="fp32"),
    ]


# Rates (operations a second, bytes a second) by which draw() bounds a case's cost, and the tokens times heads times head
# dims that a case's caches may hold.
_MOST_S = 90e-6
_MOST_CACHE = 32 * 32000 * 8 * 128


def _cost(c):
    w = work(c)
    return w["flops"] / (0.05e15 if c["dtype"] == "fp32" else 0.4e15) + w["bytes"] / 4.5e12


def _cache(c):
    kind = c["kind"]
    if kind == "compact":
        tokens = c["P"] * c["page"]
    elif kind == "beam":
        tokens = _beam_pages(c) * c["page"]
    else:
        tokens = c["B"] * c["hi"] + (c["G"] * c["phi"] if kind == "shared" else 0)
    return tokens * c["Hkv"] * c["D"] * _SIZE[c["dtype"]] / 2


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["beam", "compact", "shared", "shared", "bounds", "sparse", "sparse"])
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128), (32, 32, 128), (12, 12, 64), (20, 20, 64), (16, 2, 80)])
    t = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "beam":
        hi = _log(rng, 4, 8000)
        return dict(kind=kind, G=_log(rng, 1, 64), beams=rng.randint(1, 8), Hkv=hkv, lo=rng.randint(0, hi), hi=hi, tail=_log(rng, 1, 300), D=d,
                    page=rng.choice([16, 16, 64, 256]), n=rng.choice([1, 1, 1, rng.randint(2, 100)]), dtype=t)
    if kind == "compact":
        pages = _log(rng, 16, 16000)
        return dict(kind=kind, P=pages, used=max(1, round(pages * rng.uniform(0.1, 0.95))), B=_log(rng, 1, 128), Hkv=hkv, D=d,
                    page=rng.choice([16, 16, 64, 256]), dtype=t)
    if kind == "shared":
        g, hi, phi = rng.choice([1, 1, 2, 4, 8]), _log(rng, 1, 4096), _log(rng, 16, 32768)
        return dict(kind=kind, G=g, B=g * _log(rng, 1, 96 // g), Hq=hq, Hkv=hkv, plo=max(1, phi // rng.choice([1, 2, 4])), phi=phi,
                    lo=rng.choice([0, hi // 8, hi // 2, hi]), hi=hi, D=d, page=rng.choice([0, 0, 16, 32, 256]), dtype=t)
    page = rng.choice([0, 0, 16, 64, 256])
    block = rng.choice([b for b in (16, 32, 64, 128) if page == 0 or b <= page])
    if kind == "bounds":
        hi = _log(rng, 1, 32000)
        n = rng.choice([1, 1, _log(rng, 1, hi)])
        return dict(kind=kind, B=_log(rng, 1, 64), Hkv=hkv, n=n, lo=max(n, hi // rng.choice([1, 2, 8])), hi=hi, D=d, block=block, page=page, dtype=t)
    hi = _log(rng, 64, 65536)
    keep = max(1, hi // block // rng.choice([1, 2, 4, 8, 16])) * block
    return dict(kind=kind, B=_log(rng, 1, 64), Hq=hq, Hkv=hkv, lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, keep=keep,
                recent=max(1, keep // block // rng.choice([4, 8, 16])) * block, D=d, block=block, page=page, dtype=t)


def draw(rng):
    while True:
        c = _drawn(rng)
        if _cache(c) <= _MOST_CACHE and _cost(c) <= _MOST_S:
            return c


def _spread(lo, hi, n):
    """n whole numbers, spread evenly over [lo, hi]."""
    return [hi - (hi - lo) * i // max(n - 1, 1) for i in range(n)]


def _up(x, unit):
    return -(-x // unit) * unit


def _beam_pages(c):
    """Pages of a beam case's pool: the prompts', each beam's own behind them and a new one, and some free ones."""
    prompts = sum(n // c["page"] for n in _spread(c["lo"], c["hi"], c["G"]))
    tails = c["G"] * c["beams"] * (-(-(c["page"] + c["tail"]) // c["page"]) + -(-c["n"] // c["page"]) + 1)
    return prompts + tails + 16


def _room(c):
    """Positions of each sequence of a cache: whole blocks and pages."""
    return _up(max(c["hi"], 1), max(c["page"], c.get("block", 0), 64))


def work(c):
    d, h, kind = c["D"], c["Hkv"], c["kind"]
    e = _SIZE[c["dtype"]]
    if kind == "beam":  # rows of the table, and a last page for all beams but one of each parent, half full on average
        B = c["G"] * c["beams"]
        rows = sum(n // c["page"] for n in _spread(c["lo"], c["hi"], c["G"])) * c["beams"] + B * (c["tail"] // c["page"] + 1)
        return {"bytes": 8 * rows + 16 * B + 4 * (B // 2) * (c["page"] // 2) * h * d * e, "flops": B}
    if kind == "compact":  # of the used pages as many lie behind the last one to be kept as there are holes before it
        moved = c["used"] * (c["P"] - c["used"]) // c["P"]
        return {"bytes": 4 * moved * c["page"] * h * d * e + 8 * c["used"] + 8 * c["P"], "flops": c["P"]}
    if kind == "shared":
        prefix, tails = _prefixes(c), _spread(c["lo"], c["hi"], c["B"])
        pairs = sum(tails) + sum(prefix) * (c["B"] // c["G"])
        data = 2 * (sum(prefix) + sum(tails)) * h * d * e + 2 * c["B"] * c["Hq"] * d * e + 4 * c["B"] * c["Hq"]
        return {"bytes": data, "flops": 4 * pairs * c["Hq"] * d}
    ns = _spread(c["lo"], c["hi"], c["B"])
    if kind == "bounds":
        rows = sum(n - (n - c["n"]) // c["block"] * c["block"] for n in ns)
        blocks = sum(-(-n // c["block"]) - (n - c["n"]) // c["block"] for n in ns)
        return {"bytes": (rows + 2 * blocks) * h * d * e, "flops": 2 * rows * h * d}
    keep, recent = c["keep"] // c["block"], c["recent"] // c["block"]
    blocks = [-(-n // c["block"]) for n in ns]
    scored = sum(n - recent for n in blocks if n > keep)
    tokens = sum(min(n, c["keep"]) for n in ns)
    data = (2 * scored + 2 * tokens) * h * d * e + 2 * c["B"] * c["Hq"] * d * e + 4 * c["B"] * (c["Hq"] + h * keep)
    return {"bytes": data, "flops": (4 * tokens + 4 * scored) * c["Hq"] * d}


def _prefixes(c):
    """Shared tokens of each group; whole pages of a paged cache."""
    return [_up(n, c["page"]) if c["page"] else n for n in _spread(c["plo"], c["phi"], c["G"])]


# ---- inputs ------------------------------------------------------------------------------------------------

def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, h, d, page = c["kind"], c["Hkv"], c["D"], c["page"]
    t = _DT[c["dtype"]]
    st = {"case": c}

    def normal(*shape):
        return torch.randn(*shape, device="cuda", generator=g).to(t)

    def keys(*shape):
        return normal(*shape) * torch.exp(0.5 * torch.randn(h, 1, d, device="cuda", generator=g)).to(t)

    def perm(n):
        return torch.randperm(n, device="cuda", generator=g).to(torch.int32)

    if kind == "beam":
        B, P = c["G"] * c["beams"], _beam_pages(c)
        st["k"], st["v"] = keys(P, h, page, d), normal(P, h, page, d)
        prompts = _spread(c["lo"], c["hi"], c["G"])
        columns = (c["hi"] + c["tail"] + c["n"]) // page + 2
        ids = perm(P).tolist()
        tails = torch.randint(0, c["tail"] + 1, (B,), device="cuda", generator=g).tolist()
        table, lengths = [], []
        for i, n in enumerate(prompts):
            shared = [ids.pop() for _ in range(n // page)]
            for b in range(c["beams"]):
                length = n + tails[i * c["beams"] + b]
                row = shared + [ids.pop() for _ in range(-(-length // page) - len(shared))]
                table.append(row + [-1] * (columns - len(row)))
                lengths.append(length)
        st["table"] = torch.tensor(table, dtype=torch.int32, device="cuda")
        st["lengths"] = torch.tensor(lengths, dtype=torch.int32, device="cuda")
        first = torch.arange(B, device="cuda") // c["beams"] * c["beams"]
        st["parents"] = (first + torch.randint(0, c["beams"], (B,), device="cuda", generator=g)).to(torch.int32)
        st["parents"][perm(B)[:B // 16].long()] = -1  # sequences that have ended
        st["refs"] = _references(st["table"], P)
        return st | {n + "0": st[n].clone() for n in ("table", "lengths", "refs")}
    if kind == "compact":
        P, B = c["P"], c["B"]
        st["k"], st["v"] = keys(P, h, page, d), normal(P, h, page, d)
        columns = -(-c["used"] // B)
        table = perm(P)[:c["used"]]
        st["table"] = torch.nn.functional.pad(table, (0, B * columns - c["used"]), value=-1).view(columns, B).t().contiguous()
        st["refs"] = _references(st["table"], P)
        return st | {n + "0": st[n].clone() for n in ("table", "refs")}
    B = c["B"]
    st["lengths"] = torch.tensor(_spread(c["lo"], c["hi"], B), dtype=torch.int32, device="cuda")[perm(B).long()]
    if kind == "shared":
        st["q"] = normal(B, c["Hq"], 1, d)
        prefix = _prefixes(c)
        st["prefix"] = torch.tensor(prefix, dtype=torch.int32, device="cuda")
        if not page:
            most = _up(max(prefix), 64)
            st["kp"], st["vp"] = keys(c["G"], h, most, d), normal(c["G"], h, most, d)
            st["k"], st["v"] = keys(B, h, _room(c), d), normal(B, h, _room(c), d)
            return st
        behind = _room(c) // page
        P = sum(prefix) // page + B * behind
        st["k"], st["v"] = keys(P, h, page, d), normal(P, h, page, d)
        ids = perm(P)
        table = torch.full((B, max(prefix) // page + behind), -1, dtype=torch.int32, device="cuda")
        at, n = 0, B // c["G"]
        for i, p in enumerate(prefix):
            table[i * n:(i + 1) * n, :p // page] = ids[at:at + p // page]
            at += p // page
        for b in range(B):
            p = prefix[b // n] // page
            table[b, p:p + behind] = ids[at:at + behind]
            at += behind
        st["table"] = table
        st["lengths"] += st["prefix"].repeat_interleave(n)
        return st
    pool = (B * (_room(c) // page), h, page, d) if page else (B, h, _room(c), d)
    st["k"] = keys(*pool)
    if page:
        st["table"] = perm(pool[0]).view(B, -1)
    blocked = st["k"].unflatten(2, (-1, c["block"]))
    if kind == "bounds":
        st["kmin"] = torch.zeros_like(blocked[..., 0, :])
        st["kmax"] = torch.zeros_like(st["kmin"])
        return st
    st["q"], st["v"] = normal(B, c["Hq"], 1, d), normal(*pool)
    st["kmin"], st["kmax"] = blocked.amin(3), blocked.amax(3)
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------

def _references(table, P):
    """How many slots of the table name each page."""
    slots = table.flatten().long()
    return torch.zeros(P, dtype=torch.int32, device=table.device).scatter_add_(0, slots.clamp(min=0), (slots >= 0).to(torch.int32))


def _fork_plain(st):
    table, lengths, parents = st["table"], st["lengths"], st["parents"].long()
    lives = (parents >= 0) & (parents < len(parents))
    p = parents.clamp(0, len(parents) - 1)
    table.copy_(torch.where(lives[:, None], table[p], torch.full_like(table, -1)))
    lengths.copy_(torch.where(lives, lengths[p], torch.zeros_like(lengths)))
    st["refs"].copy_(_references(table, len(st["refs"])))


def _reserve_plain(st):
    c, table, refs, n = st["case"], st["table"], st["refs"], st["lengths"].long()
    page, B, P = c["page"], len(n), len(refs)
    first, last = n // page, (n + c["n"] - 1) // page
    slots = first[:, None] + torch.arange((c["n"] + page - 2) // page + 1, device=n.device)  # [B, slots]
    inside = (slots <= last[:, None]) & (slots < table.shape[1])
    at = slots.clamp(max=table.shape[1] - 1)
    was = torch.where(inside, table.gather(1, at).long(), torch.full_like(at, -1))
    # a page that several sequences write goes to the last of them, if no one else holds it: the others before it copy
    flat = was.flatten()
    same = (flat[:, None] == flat[None]) & (flat >= 0)[:, None]
    rank = torch.tril(same, -1).sum(1).view_as(was)
    held = refs.long()[was.clamp(min=0)]
    copies = (was >= 0) & (rank < held - 1)
    needs = copies | (inside & (was < 0))
    k = needs.flatten().cumsum(0).view_as(was) - 1  # which fresh page
    free = torch.argsort((refs > 0).to(torch.uint8), stable=True)  # free ones first, ascending
    count = (refs == 0).sum()
    fresh = torch.where(k < count, free[k.clamp(0, P - 1)], torch.full_like(k, -1))
    wider = torch.nn.functional.pad(table, (0, 1))  # a column for the slots that stay as they are
    wider.scatter_(1, torch.where(needs, at, table.shape[1]), fresh.to(torch.int32))
    table.copy_(wider[:, :-1])
    source = torch.where(copies, was, torch.zeros_like(was))
    refs.scatter_add_(0, source.flatten(), -copies.flatten().to(torch.int32))
    refs.scatter_add_(0, fresh.clamp(min=0).flatten(), (needs & (fresh >= 0)).flatten().to(torch.int32))
    # rows of tokens in a copied page: those of the first slot
    rows = torch.where(copies & (slots == first[:, None]) & (fresh >= 0), (n % page)[:, None], torch.zeros_like(was))
    b = torch.nonzero(rows.flatten())[:, 0]
    take = torch.arange(page, device=n.device) < rows.flatten()[b][:, None]
    for x in (st["k"], st["v"]):
        to = fresh.flatten()[b]
        x[to] = torch.where(take[:, None, :, None], x[flat[b]], x[to])
    return (needs.sum() - count).clamp(min=0).to(torch.int32).view(1)


def _compact_plain(st):
    table, refs = st["table"], st["refs"]
    P = len(refs)
    used = refs > 0
    count = used.sum()
    ids = torch.arange(P, device=refs.device)
    to, source = ids[~used & (ids < count)], ids[used & (ids >= count)]
    for x in (st["k"], st["v"]):
        x[to] = x[source]
    new = ids.clone()
    new[source] = to
    table.copy_(torch.where(table >= 0, new[table.clamp(min=0).long()].to(torch.int32), table))
    refs[to] = refs[source]
    refs[source] = 0
    return count.to(torch.int32).view(1)


def _own_rows(st, x, columns=None):
    """[B, Hkv, S, D] rows of a padded or paged cache (of the table's `columns`), in 32 bits."""
    if "table" not in st:
        return x.float()
    ids = st["table"].clamp(min=0).long()
    return x[ids if columns is None else ids[:, columns]].transpose(1, 2).flatten(2, 3).float()


def _shared_plain(st):
    c = st["case"]
    B, hq, _, d = st["q"].shape
    h, G = c["Hkv"], c["G"]
    n = B // G
    q = st["q"].float().view(B, h, hq // h, d)
    outs, lses = [], []
    for g, prefix in enumerate(_prefixes(c)):
        rows = slice(g * n, (g + 1) * n)
        one = {"table": st["table"][rows]} if c["page"] else {}
        lengths = st["lengths"][rows].long().view(n, 1, 1, 1)
        if c["page"]:
            many = prefix // c["page"]
            kp, vp = (_own_rows({"table": one["table"][:1, :many]}, st[x])[0] for x in "kv")
            own_columns = slice(many, many + _room(c) // c["page"])
            k, v = (_own_rows(one, st[x], own_columns) for x in "kv")
            lengths = lengths - prefix
        else:
            kp, vp = st["kp"][g, :, :prefix].float(), st["vp"][g, :, :prefix].float()
            k, v = st["k"][rows].float(), st["v"][rows].float()
        qg = q[rows]
        folded = qg.transpose(0, 1).reshape(h, -1, d)  # a kv head's rows of all sequences
        sp = folded @ kp.transpose(1, 2) / math.sqrt(d)
        s = qg @ k.transpose(2, 3) / math.sqrt(d)
        s.masked_fill_(torch.arange(s.shape[-1], device=s.device) >= lengths, -math.inf)
        m = torch.maximum(sp.amax(-1).view(h, n, -1).transpose(0, 1), s.amax(-1))[..., None]  # [n, h, group, 1]
        pp = torch.exp(sp - m.transpose(0, 1).reshape(h, -1, 1))
        p = torch.exp(s - m)
        z = p.sum(-1) + pp.sum(-1).view(h, n, -1).transpose(0, 1)
        o = p @ v + (pp @ vp).view(h, n, -1, d).transpose(0, 1)
        outs.append((o / z[..., None]).reshape(n, hq, 1, d))
        lses.append((m[..., 0] + torch.log(z)).reshape(n, hq))
    return torch.cat(outs).to(st["q"].dtype), torch.cat(lses)


def _bounds_plain(st):
    c = st["case"]
    block, n = c["block"], st["lengths"].long()
    # the blocks of the last n tokens
    first, last = (n - c["n"]).clamp(min=0) // block, (n + block - 1) // block
    blocks = first[:, None] + torch.arange((c["n"] + block - 2) // block + 1, device=n.device)  # [B, blocks]
    b, i = torch.nonzero(blocks < last[:, None], as_tuple=True)
    j = blocks[b, i]
    t = j[:, None] * block + torch.arange(block, device=n.device)
    inside = (t < n[b][:, None])[:, :, None, None]
    if c["page"]:
        slot = st["table"].long()[b, j * block // c["page"]]
        r = t % c["page"]
    else:
        slot, r = b, t
    x = st["k"][slot[:, None], :, r]  # [blocks, block, Hkv, D]
    where = r[:, 0] // block
    st["kmin"][slot, :, where] = torch.where(inside, x, torch.full_like(x, math.inf)).amin(1)
    st["kmax"][slot, :, where] = torch.where(inside, x, torch.full_like(x, -math.inf)).amax(1)
    return st["kmin"], st["kmax"]


def _select_plain(st):
    c = st["case"]
    B, hq, _, d = st["q"].shape
    block, h = c["block"], c["Hkv"]
    keep, recent = c["keep"] // block, c["recent"] // block
    lo, hi = st["kmin"], st["kmax"]
    if c["page"]:
        ids = st["table"].long()
        lo, hi = (x[ids].transpose(1, 2).flatten(2, 3) for x in (lo, hi))
    q = st["q"].double().view(B, h, hq // h, d)
    # sum over dims of the larger of q kmin and q kmax, in 64 bits: scores next to one another decide
    score = q.clamp(min=0) @ hi.double().transpose(2, 3).contiguous() + q.clamp(max=0) @ lo.double().transpose(2, 3).contiguous()
    score = score.amax(2).float()  # [B, Hkv, blocks]
    blocks = (st["lengths"].long() + block - 1) // block
    at = torch.arange(score.shape[2], device=score.device)
    old = at < (blocks - recent)[:, None, None]
    score.masked_fill_(~old, -math.inf)
    rank = torch.argsort(torch.argsort(score, dim=-1, descending=True, stable=True), dim=-1)
    there = at < blocks[:, None, None]
    stays = torch.where((blocks > keep)[:, None, None], (old & (rank < keep - recent)) | (~old & there), there).expand_as(score)
    order = torch.argsort((~stays).to(torch.uint8), dim=-1, stable=True)[..., :keep]
    order = torch.nn.functional.pad(order, (0, keep - order.shape[2]))
    return torch.where(torch.arange(keep, device=score.device) < blocks[:, None, None], order, -1).to(torch.int32)


def _blocks_plain(st, ids):
    c = st["case"]
    B, hq, _, d = st["q"].shape
    h, block = c["Hkv"], c["block"]
    t = (ids.clamp(min=0).long()[..., None] * block + torch.arange(block, device=ids.device))  # [B, Hkv, keep, block]
    there = (ids >= 0)[..., None] & (t < st["lengths"].view(B, 1, 1, 1))
    t, there = t.flatten(2), there.flatten(2)
    if c["page"]:
        slot = st["table"].long()[torch.arange(B, device=t.device)[:, None, None], t // c["page"]]
        t = t % c["page"]
    else:
        slot = torch.arange(B, device=t.device).view(B, 1, 1)
    head = torch.arange(h, device=t.device).view(1, h, 1)
    k, v = st["k"][slot, head, t].float(), st["v"][slot, head, t].float()
    s = st["q"].float().view(B, h, hq // h, d) @ k.transpose(2, 3) / math.sqrt(d)
    s.masked_fill_(~there[:, :, None], -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    return (p @ v / z).view(B, hq, 1, d).to(st["q"].dtype), (m + torch.log(z)).view(B, hq)


# ---- one pass ----------------------------------------------------------------------------------------------

def run(st):
    c = st["case"]
    kind = c["kind"]
    if own:
        from dtorch_amd.nn import functional as F
    if kind == "beam":
        for n in ("table", "lengths", "refs"):  # the tables that this step finds
            st[n].copy_(st[n + "0"])
        if own:
            F.kv_pages_fork(st["table"], st["lengths"], st["refs"], st["parents"])
            short = F.kv_pages_reserve([st["k"], st["v"]], st["table"], st["lengths"], st["refs"], c["n"])
        else:
            _fork_plain(st)
            short = _reserve_plain(st)
        return {n: st[n] for n in ("k", "v", "table", "lengths", "refs")} | {"short": short}
    if kind == "compact":
        for n in ("table", "refs"):
            st[n].copy_(st[n + "0"])
        used = F.kv_pages_compact([st["k"], st["v"]], st["table"], st["refs"]) if own else _compact_plain(st)
        return {n: st[n] for n in ("k", "v", "table", "refs")} | {"used": used}
    if kind == "shared":
        if not own:
            return _shared_plain(st)
        if c["page"]:
            return F.decode_attention_shared_paged(st["q"], st["k"], st["v"], st["table"], st["lengths"], st["prefix"])
        return F.decode_attention_shared(st["q"], st["kp"], st["vp"], st["prefix"], st["k"], st["v"], st["lengths"])
    if kind == "bounds":
        if not own:
            return _bounds_plain(st)
        if c["page"]:
            F.kv_key_bounds_paged(st["k"], st["kmin"], st["kmax"], st["table"], st["lengths"], c["n"])
        else:
            F.kv_key_bounds(st["k"], st["kmin"], st["kmax"], st["lengths"], c["n"])
        return st["kmin"], st["kmax"]
    if not own:
        ids = _select_plain(st)
        return (ids,) + _blocks_plain(st, ids)
    if c["page"]:
        ids = F.select_key_blocks_paged(st["q"], st["kmin"], st["kmax"], st["table"], st["lengths"], c["keep"], c["recent"], c["block"])
        return (ids,) + F.decode_attention_blocks_paged(st["q"], st["k"], st["v"], st["table"], st["lengths"], ids, c["block"])
    ids = F.select_key_blocks(st["q"], st["kmin"], st["kmax"], st["lengths"], c["keep"], c["recent"], c["block"])
    return (ids,) + F.decode_attention_blocks(st["q"], st["k"], st["v"], st["lengths"], ids, c["block"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def _rows64(st, x, b, n, head=None):
    """Rows [Hkv, n, D] (of one kv head: [n, D]) of the first n tokens of sequence b."""
    if "table" not in st:
        return (x[b] if head is None else x[b, head])[..., :n, :].double()
    many = -(-n // x.shape[2])
    pages = x[st["table"][b, :many].long()]  # [pages, Hkv, page, D]
    if head is not None:
        return pages[:, head].double().flatten(0, 1)[:n]
    return pages.double().transpose(0, 1).flatten(1, 2)[:, :n]


def _attention64(q, k, v):
    """q [group, D], k and v [n, D] of one kv head."""
    s = (q @ k.t().contiguous()) * q.shape[-1] ** -0.5
    return torch.softmax(s, -1) @ v, torch.logsumexp(s, -1)


def exact(c, seed):
    kind = c["kind"]
    if kind in ("beam", "compact"):
        return None  # values moved as they are, and whole numbers
    st = prepare(c, seed)
    ns = st["lengths"].tolist()
    if kind == "bounds":
        if c["B"] * (c["n"] // c["block"] + 2) > 6000:
            return None
        lo, hi = st["kmin"].double(), st["kmax"].double()
        for b, n in enumerate(ns):
            x = _rows64(st, st["k"], b, n)
            for j in range((n - c["n"]) // c["block"], -(-n // c["block"])):
                rows = x[:, j * c["block"]:(j + 1) * c["block"]]
                at = (int(st["table"][b, j * c["block"] // c["page"]]), slice(None), j * c["block"] % c["page"] // c["block"]) if c["page"] else (b, slice(None), j)
                lo[at], hi[at] = rows.min(1).values, rows.max(1).values
        return lo, hi
    B, h, d = c["B"], c["Hkv"], c["D"]
    group = c["Hq"] // h
    q = st["q"].double().view(B, h, group, d)
    out = torch.zeros(B, h, group, d, dtype=torch.float64, device="cuda")
    lse = torch.zeros(B, h, group, dtype=torch.float64, device="cuda")
    if B * h > 2000:
        return None
    if kind == "shared":
        prefix = st["prefix"].tolist()
        for b in range(B):
            g = b // (B // c["G"])
            k, v = _rows64(st, st["k"], b, ns[b]), _rows64(st, st["v"], b, ns[b])
            if not c["page"]:
                k = torch.cat([st["kp"][g, :, :prefix[g]].double(), k], 1)
                v = torch.cat([st["vp"][g, :, :prefix[g]].double(), v], 1)
            for i in range(h):
                out[b, i], lse[b, i] = _attention64(q[b, i], k[i], v[i])
        return out.view(B, -1, 1, d), lse.view(B, -1)
    block, keep, recent = c["block"], c["keep"] // c["block"], c["recent"] // c["block"]
    for b, n in enumerate(ns):
        blocks = -(-n // block)
        for i in range(h):
            chosen = list(range(blocks))
            if blocks > keep:
                if c["page"]:
                    ids = st["table"][b].long()
                    lo, hi = (st[x][ids, i].flatten(0, 1)[:blocks - recent].double() for x in ("kmin", "kmax"))
                else:
                    lo, hi = (st[x][b, i, :blocks - recent].double() for x in ("kmin", "kmax"))
                score = torch.stack([torch.maximum(lo * row, hi * row).sum(1) for row in q[b, i]]).max(0).values.float()
                best = torch.sort(score, descending=True, stable=True)[1][:keep - recent]
                chosen = sorted(best.tolist()) + chosen[blocks - recent:]
            at = (torch.tensor(chosen, device="cuda")[:, None] * block + torch.arange(block, device="cuda")).flatten()
            at = at[at < n]
            out[b, i], lse[b, i] = _attention64(q[b, i], _rows64(st, st["k"], b, n, i)[at], _rows64(st, st["v"], b, n, i)[at])
    return None, out.view(B, -1, 1, d), lse.view(B, -1)
