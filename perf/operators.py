"""Performance cases of the 8-bit KV cache and of the bounded one: quantised append, decode attention over 8-bit
codes, accumulated attention weights, and eviction by them, through dtorch_amd.nn.functional.

A case is a dict with a "kind" (the operator), its sizes and its types; `listed()` holds two or more of each
operator, `draw()` gives more over the same ranges.  `run()` computes a case in elementary torch operations, or
with `own` set through the package's operators.  Heads and head dims are those of the models that the package
names (Llama: 32 query / 8 kv heads of 128) and of generic multi-head layers.  Inputs are unit normals, which is
what projections behind a norm layer give; where a layer's channels differ in size (keys do), each channel gets
a size of its own.
"""
import math

import torch

own = False

_DT = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}
_SIZE = {"bf16": 2, "fp16": 2, "fp32": 4, "fp8": 1}
_CODE = torch.float8_e4m3fn


def listed():
    return [
        # one token of one sequence into its 8-bit cache, behind 4000 others
        dict(name="append_token", kind="append", B=1, Hkv=8, n=1, lo=4000, hi=4000, D=128, block=32, page=0, dtype="bf16"),
        # four prompts of 2000 tokens into empty caches
        dict(name="append_prompts", kind="append", B=4, Hkv=8, n=2000, lo=0, hi=0, D=128, block=64, page=0, dtype="bf16"),
        # the next 333 tokens of 16 requests of mixed lengths into 16-token pages
        dict(name="append_pages", kind="append", B=16, Hkv=8, n=333, lo=5, hi=1500, D=128, block=16, page=16, dtype="fp16"),
        # one token's attention over 4000 cached ones (one sequence: latency)
        dict(name="decode_one", kind="decode", B=1, Hq=32, Hkv=8, lo=4000, hi=4000, D=128, block=32, page=0, dtype="bf16"),
        # a serving batch of mixed lengths over 16-token pages
        dict(name="decode_pages", kind="decode", B=64, Hq=32, Hkv=8, lo=512, hi=8192, D=128, block=16, page=16, dtype="bf16"),
        # sixteen long contexts, 64 query heads
        dict(name="decode_long", kind="decode", B=16, Hq=64, Hkv=8, lo=20000, hi=32768, D=128, block=64, page=0, dtype="fp16"),
        # a full-precision multi-head layer over an 8-bit cache
        dict(name="decode_fp32", kind="decode", B=6, Hq=12, Hkv=12, lo=100, hi=2047, D=64, block=32, page=32, dtype="fp32"),
        # weights that the prompts' queries give to each key (causal)
        dict(name="weights_prompts", kind="weights", B=4, Hq=32, Hkv=8, L=2048, lo=2048, hi=2048, D=128, keys="bf16", block=0, dtype="bf16"),
        # one token's weights over a batch of 8-bit caches of mixed lengths
        dict(name="weights_token", kind="weights", B=16, Hq=28, Hkv=4, L=1, lo=700, hi=8191, D=128, keys="fp8", block=32, dtype="bf16"),
        # a right-padded batch of short full-precision prompts
        dict(name="weights_fp32", kind="weights", B=2, Hq=12, Hkv=12, L=777, lo=300, hi=777, D=64, keys="fp32", block=0, dtype="fp32"),
        # half of 4096 tokens of a 16-bit cache, token by token and kv head by kv head
        dict(name="evict_tokens", kind="evict", B=8, Hkv=8, lo=4096, hi=4096, keep=2048, recent=256, D=128, block=1, dtype="bf16"),
        # blocks of 32 tokens of 8-bit caches of mixed lengths
        dict(name="evict_blocks", kind="evict", B=16, Hkv=8, lo=3000, hi=8190, keep=4096, recent=512, D=128, block=32, dtype="fp8"),
    ]


# Rates (operations a second, bytes a second) by which draw() bounds a case's cost; the most it may cost is that of
# the listed long contexts.
_MOST_S = 220e-6


def _cost(c):
    w = work(c)
    rate = 0.05e15 if "fp32" in (c["dtype"], c.get("keys")) else 0.4e15
    return w["flops"] / rate + w["bytes"] / 4.5e12


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def _drawn(rng):
    kind = rng.choice(["append", "decode", "decode", "weights", "weights", "evict"])
    hq, hkv, d = rng.choice([(32, 8, 128), (32, 8, 128), (64, 8, 128), (28, 4, 128), (32, 32, 128), (12, 12, 64), (20, 20, 64), (16, 2, 80)])
    t = rng.choice(["bf16", "bf16", "fp16", "fp32"])
    if kind == "append":
        page = rng.choice([0, 0, 16, 64, 256])
        block = rng.choice([b for b in (16, 32, 64, 128) if page == 0 or b <= page])
        hi = _log(rng, 1, 16384)
        return dict(kind=kind, B=_log(rng, 1, 64), Hkv=hkv, n=rng.choice([1, 1, _log(rng, 2, 4000)]), lo=rng.randint(0, hi), hi=hi, D=d,
                    block=block, page=page, dtype=t)
    if kind == "decode":
        page = rng.choice([0, 0, 16, 32, 256])
        block = rng.choice([b for b in (16, 32, 64, 256) if page == 0 or b <= page])
        hi = _log(rng, 16, 32768)
        return dict(kind=kind, B=_log(rng, 1, 96), Hq=hq, Hkv=hkv, lo=max(1, hi // rng.choice([1, 2, 8, 16])), hi=hi, D=d, block=block, page=page, dtype=t)
    if kind == "weights":
        if rng.random() < 0.5:
            hi = _log(rng, 16, 32768)
            keys = rng.choice([t, "fp8"])
            return dict(kind=kind, B=_log(rng, 1, 64), Hq=hq, Hkv=hkv, L=1, lo=max(1, hi // rng.choice([1, 2, 8])), hi=hi, D=d, keys=keys,
                        block=rng.choice([16, 32, 128]) if keys == "fp8" else 0, dtype=t)
        n = _log(rng, 16, 4096)
        return dict(kind=kind, B=_log(rng, 1, 8), Hq=hq, Hkv=hkv, L=n, lo=rng.choice([n, max(1, n // 3)]), hi=n, D=d, keys=t, block=0, dtype=t)
    t = rng.choice(["bf16", "fp16", "fp32", "fp8"])
    block = rng.choice([16, 32, 64]) if t == "fp8" else rng.choice([1, 1, 1, 8])
    hi = _log(rng, 256, 32768)
    keep = max(2, hi // block // rng.choice([2, 2, 3, 4])) * block
    return dict(kind=kind, B=_log(rng, 1, 32), Hkv=hkv, lo=max(1, hi // rng.choice([1, 1, 2, 4])), hi=hi, keep=keep,
                recent=max(1, keep // block // rng.choice([4, 8])) * block, D=d, block=block, dtype=t)


def draw(rng):
    while True:
        c = _drawn(rng)
        if _cost(c) <= _MOST_S:
            return c


def _lengths(c):
    """Cached tokens of each sequence, spread evenly over [lo, hi]."""
    return [c["hi"] - (c["hi"] - c["lo"]) * i // max(c["B"] - 1, 1) for i in range(c["B"])]


def _room(c):
    """Capacity of each sequence: room for the longest one (and for the new tokens), whole blocks and pages."""
    need = c["hi"] + (c["n"] if c["kind"] == "append" else 0)
    unit = max(c.get("page", 0), c["block"], 64)
    return -(-need // unit) * unit


def work(c):
    d, h, kind = c["D"], c["Hkv"], c["kind"]
    e = _SIZE[c["dtype"]]
    ns = _lengths(c)
    if kind == "append":
        rows = c["B"] * h * c["n"]
        return {"bytes": 2 * rows * d * (e + 1) + 8 * (rows // c["block"] + c["B"] * h) + 8 * c["B"], "flops": 4 * rows * d}
    if kind == "decode":
        tokens = sum(ns)
        data = 2 * tokens * h * d + 8 * h * (tokens // c["block"]) + 2 * c["B"] * c["Hq"] * d * e + 4 * c["B"] * c["Hq"]
        return {"bytes": data, "flops": 4 * tokens * c["Hq"] * d}
    if kind == "weights":
        pairs = sum(ns) if c["L"] == 1 else sum(n * (n + 1) // 2 for n in ns)
        rows = c["B"] if c["L"] == 1 else sum(ns)
        data = sum(ns) * h * (d * _SIZE[c["keys"]] + 8) + rows * c["Hq"] * (d * e + 4)
        return {"bytes": data, "flops": 2 * pairs * c["Hq"] * d}
    moved = sum(c["keep"] for n in ns if n > c["keep"])  # rows read and written, and every weight read
    return {"bytes": 4 * moved * h * d * e + 4 * h * sum(ns) + 8 * h * moved, "flops": h * sum(ns)}


# ---- inputs ------------------------------------------------------------------------------------------------

def _pow2(k):
    return ((k + 127) << 23).to(torch.int32).view(torch.float32)


def _scale_of(amax):
    """The smallest power of two s with amax <= 448 s (at least 2^-126), 1 for amax = 0."""
    m, e = torch.frexp(amax)
    k = torch.where(m <= 0.875, e - 9, e - 8).clamp(min=-126).to(torch.int64)
    return torch.where(amax > 0, _pow2(k), torch.ones_like(amax))


def _encode(x, block):
    """Codes and scales of [..., S, D] values, S a multiple of block."""
    b = x.unflatten(-2, (-1, block))
    s = _scale_of(b.abs().amax((-1, -2)))
    return (b / s[..., None, None]).to(_CODE).flatten(-3, -2), s


def _decoded(codes, scale):
    """[..., S, D] values of codes with a scale for each of scale.shape[-1] equal blocks of rows."""
    block = codes.shape[-2] // scale.shape[-1]
    return codes.float() * scale.repeat_interleave(block, -1)[..., None]


def prepare(c, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    kind, B, h, d = c["kind"], c["B"], c["Hkv"], c["D"]
    st = {"case": c}

    def normal(*shape, t="fp32"):
        return torch.randn(*shape, device="cuda", generator=g).to(_DT[t])

    def sizes():
        return torch.exp(0.5 * normal(h, 1, d))

    order = torch.randperm(B, device="cuda", generator=g)
    st["lengths"] = torch.tensor(_lengths(c), dtype=torch.int32, device="cuda")[order]
    room, page = _room(c), c.get("page", 0)
    if kind in ("append", "decode") or (kind == "weights" and c["keys"] == "fp8"):
        pool = (B * (room // page), h, page, d) if page else (B, h, room, d)
        st["k"], st["ks"] = _encode(normal(*pool) * sizes(), c["block"])
        if kind != "weights":
            st["v"], st["vs"] = _encode(normal(*pool), c["block"])
        if page:
            st["table"] = torch.randperm(pool[0], device="cuda", generator=g).view(B, -1).to(torch.int32)
    if kind == "append":
        st["before"] = st["lengths"].clone()
        st["kn"] = normal(B, c["n"], h, d, t=c["dtype"]).transpose(1, 2) * sizes().to(_DT[c["dtype"]])
        st["vn"] = normal(B, c["n"], h, d, t=c["dtype"]).transpose(1, 2)
    if kind == "decode":
        st["q"] = normal(B, c["Hq"], 1, d, t=c["dtype"])
    if kind == "weights":
        L = c["L"]
        st["q"] = normal(B, c["Hq"], L, d, t=c["dtype"])
        if c["keys"] != "fp8":  # a prompt's keys, or a cache of the longest sequence's capacity
            st["k"] = normal(B, h, L if L > 1 else room, d, t=c["keys"])
        s = _scores(st)
        st["lse"] = torch.logsumexp(s, -1).reshape((B, c["Hq"]) if L == 1 else (B, c["Hq"], L))
        st["weights"] = torch.zeros(B, h, st["k"].shape[2], device="cuda")  # a new request's
    if kind == "evict":
        st["before"] = st["lengths"].clone()
        for n in "kv":
            if c["dtype"] == "fp8":
                st[n], st[n + "s"] = _encode(normal(B, h, room, d), c["block"])
            else:
                st[n] = normal(B, h, room, d, t=c["dtype"])
        # a few tokens collect most of the weight
        st["seen"] = torch.exp(2 * normal(B, h, room))
        st["weights"] = st["seen"].clone()
    return st


# ---- the plain forms ---------------------------------------------------------------------------------------

def _scores(st):
    """Scaled scores [B, Hkv, group, L, S] in 32 bits, -inf where a key is not visible to a query."""
    c = st["case"]
    q, k = st["q"].float(), st["k"]
    k = _decoded(k, st["ks"]) if k.dtype == _CODE else k.float()
    B, hq, L, d = q.shape
    h, S = k.shape[1], k.shape[2]
    s = (q.reshape(B, h, -1, d) @ k.transpose(-1, -2)).view(B, h, hq // h, L, S) / math.sqrt(d)
    at = torch.arange(S, device=q.device)
    n = st["lengths"].long().view(B, 1, 1, 1, 1)
    hidden = at >= n
    if c["L"] > 1:
        hidden = hidden | (at > torch.arange(L, device=q.device)[:, None])
    return s.masked_fill_(hidden, -math.inf)


def _places(st, t):
    """Where token t[b, i] of sequence b lies: the first and third index of a cache."""
    if "table" not in st:
        return torch.arange(t.shape[0], device=t.device)[:, None].expand_as(t), t
    page = st["case"]["page"]
    return st["table"].long().gather(1, t // page), t % page


def _append_plain(st, codes, scale, new):
    """New tokens behind the cached ones of each sequence, through the rows of the blocks they touch."""
    c = st["case"]
    block, n = c["block"], c["n"]
    start, room = st["lengths"].clamp(min=0).long(), _room(c)
    rows = min(((n + block - 1) // block + 1) * block, room)
    first = torch.minimum(start // block * block, start.new_full((), room - rows))
    t = first[:, None] + torch.arange(rows, device=start.device)
    j = t - start[:, None]
    fresh, old = (j >= 0) & (j < n), j < 0
    p, r = _places(st, t)
    bits = codes.view(torch.uint8)
    was = bits[p, :, r]  # [B, rows, Hkv, D]
    tp, tr = p[:, ::block], r[:, ::block] // block
    s0 = scale[tp, :, tr]  # [B, blocks, Hkv]
    x = new.float().transpose(1, 2).gather(1, j.clamp(0, n - 1)[:, :, None, None].expand(-1, -1, *was.shape[2:]))
    x = x * fresh[:, :, None, None]
    need = _scale_of(x.abs().unflatten(1, (-1, block)).amax((2, 4)))
    s1 = torch.where(old[:, ::block, None], torch.maximum(s0, need), need)
    s1 = torch.where(fresh.unflatten(1, (-1, block)).any(2)[..., None], s1, s0)
    x = torch.where(fresh[:, :, None, None], x, was.view(_CODE).float() * s0.repeat_interleave(block, 1)[..., None])
    now = (x / s1.repeat_interleave(block, 1)[..., None]).to(_CODE).view(torch.uint8)
    bits[p, :, r] = torch.where((fresh | old)[:, :, None, None], now, was)
    scale[tp, :, tr] = s1


def _gathered(st, codes, scale):
    """[B, Hkv, S, D] values of a padded or paged cache."""
    if "table" not in st:
        return _decoded(codes, scale)
    ids = st["table"].long()
    return _decoded(codes.view(torch.uint8)[ids].view(_CODE), scale[ids]).transpose(1, 2).flatten(2, 3)


def _decode_plain(st):
    k, v = _gathered(st, st["k"], st["ks"]), _gathered(st, st["v"], st["vs"])
    q = st["q"].float()
    B, hq, _, d = q.shape
    s = q.view(B, k.shape[1], -1, d) @ k.transpose(-1, -2) / math.sqrt(d)
    s.masked_fill_(torch.arange(k.shape[2], device=q.device) >= st["lengths"].view(-1, 1, 1, 1), -math.inf)
    m = s.amax(-1, keepdim=True)
    p = torch.exp(s - m)
    z = p.sum(-1, keepdim=True)
    o = p @ v / z
    return o.view(B, hq, 1, d).to(st["q"].dtype), (m + torch.log(z)).view(B, hq)


def _weights_plain(st):
    c, s = st["case"], _scores(st)
    lse = st["lse"].view(s.shape[:4] + (1,))
    p = torch.exp(s - lse)
    if c["L"] > 1:  # queries past the prompt's end are padding
        p *= (torch.arange(c["L"], device=p.device) < st["lengths"].view(-1, 1)).view(c["B"], 1, 1, -1, 1)
    st["weights"] += p.sum((2, 3))
    return st["weights"]


def _evict_plain(st):
    c = st["case"]
    B, h, block = c["B"], c["Hkv"], c["block"]
    n, w = st["lengths"].long(), st["weights"]
    keep, recent = c["keep"] // block, c["recent"] // block
    blocks = (n + block - 1) // block
    evicts = blocks > keep
    at = torch.arange(w.shape[2], device=w.device)
    mass = (w * (at < n.view(-1, 1, 1))).double().unflatten(2, (-1, block)).sum(-1).float()  # [B, Hkv, all blocks]
    bt = torch.arange(mass.shape[2], device=w.device)
    old = bt < (blocks - recent)[:, None]  # candidates
    mass = torch.where(old[:, None], mass, torch.full_like(mass, -math.inf))
    rank = torch.argsort(torch.argsort(mass, dim=-1, descending=True, stable=True), dim=-1)
    stays = torch.where(old, False, bt < blocks[:, None])[:, None] | (old[:, None] & (rank < keep - recent))
    stays = torch.where(evicts[:, None, None], stays, (bt < blocks[:, None])[:, None])
    kept = torch.argsort((~stays).to(torch.uint8), dim=-1, stable=True)  # those that stay, in order, then the others
    left = torch.where(evicts, (keep - 1) * block + n - (blocks - 1) * block, n)
    source = (kept[..., None] * block + torch.arange(block, device=w.device)).flatten(2)
    inside = at < left[:, None, None]
    for name in ("k", "v"):
        x = st[name]
        bits = x.view(torch.uint8) if x.dtype == _CODE else x
        moved = bits.gather(2, source[..., None].expand(-1, -1, -1, bits.shape[3]))
        bits.copy_(torch.where(inside[..., None], moved, bits))
        if x.dtype == _CODE:
            s = st[name + "s"]
            s.copy_(torch.where(bt < torch.minimum(blocks, blocks.new_full((), keep))[:, None, None], s.gather(2, kept), s))
    w.copy_(torch.where(inside, w.gather(2, source), torch.where(at < n.view(-1, 1, 1), torch.zeros_like(w), w)))
    st["lengths"].copy_(left)
    first = kept if kept.shape[2] >= keep else torch.nn.functional.pad(kept, (0, keep - kept.shape[2]))
    first = first[..., :keep]
    return torch.where(torch.arange(keep, device=w.device) < blocks[:, None, None], first, -1).to(torch.int32)


# ---- one pass ----------------------------------------------------------------------------------------------

def run(st):
    c = st["case"]
    kind = c["kind"]
    if own:
        from dtorch_amd.nn import functional as F
    if kind == "append":
        st["lengths"].copy_(st["before"])  # the scheduler's lengths of this step
        if not own:
            _append_plain(st, st["k"], st["ks"], st["kn"])
            _append_plain(st, st["v"], st["vs"], st["vn"])
            st["lengths"].copy_((st["lengths"].clamp(min=0) + c["n"]).clamp(max=_room(c)))
        elif c["page"]:
            F.kv_cache_append_fp8_paged(st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lengths"], st["kn"], st["vn"])
        else:
            F.kv_cache_append_fp8(st["k"], st["v"], st["ks"], st["vs"], st["lengths"], st["kn"], st["vn"])
        return st["k"], st["v"], st["ks"], st["vs"], st["lengths"]
    if kind == "decode":
        if not own:
            return _decode_plain(st)
        if c["page"]:
            return F.decode_attention_fp8_paged(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["table"], st["lengths"])
        return F.decode_attention_fp8(st["q"], st["k"], st["v"], st["ks"], st["vs"], st["lengths"])
    if kind == "weights":
        if not own:
            return _weights_plain(st)
        return F.attention_weight_accumulate(st["weights"], st["q"], st["k"], st["lse"], lengths=st["lengths"], is_causal=c["L"] > 1,
                                             key_scale=st.get("ks"))
    st["lengths"].copy_(st["before"])  # another sequence of the same length with the same weights
    st["weights"].copy_(st["seen"])
    if own:
        kept = F.kv_cache_evict(st["k"], st["v"], st["lengths"], st["weights"], c["keep"], c["recent"], block=c["block"],
                                k_scale=st.get("ks"), v_scale=st.get("vs"))
    else:
        kept = _evict_plain(st)
    return {n: st[n] for n in ("k", "v", "ks", "vs", "weights", "lengths") if n in st} | {"kept": kept}


# ---- the definitions in 64 bits ----------------------------------------------------------------------------

def _rows64(codes, scale, st, b, n):
    """Values [Hkv, n, D] of the first n tokens of sequence b."""
    if "table" in st:
        ids = st["table"][b].long()
        x = codes.view(torch.uint8)[ids].view(_CODE).double()  # [pages, Hkv, page, D]
        s = scale[ids].double()
        x = x * s.repeat_interleave(x.shape[2] // s.shape[2], 2)[..., None]
        return x.permute(1, 0, 2, 3).reshape(x.shape[1], -1, x.shape[3])[:, :n]
    if scale is None:
        return codes[b, :, :n].double()
    block = codes.shape[2] // scale.shape[2]
    at = torch.arange(n, device=codes.device) // block
    return codes[b, :, :n].double() * scale[b].double()[:, at, None]


def _append64(st, codes, scale, new):
    c = st["case"]
    block, page = c["block"], c["page"]
    values, scales = codes.double(), scale.double()
    starts = st["before"].tolist()
    for b in range(c["B"]):
        x = new[b].double()  # [Hkv, n, D]
        t, end = starts[b], starts[b] + c["n"]
        while t < end:
            t0 = t // block * block
            stop = min(end, t0 + block)
            p, r0 = (int(st["table"][b, t0 // page]), t0 % page) if page else (b, t0)
            part = x[:, t - starts[b]:stop - starts[b]]
            top = part.abs().amax((1, 2))
            need = torch.exp2(torch.ceil(torch.log2(top / 448)).clamp(min=-126))
            need = torch.where(need / 2 * 448 >= top, need / 2, need)
            s = torch.where(top > 0, need, torch.ones_like(need))
            if t > t0:
                s = torch.maximum(s, scales[p, :, r0 // block])
                before = values[p, :, r0:r0 + t - t0] * scales[p, :, r0 // block][:, None, None]
                values[p, :, r0:r0 + t - t0] = (before / s[:, None, None]).float().to(_CODE).double()
            values[p, :, r0 + t - t0:r0 + stop - t0] = (part / s[:, None, None]).float().to(_CODE).double()
            scales[p, :, r0 // block] = s
            t = stop
    return values, scales


def exact(c, seed):
    st = prepare(c, seed)
    ns, kind = st["lengths"].tolist(), c["kind"]
    if kind == "append":
        if c["B"] * (c["n"] // c["block"] + 1) > 4000:
            return None
        (k, ks), (v, vs) = _append64(st, st["k"], st["ks"], st["kn"]), _append64(st, st["v"], st["vs"], st["vn"])
        return k, v, ks, vs, None
    if kind == "decode":
        os, ls = [], []
        for b in range(c["B"]):
            k, v = _rows64(st["k"], st["ks"], st, b, ns[b]), _rows64(st["v"], st["vs"], st, b, ns[b])
            s = (st["q"][b, :, 0].double().view(k.shape[0], -1, c["D"]) @ k.transpose(1, 2).contiguous()) * c["D"] ** -0.5
            os.append((torch.softmax(s, -1) @ v).reshape(c["Hq"], 1, c["D"]))
            ls.append(torch.logsumexp(s, -1).reshape(c["Hq"]))
        return torch.stack(os), torch.stack(ls)
    if kind == "weights":
        w = st["weights"].double()
        group = c["Hq"] // c["Hkv"]
        for b in range(c["B"]):
            n = ns[b]
            k = _rows64(st["k"], st.get("ks"), st, b, n)
            for hq in range(c["Hq"]):
                q = st["q"][b, hq, :n].double()
                lse = st["lse"][b, hq].double().reshape(-1, 1)[:n]
                p = torch.exp(q @ k[hq // group].t().contiguous() * c["D"] ** -0.5 - lse)
                w[b, hq // group, :n] += (torch.tril(p) if c["L"] > 1 else p).sum(0)
        return w
    if st["k"].numel() > 2e8:
        return None
    # the definition, one kv head of one sequence after another
    block, keep, recent = c["block"], c["keep"] // c["block"], c["recent"] // c["block"]
    out = {n: st[n].double() for n in ("k", "v", "ks", "vs", "weights") if n in st}
    for b in range(c["B"]):
        n = ns[b]
        blocks = -(-n // block)
        if blocks <= keep:
            continue
        for h in range(c["Hkv"]):
            old = (blocks - recent) * block
            mass = st["weights"][b, h, :old].double().view(-1, block).sum(1).float()
            chosen = torch.sort(mass, descending=True, stable=True)[1][:keep - recent].sort()[0].tolist()
            chosen += range(blocks - recent, blocks)
            at = torch.cat([torch.arange(i * block, min((i + 1) * block, n)) for i in chosen]).cuda()
            for name, x in out.items():
                if name in ("ks", "vs"):
                    x[b, h, :keep] = x[b, h, torch.tensor(chosen, device="cuda")]
                else:
                    x[b, h, :len(at)] = x[b, h, at]
            out["weights"][b, h, len(at):n] = 0
    return out | {"lengths": None, "kept": None}
