"""The 8-bit and the bounded KV cache as they are used: generation loops of the cache classes with everything together, graph
capture, concurrent streams, and what the operators refuse.

The loops follow the device exactly where the result is exact (codes, scales, lengths, what an eviction keeps, which is decided
on the device's own weights) and by bounds elsewhere.  Outputs: 16-bit queries round P and O (half a step u each, relative to
A = softmax |V| and |O|); scores are fp32 sums of D products, and sums over n tokens add (n + 64) e A, e = 2^-24.  Weights of one
step: relative (2 (3 D + 8) e M + 8 e |lse| + (n + 16) e) of each term, M = max sum |q_d k_d| scale; the bound of a sum over steps is the
sum of the steps' bounds and half an fp32 step of the running sum for each."""
import threading

import numpy as np
import pytest
import torch

from oracle import cache as orc

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
U = {torch.bfloat16: 2.0 ** -8, torch.float16: 2.0 ** -11, torch.float32: E}
CODES = torch.float8_e4m3fn


def _F():
    import dtorch_amd.nn.functional as F
    return F


class _Mirror:
    """A padded cache in NumPy: what the loop should hold."""

    def __init__(self, cache, block):
        self.cache, self.block = cache, block
        B, H, S, D = cache.k.shape
        self.n = np.zeros(B, np.int64)
        self.codes = cache.k_scale is not None
        self.k, self.v = (np.zeros((B, H, S, D), np.uint8 if self.codes else np.float64) for _ in range(2))
        self.ks, self.vs = (np.ones((B, H, S // block if self.codes else 1), np.float32) for _ in range(2))
        self.w, self.err = np.zeros((B, H, S)), np.zeros((B, H, S))

    def append(self, k, v):
        for c, s, x in ((self.k, self.ks, k), (self.v, self.vs, v)):
            x = x.double().cpu().numpy()
            if self.codes:
                orc.append_fp8(c, s, None, self.n, x, self.block)
            else:
                for b in range(len(self.n)):
                    c[b, :, self.n[b]:self.n[b] + x.shape[2]] = x[b]
        self.n += k.shape[2]

    def values(self):
        if not self.codes:
            return self.k, self.v
        return orc.values(self.k, self.ks), orc.values(self.v, self.vs)

    def accumulate(self, q, k, causal):
        """q [B, Hq, L, D], k [B, Hkv, S, D] float64 over the first n of each."""
        B, hq, L, D = q.shape
        g, sc = hq // k.shape[1], D ** -0.5
        for b in range(B):
            n = int(self.n[b])
            for h in range(hq):
                s = q[b, h] @ k[b, h // g, :n].T * sc
                if causal:
                    s[np.triu_indices(L, 1, n)] = -np.inf
                m = s.max(-1, keepdims=True)
                lse = m + np.log(np.exp(s - m).sum(-1, keepdims=True))
                p = np.exp(s - lse)
                mag = (np.abs(q[b, h]) @ np.abs(k[b, h // g, :n]).T).max() * sc
                self.w[b, h // g, :n] += p.sum(0)
                self.err[b, h // g, :n] += p.sum(0) * (2 * (3 * D + 8) * mag + 8 * np.abs(lse).max() + n + L + 16) * E
        self.err += self.w * E

    def check_state(self):
        c = self.cache
        assert c.lengths.tolist() == self.n.tolist() and c._host_len.tolist() == self.n.tolist()
        for b, n in enumerate(self.n):
            for dev, want in ((c.k, self.k), (c.v, self.v)):
                got = dev[b, :, :n]
                got = got.view(torch.uint8).cpu().numpy() if self.codes else got.double().cpu().numpy()
                assert np.array_equal(got, want[b, :, :n])
            if self.codes:
                blocks = -(-int(n) // self.block)
                for dev, want in ((c.k_scale, self.ks), (c.v_scale, self.vs)):
                    assert np.array_equal(dev[b, :, :blocks].cpu().numpy(), want[b, :, :blocks])
        if c.weights is not None:
            assert (np.abs(c.weights.double().cpu().numpy() - self.w) <= self.err).all()
            assert (self.w == 0)[..., int(self.n.max()):].all() and (c.weights[..., int(self.n.max()):] == 0).all()

    def evict(self, kept, keep, recent):
        """By the device's weights, taken before the call."""
        w = self.before.copy()
        n = self.n.copy()
        scales = [self.ks, self.vs] if self.codes else []
        want = orc.evict([self.k, self.v, self.w, self.err], scales, w, n, keep, recent, self.block, self.block)
        assert np.array_equal(kept.cpu().numpy(), want)
        for b in range(len(n)):
            if n[b] != self.n[b]:
                self.w[b, :, n[b]:self.n[b]] = 0
                self.err[b, :, n[b]:self.n[b]] = 0
        self.n = n


def _check_out(out, q, k, v, n, dtype):
    """One query per sequence."""
    B, hq, _, D = q.shape
    g, u, sc = hq // k.shape[1], U[dtype], D ** -0.5
    for b in range(B):
        for h in range(hq):
            o, lse, a = orc.attend(q[b, h], k[b, h // g, :n[b]], v[b, h // g, :n[b]], sc)
            mag = (np.abs(q[b, h]) @ np.abs(k[b, h // g, :n[b]]).T).max() * sc
            tol = (u + (2 * (3 * D + 8) * mag + n[b] + 64) * E) * a + u * np.abs(o) + 2.0 ** -24 * np.abs(v[b, h // g, :n[b]]).max()
            assert (np.abs(out[b, h].double().cpu().numpy() - o) <= tol).all(), (b, h)


@pytest.mark.parametrize("dtype,codes,block,Hq,Hkv,D", [(torch.bfloat16, True, 32, 8, 2, 128), (torch.float16, True, 16, 6, 6, 64),
                                                        (torch.float32, True, 16, 4, 1, 80), (torch.bfloat16, False, 1, 8, 2, 128),
                                                        (torch.float32, False, 1, 3, 3, 64)])
def test_bounded_generation(dtype, codes, block, Hq, Hkv, D):
    """Prompt, steps, an eviction whenever the cache is full, more steps: more tokens than the cache holds."""
    from dtorch_amd.nn.kv_cache import KVCache
    g = torch.Generator(device="cuda").manual_seed(3)
    B, prompt, cap = 2, 40, 96
    r = lambda h, n: torch.randn(B, n, h, D, device="cuda", generator=g).to(dtype).transpose(1, 2)
    cache = KVCache(B, Hkv, cap, D, dtype=CODES if codes else dtype, block=block, track_weights=True)
    m = _Mirror(cache, block)
    q, k, v = r(Hq, prompt), r(Hkv, prompt), r(Hkv, prompt)
    out = cache.prefill(q, k, v)
    assert torch.equal(out, _F().scaled_dot_product_attention(q, k, v, is_causal=True, enable_gqa=True))
    m.append(k, v)
    m.accumulate(q.double().cpu().numpy(), k.double().cpu().numpy(), True)
    m.check_state()
    evictions = 0
    for step in range(150):
        if m.n.max() == cache.capacity:
            m.before = cache.weights.cpu().numpy()
            m.evict(cache.evict(64, 32), 64, 32)
            m.check_state()
            evictions += 1
        q, k, v = r(Hq, 1), r(Hkv, 1), r(Hkv, 1)
        out = cache.decode(q, k, v)
        m.append(k, v)
        kv, vv = m.values()
        qd = q.double().cpu().numpy()
        m.accumulate(qd, kv, False)
        if step % 7 == 0:
            _check_out(out, qd, kv, vv, m.n, dtype)
    m.check_state()
    assert evictions >= 3


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_paged_generation_over_codes(dtype):
    """Two sequences whose values grow step by step, so that blocks outgrow their scales.

    What is held: half a step of a code, 2^-4 of the value, or 2^-10 of the scale below the normals; every growth of the scale after
    which a code is subnormal adds half a step of that scale, and scales at least double, so all is below 3 of the last scale's."""
    from dtorch_amd.nn.kv_cache import PagedKVCache
    g = torch.Generator(device="cuda").manual_seed(5)
    B, Hq, Hkv, D, page = 2, 8, 2, 64, 32
    r = lambda h, n, mul=1.0: (mul * torch.randn(B, n, h, D, device="cuda", generator=g)).to(dtype).transpose(1, 2)
    cache = PagedKVCache(B, Hkv, 9, page, 4, D, dtype=CODES, block=16)
    held = [[np.zeros((Hkv, 0, D)) for _ in range(2)] for _ in range(B)]
    for step in range(60):
        n = 33 if step == 0 else 1
        mul = 2.0 ** (step % 5)  # scales that grow inside a block
        k, v = r(Hkv, n, mul), r(Hkv, n, mul)
        q = r(Hq, 1, 0.25)
        if n > 1:
            cache.append(k, v)
        else:
            out = cache.decode(q, k, v)
        for b in range(B):
            for i, x in enumerate((k, v)):
                held[b][i] = np.concatenate([held[b][i], x[b].double().cpu().numpy()], 1)
        if n == 1 and step % 5 == 4:
            table = cache.block_table.cpu().numpy()
            kc, vc = (t.view(torch.uint8).cpu().numpy() for t in (cache.k, cache.v))
            ks, vs = cache.k_scale.cpu().numpy(), cache.v_scale.cpu().numpy()
            ln = [x[0].shape[1] for x in held]
            assert cache.lengths.tolist() == ln
            for b in range(B):
                kv, vv = orc.values(kc, ks, table, b, ln[b]), orc.values(vc, vs, table, b, ln[b])
                for have, want, s, codes in ((kv, held[b][0], ks, kc), (vv, held[b][1], vs, vc)):
                    t = np.arange(ln[b])
                    sc = s[table[b, t // page], :, t % page // 16].T[..., None].astype(np.float64)
                    assert (np.abs(have - want) <= np.maximum(np.abs(want) * 2.0 ** -4, sc * 2.0 ** -10 * 3)).all()
                _check_out(out[b:b + 1], q[b:b + 1].double().cpu().numpy(), kv[None], vv[None], [ln[b]], dtype)


CASES = ["append", "append_pages", "decode", "decode_pages", "weights", "weights_prompt", "weights_parts", "evict", "evict_codes", "evict_long"]


def _case(name, seed):
    """(inputs of one call, the call on such tensors: it returns new tensors only)."""
    F = _F()
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s, dtype=torch.bfloat16: torch.randn(*s, device="cuda", generator=g).to(dtype)
    ints = lambda lo, hi, *s, dtype=torch.int32: torch.randint(lo, hi, s, device="cuda", generator=g, dtype=dtype)
    B, Hq, Hkv, S, D, block = 6, 8, 2, 512, 128, 32
    codes = lambda *s: ints(0, 127, *s, dtype=torch.uint8)
    scale = lambda *s: torch.exp2(ints(-8, 2, *s).float())
    as8 = lambda *x: [t.view(CODES) for t in x]
    if name.startswith("append"):
        n = 1 if name == "append" else 70
        x = [codes(B, Hkv, S, D), codes(B, Hkv, S, D), scale(B, Hkv, S // block), scale(B, Hkv, S // block), ints(0, S - n, B),
             r(B, Hkv, n, D), r(B, Hkv, n, D)]
        if name == "append":
            def call(*x):
                y = [t.clone() for t in x[:5]]
                F.kv_cache_append_fp8(*as8(*y[:2]), *y[2:], *x[5:])
                return y
            return x, call
        page = 64
        table = torch.randperm(B * S // page, device="cuda", generator=g).view(B, -1).int()
        x = [codes(B * S // page, Hkv, page, D), codes(B * S // page, Hkv, page, D), scale(B * S // page, Hkv, page // block),
             scale(B * S // page, Hkv, page // block), table] + x[4:]

        def call(*x):
            y = [t.clone() for t in x[:4]] + [x[5].clone()]
            F.kv_cache_append_fp8_paged(*as8(*y[:2]), *y[2:4], x[4], y[4], *x[6:])
            return y
        return x, call
    if name.startswith("decode"):
        q, ln = r(B, Hq, 1, D), ints(0, S + 1, B)
        if name == "decode":
            x = [q, codes(B, Hkv, S, D), codes(B, Hkv, S, D), scale(B, Hkv, S // block), scale(B, Hkv, S // block), ln]
            return x, lambda q, k, v, *a: F.decode_attention_fp8(q, *as8(k, v), *a)
        table = torch.randperm(B * S // 16, device="cuda", generator=g).view(B, -1).int()
        P = B * S // 16
        x = [q, codes(P, Hkv, 16, D), codes(P, Hkv, 16, D), scale(P, Hkv, 1), scale(P, Hkv, 1), table, ln]
        return x, lambda q, k, v, *a: F.decode_attention_fp8_paged(q, *as8(k, v), *a)
    if name.startswith("weights"):
        w, ln = torch.rand(B, Hkv, S, device="cuda", generator=g), ints(0, S + 1, B)
        if name == "weights":
            x = [w, r(B, Hq, 1, D), r(B, Hkv, S, D), r(B, Hq, 1, dtype=torch.float32) + 8, ln]
            return x, lambda w, q, k, l, n: (F.attention_weight_accumulate(w.clone(), q, k, l, lengths=n),)
        L = 40 if name == "weights_prompt" else 700
        x = [w[:1] if L == 700 else w, r(B, Hq, L, D), r(B, Hkv, S, D), r(B, Hq, L, dtype=torch.float32) + 8, ln]
        if L == 700:  # few sequences: the queries are cut in parts that meet in the workspace
            x = [t[:1].contiguous() for t in x]
        return x, lambda w, q, k, l, n: (F.attention_weight_accumulate(w.clone(), q, k, l, lengths=n, is_causal=True),)
    S = 20000 if name == "evict_long" else S
    B = 2 if name == "evict_long" else B
    x = [codes(B, Hkv, S, D), codes(B, Hkv, S, D), ints(0, S + 1, B), torch.rand(B, Hkv, S, device="cuda", generator=g)]
    if name == "evict_codes":
        x += [scale(B, Hkv, S // block), scale(B, Hkv, S // block)]

    def call(*x):
        y = [t.clone() for t in x]
        if name == "evict_codes":
            k = F.kv_cache_evict(*as8(*y[:2]), *y[2:4], 128, 64, k_scale=y[4], v_scale=y[5])
        else:
            k = F.kv_cache_evict(*(t.view(torch.bfloat16) for t in y[:2]), *y[2:4], 100, 30)
        return y + [k]
    return x, call


def _equal(got, want):
    return len(got) == len(want) and all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("name", CASES)
def test_graph_replays_match_eager(name):
    """Two graphs captured of one call, replayed in turn with eager calls between."""
    inputs = [_case(name, 10 + i)[0] for i in range(3)]
    static, call = _case(name, 9)
    ref = [tuple(t.clone() for t in call(*x)) for x in inputs]
    torch.cuda.synchronize()
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = call(*static)
        graphs.append((graph, out))
    torch.cuda.synchronize()
    for n in (0, 1, 2, 0):
        for dst, src in zip(static, inputs[n]):
            dst.copy_(src)
        for graph, _ in graphs:
            graph.replay()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert _equal(out, ref[n]), (name, n)
        torch.ones(1000, device="cuda").sum().item()  # eager work between the replays
        assert _equal(call(*inputs[1]), ref[1])


def test_concurrent_streams_match_serial():
    work = [_case(name, 20 + i) for i, name in enumerate(CASES)]
    serial = [tuple(t.clone() for t in call(*x)) for x, call in work]
    torch.cuda.synchronize()
    results, errors = [None] * 4, []
    start = threading.Barrier(4)

    def worker(i):
        try:
            s = torch.cuda.Stream()  # default priority
            with torch.cuda.stream(s):
                start.wait()
                for _ in range(4):
                    got = [call(*x) for x, call in work[i:] + work[:i]]
                s.synchronize()
                results[i] = got
        except Exception as e:  # surfaced in the main thread
            errors.append((i, repr(e)))

    threads = [threading.Thread(target=worker, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=60)
    assert not any(t.is_alive() for t in threads) and not errors, errors
    torch.cuda.synchronize()
    for i, got in enumerate(results):
        for o, want in zip(got, serial[i:] + serial[:i]):
            assert _equal(o, want), i


def test_captured_steps_and_evictions():
    """Eight replays of four decode steps and an eviction are what the eager calls do."""
    from dtorch_amd.nn.kv_cache import KVCache
    g = torch.Generator(device="cuda").manual_seed(8)
    B, Hq, Hkv, D = 2, 8, 2, 64
    r = lambda h, n: torch.randn(B, h, n, D, device="cuda", generator=g).to(torch.bfloat16)
    prompt = [r(Hq, 48), r(Hkv, 48), r(Hkv, 48)]
    steps = [[r(Hq, 4), r(Hkv, 4), r(Hkv, 4)] for _ in range(9)]

    def four(c, q, k, v):
        out = [c.decode(q[:, :, i:i + 1].contiguous(), k[:, :, i:i + 1], v[:, :, i:i + 1]) for i in range(4)]
        return out, c.evict(48, 16)

    caches = [KVCache(B, Hkv, 96, D, dtype=CODES, block=16, track_weights=True) for _ in range(2)]
    for c in caches:
        c.prefill(*prompt)
        four(c, *steps[0])
    eager, c = caches
    static = [x.clone() for x in steps[0]]
    keep = [t.clone() for t in (c.k, c.v, c.k_scale, c.v_scale, c.weights, c.lengths)]
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out, kept = four(c, *static)
    torch.cuda.synchronize()
    for dst, src in zip((c.k, c.v, c.k_scale, c.v_scale, c.weights, c.lengths), keep):
        assert torch.equal(dst.view(torch.uint8) if dst.dtype == CODES else dst, src.view(torch.uint8) if src.dtype == CODES else src)
    for x in steps[1:]:
        for dst, src in zip(static, x):
            dst.copy_(src)
        graph.replay()
        torch.cuda.synchronize()
        want, want_kept = four(eager, *x)
        # (the captured step covers the whole capacity, so its sums are cut elsewhere: outputs by rounding, state exactly)
        assert torch.equal(kept, want_kept)
        for a, b in zip(out, want):
            assert (a.float() - b.float()).abs().max() <= 2.0 ** -7 * b.float().abs().max()
    want = eager._host_len.tolist()
    assert c.sync_lengths().tolist() == eager.sync_lengths().tolist() == want
    for a, b in ((c.k, eager.k), (c.v, eager.v)):
        assert torch.equal(a[:, :, :want[0]].contiguous().view(torch.uint8), b[:, :, :want[0]].contiguous().view(torch.uint8))


def test_lengths_cut_by_the_caller():
    """A caller that takes tokens back: sync_lengths clears their weights, and the next tokens start from none."""
    from dtorch_amd.nn.kv_cache import KVCache
    x = torch.randn(1, 2, 20, 64, device="cuda").bfloat16()
    c = KVCache(1, 2, 64, 64, track_weights=True)
    c.prefill(x, x, x)
    assert (c.weights[..., :20] > 0).all()
    c.lengths.fill_(12)
    assert c.sync_lengths().tolist() == [12]
    assert (c.weights[..., :12] > 0).all() and (c.weights[..., 12:] == 0).all()


def _refusal_inputs():
    z = lambda *s, dtype=torch.bfloat16: torch.zeros(*s, device="cuda", dtype=dtype)
    k = lambda: z(2, 2, 64, 64, dtype=torch.uint8).view(CODES)
    return dict(k=k(), v=k(), ks=torch.ones(2, 2, 2, device="cuda"), vs=torch.ones(2, 2, 2, device="cuda"),
                n=z(2, dtype=torch.int32), kn=z(2, 2, 3, 64), vn=z(2, 2, 3, 64), q=z(2, 4, 1, 64), w=z(2, 2, 64, dtype=torch.float32),
                lse=z(2, 4, dtype=torch.float32), k16=z(2, 2, 64, 64), v16=z(2, 2, 64, 64))


CALLS = {
    "append": lambda F, i: F.kv_cache_append_fp8(i["k"], i["v"], i["ks"], i["vs"], i["n"], i["kn"], i["vn"]),
    "decode": lambda F, i: F.decode_attention_fp8(i["q"], i["k"], i["v"], i["ks"], i["vs"], i["n"]),
    "weights": lambda F, i: F.attention_weight_accumulate(i["w"], i["q"], i["k16"], i["lse"]),
    "weights8": lambda F, i: F.attention_weight_accumulate(i["w"], i["q"], i["k"], i["lse"], key_scale=i["ks"]),
    "evict": lambda F, i: F.kv_cache_evict(i["k16"], i["v16"], i["n"], i["w"], 16, 4),
    "evict8": lambda F, i: F.kv_cache_evict(i["k"], i["v"], i["n"], i["w"], 32, 32, k_scale=i["ks"], v_scale=i["vs"]),
}


@pytest.mark.parametrize("call", list(CALLS))
def test_calls_that_are_refused_below_are_right_otherwise(call):
    CALLS[call](_F(), _refusal_inputs())


@pytest.mark.parametrize("calls,name,change,text", [
    ("append decode evict8", "k", lambda i: i["k16"], "differ|float8"),
    ("append decode evict8", "v", lambda i: i["v"][:, :, :32], "differ"),
    ("append decode evict8", "ks", lambda i: i["ks"].double(), "fp32"),
    ("append decode evict8", "ks", lambda i: i["ks"][:, :1], "same shape"),
    ("append decode evict8", "ks vs", lambda i: i["ks"][:, :1], "do not match"),
    ("append decode evict8", "ks vs", lambda i: torch.ones(2, 2, 3, device="cuda"), "whole number"),
    ("append decode", "ks vs", lambda i: torch.ones(2, 2, 8, device="cuda"), "block 8"),
    ("append decode", "ks vs", lambda i: torch.ones(2, 2, 4, device="cuda")[..., ::2], "unit stride"),
    ("append evict8", "k", lambda i: i["k"][:1].expand(2, 2, 64, 64), "expanded"),
    ("append evict8", "vs", lambda i: i["vs"][:1].expand(2, 2, 2), "expanded"),
    ("append", "v", lambda i: i["k"], "share memory"), ("evict8", "v", lambda i: i["k"], "share memory"),
    ("evict", "v16", lambda i: i["k16"], "share memory"), ("evict8", "vs", lambda i: i["ks"], "share memory"),
    ("append decode evict evict8", "n", lambda i: i["n"].long(), "int32"),
    ("append decode evict evict8", "n", lambda i: i["n"][:1], "lengths"),
    ("append", "kn", lambda i: i["kn"].half(), "bf16, fp16 or fp32|both"), ("append", "kn vn", lambda i: i["kn"].double(), "bf16, fp16 or fp32"),
    ("append", "kn vn", lambda i: i["kn"][..., :32], "matching the cache"), ("append", "vn", lambda i: i["vn"][:, :, :2], "same shape"),
    ("decode", "q", lambda i: i["q"][:, :3], "multiple"), ("decode", "q", lambda i: i["q"].double(), "bf16, fp16 and fp32"),
    ("decode", "q", lambda i: i["q"].expand(2, 4, 2, 64), "one token"), ("decode weights weights8", "q", lambda i: i["q"][..., :32], "differ|match"),
    ("weights weights8", "q", lambda i: i["q"][:, :3], "multiple"), ("weights", "q", lambda i: i["q"].half(), "query's dtype"),
    ("weights weights8", "w", lambda i: i["w"].double(), "fp32"), ("weights weights8 evict", "w", lambda i: i["w"][..., :32], "shape"),
    ("weights weights8 evict", "w", lambda i: i["w"][:, :1].expand(2, 2, 64), "expanded"),
    ("weights evict", "w", lambda i: torch.zeros(2, 2, 128, device="cuda")[..., ::2], "unit stride"),
    ("weights weights8", "lse", lambda i: i["lse"][:, :2], "lse"), ("weights", "lse", lambda i: i["lse"].half(), "lse"),
    ("weights8", "ks", lambda i: None, "key_scale"), ("weights8", "ks", lambda i: i["ks"][:, :1], "key_scale"),
    ("evict8", "ks vs", lambda i: None, "float8_e4m3fn with"), ("evict8", "ks", lambda i: None, "go together"),
    ("evict", "v16", lambda i: i["v16"].half(), "differ"),
    ("append decode weights evict", "n w", lambda i: {"n": i["n"].cpu(), "w": i["w"].cpu()}, "device"),
])
def test_refusals(calls, name, change, text):
    for call in calls.split():
        i = _refusal_inputs()
        new = change(i)
        for n in name.split():
            i[n] = new[n] if isinstance(new, dict) else (new.clone() if n == "vs" and name == "ks vs" and new is not None and new.is_contiguous() else new)
        with pytest.raises((ValueError, RuntimeError), match=text):
            CALLS[call](_F(), i)


@pytest.mark.parametrize("kw,text", [(dict(keep=0, recent=0), "keep"), (dict(keep=16, recent=0), "recent"), (dict(keep=16, recent=17), "recent"),
                                     (dict(keep=24, recent=16, block=16), "keep"), (dict(keep=16, recent=8, block=16), "recent"),
                                     (dict(keep=1 << 33, recent=4), "keep"), (dict(keep=16, recent=4, block=-1), "block"),
                                     (dict(keep=15, recent=3, block=3), "block 3")])
def test_evict_refusals(kw, text):
    i = _refusal_inputs()
    with pytest.raises((ValueError, RuntimeError), match=text):
        _F().kv_cache_evict(i["k16"], i["v16"], i["n"], i["w"], **kw)


def test_evict_block_below_the_scales():
    i = _refusal_inputs()
    with pytest.raises((ValueError, RuntimeError), match="multiple of"):
        _F().kv_cache_evict(i["k"], i["v"], i["n"], i["w"], 32, 16, block=16, k_scale=i["ks"], v_scale=i["vs"])


@pytest.mark.parametrize("L,Hq,Hkv,D,dtype", [(1, 1, 1, 128, torch.bfloat16), (1, 1, 1, 128, torch.float16), (1, 3, 1, 36, torch.float32),
                                              (3, 3, 3, 80, torch.bfloat16), (3, 3, 3, 80, torch.float16), (50, 3, 1, 96, torch.bfloat16),
                                              (50, 3, 1, 96, torch.float16), (200, 40, 1, 64, torch.bfloat16), (200, 40, 1, 64, torch.float16)])
def test_infinite_keys_of_weight_zero(dtype, L, Hq, Hkv, D):
    """A key whose score is -inf for every query weighs 0, in the padding of head dims and of columns too (fp32 with many
    queries apart: of its three bf16 parts an infinite key's product with a zero one is NaN)."""
    g = torch.Generator(device="cuda").manual_seed(2)
    S = 70
    q = torch.randn(1, Hq, L, D, device="cuda", generator=g).to(dtype)
    k = torch.randn(1, Hkv, S, D, device="cuda", generator=g).to(dtype)
    q[..., 0] = 1.0 + 2.0 ** -7
    k[:, :, 5, 0] = float("-inf")
    s = (q.double() @ k.double().repeat_interleave(Hq // Hkv, 1).transpose(2, 3)) * D ** -0.5
    lse = torch.logsumexp(s, -1).float()
    w = torch.zeros(1, Hkv, S, device="cuda")
    _F().attention_weight_accumulate(w, q, k, lse)
    want = torch.exp(s - lse.double()[..., None]).sum(2).view(1, Hkv, Hq // Hkv, S).sum(2)
    assert (w[:, :, 5] == 0).all() and torch.isfinite(w).all()
    mag = (q.double().abs().sum(-1).max() * 6 * D ** -0.5).item()
    assert ((w.double() - want).abs() <= want * (2 * (2 * D + 8) * mag + 8 * lse.abs().max().item() + L * Hq + 16) * E).all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_empty_shapes(dtype):
    F = _F()
    z = lambda *s, dtype=dtype: torch.zeros(*s, device="cuda", dtype=dtype)
    k0 = z(0, 2, 64, 64, dtype=torch.uint8).view(CODES)
    s0, n0 = z(0, 2, 2, dtype=torch.float32), z(0, dtype=torch.int32)
    F.kv_cache_append_fp8(k0, k0.clone(), s0, s0.clone(), n0, z(0, 2, 3, 64), z(0, 2, 3, 64))
    o, lse = F.decode_attention_fp8(z(0, 4, 1, 64), k0, k0, s0, s0, n0)
    assert o.shape == (0, 4, 1, 64) and lse.shape == (0, 4)
    w = z(0, 2, 64, dtype=torch.float32)
    assert F.attention_weight_accumulate(w, z(0, 4, 1, 64), z(0, 2, 64, 64), z(0, 4, dtype=torch.float32)).shape == w.shape
    assert F.kv_cache_evict(z(0, 2, 64, 64), z(0, 2, 64, 64), n0, w, 16, 4).shape == (0, 2, 16)
    w = z(2, 2, 0, dtype=torch.float32)
    F.attention_weight_accumulate(w, z(2, 4, 1, 64), z(2, 2, 0, 64), z(2, 4, dtype=torch.float32))
    w = torch.ones(2, 2, 64, device="cuda")
    F.attention_weight_accumulate(w, z(2, 4, 0, 64), z(2, 2, 64, 64), z(2, 4, 0, dtype=torch.float32))
    assert (w == 1).all()


def test_weights_of_more_slices_than_a_grid_axis():
    """65920 (sequence, kv head) pairs of 33 heads each: one query, and two as a prompt of two head sets whose sums meet."""
    g = torch.Generator(device="cuda").manual_seed(6)
    B, Hkv, group, S, D = 1030, 64, 33, 16, 8
    r = lambda *s: torch.randn(*s, device="cuda", generator=g).bfloat16()
    k = r(B, Hkv, S, D)
    for L in (1, 2):
        q = r(B, Hkv * group, L, D)
        s = (q.float().view(B, Hkv, group * L, D) @ k.float().transpose(2, 3).contiguous()) * D ** -0.5
        lse = torch.logsumexp(s, -1).view(B, Hkv * group, L)
        w = torch.zeros(B, Hkv, S, device="cuda")
        _F().attention_weight_accumulate(w, q, k, lse)
        want = torch.softmax(s.double(), -1).sum(2)
        # scores and lse below 32 in fp32 on both sides, and sums of 66 terms
        assert ((w.double() - want).abs() <= want * (2 * (2 * D + 8) * 32 + 8 * 32 + 2 * 66 + 32) * E).all()
