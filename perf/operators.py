"""The serving operators: writing tokens into a paged key/value cache, reading them back, attention of
one new token per sequence over that cache, and sampling the next token from the logits.

Every case has a plain form (elementary torch operations in 32 bits, in 64 for the sampling sums,
whose borders decide whole numbers) and the framework's own calls, which write the same outputs.

    from perf import operators; operators.own = True; s = operators.prepare(case, 1); operators.run(s)
"""
import math
import os
import random
import sys

import numpy as np
import torch

own = False

_TYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.uint8}
_BYTES = {"f32": 4, "f16": 2, "bf16": 2, "e4m3": 1}


# ---- the cases ---------------------------------------------------------------------------------
def listed():
    return [
        # one decode step of a small batch at GPT-2's heads: a call whose latency is the cost
        dict(name="append-decode", op="append", seqs=8, longest=1024, new=1, hk=12, d=64, dv=64, page=16, input="bf16",
             cache="bf16", packed=True, padded=0),
        # prompts of a batch written at once into an 8-bit cache, the tail of the padded batch left out
        dict(name="append-prompts-8bit", op="append", seqs=8, longest=4096, new=4096, hk=8, d=128, dv=128, page=16,
             input="bf16", cache="e4m3", packed=False, padded=1000),
        # ragged additions with odd head sizes and a page size that is no power of two
        dict(name="append-odd-8bit", op="append", seqs=5, longest=1001, new=333, hk=5, d=80, dv=72, page=24, input="f32",
             cache="e4m3", packed=False, padded=7),
        # a cached prefix gathered for a further stretch of the prompt, at GPT-2's heads
        dict(name="read-prefix", op="read", seqs=4, longest=777, hk=12, d=64, dv=64, page=16, cache="f16", output="f16"),
        # a long 8-bit prefix gathered for the dense attention
        dict(name="read-long-8bit", op="read", seqs=4, longest=16384, hk=8, d=128, dv=128, page=64, cache="e4m3",
             output="bf16"),
        # one sequence of GPT-2's context: the smallest step of a conversation
        dict(name="attend-one", op="attend", seqs=1, shortest=1024, longest=1024, h=12, hk=12, d=64, dv=64, page=16,
             input="bf16", cache="bf16"),
        # a served batch at GPT-2's heads, each sequence somewhere else in its context
        dict(name="attend-batch", op="attend", seqs=64, shortest=1, longest=1024, h=12, hk=12, d=64, dv=64, page=16,
             input="bf16", cache="bf16"),
        # grouped heads, middle to long contexts
        dict(name="attend-grouped", op="attend", seqs=32, shortest=500, longest=8191, h=32, hk=8, d=128, dv=128, page=32,
             input="f16", cache="f16"),
        # two very long contexts in 8 bits: the work is along the cache, not across rows
        dict(name="attend-long-8bit", op="attend", seqs=2, shortest=99999, longest=131072, h=64, hk=8, d=128, dv=128,
             page=64, input="bf16", cache="e4m3"),
        # 32-bit rows of odd size
        dict(name="attend-odd-f32", op="attend", seqs=7, shortest=3, longest=2050, h=10, hk=5, d=80, dv=72, page=24,
             input="f32", cache="f32"),
        # the next token of a few conversations, GPT-2's vocabulary, every row with its own settings
        dict(name="sample-few", op="sample", rows=4, vocab=50257, input="bf16", spread=3.0, kind="mixed"),
        # a large batch over a large vocabulary of odd size
        dict(name="sample-batch", op="sample", rows=256, vocab=131071, input="f32", spread=2.5, kind="mixed"),
    ]


def _between(rng, lo, hi):
    """A whole number spread over the logarithm of the range."""
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "read", "attend", "attend", "sample"])
    if op == "sample":
        vocab = _between(rng, 100, 131071)
        return dict(op=op, rows=_between(rng, 1, 256), vocab=vocab, input=rng.choice(["f32", "f16", "bf16"]),
                    spread=round(rng.uniform(0.5, 6.0), 3), kind=rng.choice(["mixed", "top_p", "plain"]))
    d = rng.choice([32, 64, 64, 80, 96, 128, 128, 256, 8 * rng.randint(2, 30)])
    c = dict(op=op, hk=rng.choice([1, 2, 3, 4, 8, 12]), d=d, dv=rng.choice([d, d, d, 8 * rng.randint(2, 30)]),
             page=rng.choice([1, 8, 16, 16, 24, 32, 64, 128]))
    if op == "append":
        c.update(input=rng.choice(["f32", "f16", "bf16", "bf16"]), packed=c["d"] == c["dv"] and rng.random() < 0.5)
        c["cache"] = rng.choice([c["input"], "e4m3"])
        new = _between(rng, 1, 2048)
        c.update(seqs=_between(rng, 1, 8), new=new, longest=new + rng.randint(0, 1000))
        c["padded"] = rng.randint(0, c["seqs"] * new // 2)
        return c
    c["cache"] = rng.choice(["f32", "f16", "bf16", "e4m3", "e4m3"])
    if op == "read":
        c["output"] = rng.choice(["f32", "f16", "bf16"])
        row = c["hk"] * (c["d"] + c["dv"]) * (_BYTES[c["cache"]] + _BYTES[c["output"]])
        c["seqs"] = _between(rng, 1, 4)
        c["longest"] = _between(rng, 1, min(16384, (1 << 28) // (c["seqs"] * row)))
        return c
    c["input"] = rng.choice(["f16", "bf16", "f32"]) if c["cache"] == "e4m3" else c["cache"]
    c["h"] = c["hk"] * rng.choice([1, 1, 2, 3, 4, 8, 16])
    c["seqs"] = _between(rng, 1, 64)
    row = c["hk"] * (c["d"] + c["dv"]) * _BYTES[c["cache"]]
    c["longest"] = _between(rng, 1, min(131072, (1 << 28) // (c["seqs"] * row)))
    c["shortest"] = rng.randint(0, c["longest"])
    return c


def _lengths(case):
    """The sequences' lengths, a ladder from the shortest to the longest (the seed only orders them)."""
    n, hi = case["seqs"], case["longest"]
    lo = case.get("shortest", max(1, hi // 2))
    return [hi if n == 1 else lo + (hi - lo) * i // (n - 1) for i in range(n)]


def _counts(case):
    """How many tokens each sequence of an append adds: the padded tokens come off the first sequences."""
    left, out = case["padded"], []
    for _ in range(case["seqs"]):
        cut = min(left, case["new"])
        out.append(case["new"] - cut)
        left -= cut
    return out


def work(case):
    if case["op"] == "sample":
        n = case["rows"] * case["vocab"]
        return {"bytes": n * _BYTES[case["input"]] + case["rows"] * 32, "flops": 4 * n}
    row, eb = case["d"] + case["dv"], _BYTES[case["cache"]]
    scales = 2 if case["cache"] == "e4m3" else 0
    if case["op"] == "append":
        tokens = sum(_counts(case))
        n = tokens * case["hk"]
        return {"bytes": n * (row * (_BYTES[case["input"]] + eb) + scales) + 8 * case["seqs"] * case["new"],
                "flops": 2 * n * row if scales else 0}
    tokens = sum(_lengths(case))
    n = tokens * case["hk"]
    pages = sum(-(-x // case["page"]) for x in _lengths(case))
    if case["op"] == "read":
        return {"bytes": n * (row * (_BYTES[case["output"]] + eb) + scales) + 8 * tokens, "flops": n * row if scales else 0}
    heads = case["seqs"] * case["h"]
    return {"bytes": n * (row * eb + scales) + 4 * pages + heads * (row * _BYTES[case["input"]] + 4),
            "flops": 2 * tokens * case["h"] * row}


# ---- inputs --------------------------------------------------------------------------------------
def _tables(case, seed, lengths):
    """A block table over shuffled pages, and the number of pages of the pool."""
    r = np.random.RandomState(seed % (1 << 31))
    wide = max(1, -(-case["longest"] // case["page"]))
    need = [-(-x // case["page"]) for x in lengths]
    pages = sum(need) + 3
    order = r.permutation(pages)
    table = np.full((case["seqs"], wide), -1, np.int32)  # entries behind a sequence's end are never looked at
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    return torch.from_numpy(table).cuda(), pages


def _pools(case, g, pages):
    """Pages as a cache holds them after some use: 8-bit rows with their scale bytes."""
    out = {}
    for name, d in (("k", case["d"]), ("v", case["dv"])):
        shape = (pages, case["hk"], case["page"], d)
        x = torch.randn(shape, generator=g, device="cuda", dtype=torch.float32 if case["cache"] == "f32" else torch.float16)
        if case["cache"] == "e4m3":
            out[name] = (x * 110.0).clamp(-448, 448).to(torch.float8_e4m3fn).view(torch.uint8)
            out[name + "_scale"] = torch.randint(118, 121, shape[:3], generator=g, device="cuda", dtype=torch.uint8)
        else:
            out[name] = x.to(_TYPES[case["cache"]])
            out[name + "_scale"] = None
    return out


def prepare(case, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = np.random.RandomState((seed * 7919 + 13) % (1 << 31))
    op = case["op"]
    s = {"case": case}
    if op == "sample":
        rows, vocab = case["rows"], case["vocab"]
        x = torch.randn((rows, vocab), generator=g, device="cuda") * case["spread"]
        x[:, :: 97] = float("-inf")  # tokens that a grammar or a block list rules out
        s["logits"] = x.to(_TYPES[case["input"]])
        s["u"] = torch.rand(rows, generator=g, device="cuda")
        pick = lambda *v: torch.from_numpy(r.choice(np.asarray(v), rows)).cuda()  # noqa: E731
        ones = torch.ones(rows, device="cuda")
        s["temperature"], s["top_p"], s["min_p"] = ones, ones.clone(), 0 * ones
        s["top_k"] = torch.zeros(rows, device="cuda", dtype=torch.int32)
        if case["kind"] != "plain":
            s["temperature"] = pick(0.6, 0.8, 1.0, 1.3).float()
            s["top_p"] = pick(0.8, 0.9, 0.95).float()
        if case["kind"] == "mixed":
            s["temperature"] = s["temperature"] * pick(1.0, 1.0, 1.0, 0.0).float()  # every fourth row takes the best token
            s["top_p"] = torch.where(pick(0, 1) > 0, s["top_p"], ones)
            s["top_k"] = pick(0, 0, 20, 50, 1000).int()
            s["min_p"] = pick(0.0, 0.0, 0.02, 0.1).float()
    else:
        lengths = _lengths(case)
        if op == "append":
            counts, lengths = _counts(case), [case["longest"]] * case["seqs"]
        else:
            lengths = [lengths[i] for i in r.permutation(len(lengths))]
        s["table"], pages = _tables(case, seed, lengths)
        s.update(_pools(case, g, pages))
        if op == "append":
            seq = np.repeat(np.arange(case["seqs"]), case["new"])
            pos = np.concatenate([np.r_[np.arange(case["longest"] - n, case["longest"]), np.full(case["new"] - n, -1)]
                                  for n in counts])
            s["seq"], s["pos"] = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (seq, pos))
            tokens, hk = len(seq), case["hk"]
            t = _TYPES[case["input"]]
            if case["packed"]:  # the in-projection's output: as many query heads as key heads, then K and V
                s["qkv"] = torch.randn((tokens, 3 * hk * case["d"]), generator=g, device="cuda").to(t)
            else:
                s["k_new"] = torch.randn((tokens, hk, case["d"]), generator=g, device="cuda").to(t)
                s["v_new"] = torch.randn((tokens, hk, case["dv"]), generator=g, device="cuda").to(t)
        elif op == "read":
            seq = np.repeat(np.arange(case["seqs"]), lengths)
            pos = np.concatenate([np.arange(n) for n in lengths])
            s["seq"], s["pos"] = (torch.from_numpy(a.astype(np.int32)).cuda() for a in (seq, pos))
        else:
            s["lengths"] = torch.tensor(lengths, device="cuda", dtype=torch.int32)
            q = torch.randn((case["seqs"], case["h"], case["d"]), generator=g, device="cuda")
            s["q"] = q.to(_TYPES[case["input"]])
            s["scale"] = 1.0 / math.sqrt(case["d"])
    if own:
        _handles(s)
    return s


# ---- the framework's calls -----------------------------------------------------------------------
def _backend():
    root = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "math-plus_b200")
    if root not in sys.path:
        sys.path.insert(0, root)
    from tensor_cuda.backend import CudaBackend
    from tensor_cuda.runtime import Device
    return CudaBackend(Device.shared(0))


_NAMES = {torch.float32: "f32", torch.float16: "f16", torch.bfloat16: "bf16", torch.int32: "i32"}


def _handles(s):
    """What a serving program holds all along: the backend, its cache and its tensors' handles, over
    the memory of the tensors above, and the buffers that its answers go to."""
    be, case = _backend(), s["case"]
    h = {"be": be}
    for name in ("table", "pos", "seq", "qkv", "k_new", "v_new", "lengths", "q", "logits", "u", "temperature", "top_k",
                 "top_p", "min_p"):
        if name in s:
            h[name] = be.external(s[name].data_ptr(), s[name].shape, _NAMES[s[name].dtype])
    if case["op"] == "sample":
        outs = [torch.empty(case["rows"], device="cuda", dtype=t) for t in (torch.int32, torch.float32, torch.int32)]
    else:
        from tensor_cuda.kv_cache import PagedKVCache
        at = [None if s[n] is None else s[n].data_ptr() for n in ("k", "v", "k_scale", "v_scale")]
        h["cache"] = PagedKVCache(be, s["k"].shape[0], case["page"], case["hk"], case["d"], case["cache"],
                                  head_dim_v=case["dv"], pools=at)
        if case["op"] == "attend":
            outs = [torch.empty((case["seqs"], case["h"], case["dv"]), device="cuda", dtype=s["q"].dtype),
                    torch.empty((case["seqs"], case["h"]), device="cuda")]
        elif case["op"] == "read":
            t = _TYPES[case["output"]]
            outs = [torch.empty((s["pos"].shape[0], case["hk"], d), device="cuda", dtype=t) for d in (case["d"], case["dv"])]
        else:
            outs = []
    s["outs"] = outs
    h["outs"] = tuple(be.external(t.data_ptr(), t.shape, _NAMES[t.dtype]) for t in outs)
    s["handles"] = h


def _run_own(s):
    h, case = s["handles"], s["case"]
    be, op = h["be"], case["op"]
    if op == "append":
        if case["packed"]:
            be.kv_append_packed(h["cache"], h["qkv"], h["table"], h["pos"], h["seq"])
        else:
            be.kv_append(h["cache"], h["k_new"], h["v_new"], h["table"], h["pos"], h["seq"])
        return _pool_outputs(s)
    if op == "read":
        be.kv_read(h["cache"], h["table"], h["pos"], h["seq"], dtype=case["output"], out=h["outs"])
    elif op == "attend":
        be.sdpa_paged(h["q"], h["cache"], h["table"], h["lengths"], s["scale"], lse=True, out=h["outs"])
    else:
        be.sample(h["logits"], h["u"], h["temperature"], h["top_k"], h["top_p"], h["min_p"], details=True, out=h["outs"])
    return s["outs"]


# ---- the plain forms ------------------------------------------------------------------------------
def _pool_outputs(s):
    if s["case"]["cache"] != "e4m3":
        return [s["k"], s["v"]]
    return [s["k"].view(torch.float8_e4m3fn), s["v"].view(torch.float8_e4m3fn), s["k_scale"], s["v_scale"]]


def _plain_append(s):
    case = s["case"]
    if case["packed"]:
        t = s["qkv"].reshape(-1, 3, case["hk"], case["d"])
        k, v = t[:, 1], t[:, 2]
    else:
        k, v = s["k_new"], s["v_new"]
    there = s["pos"] >= 0
    pos, seq = s["pos"][there].long(), s["seq"][there].long()
    page, off = s["table"][seq, pos // case["page"]].long(), pos % case["page"]

    def put(x, pool, scales):
        x = x[there]
        if scales is None:
            pool[page, :, off] = x.to(pool.dtype)
            return
        x = x.float()
        a = torch.where(x.isfinite(), x.abs(), 0).amax(-1)
        m, e = torch.frexp(a)  # a = m 2^e with m in [1/2, 1); 448 = (7/8) 2^9
        e = torch.where(a > 0, e - 9 + (m > 0.875).int(), -126).clamp(-126, 127)  # the least e with a <= 448 2^e
        codes = (x * torch.exp2(-e.double()).float()[..., None]).clamp(-448, 448).to(torch.float8_e4m3fn)
        pool[page, :, off] = codes.view(torch.uint8)
        scales[page, :, off] = (e + 127).to(torch.uint8)

    put(k, s["k"], s["k_scale"])
    put(v, s["v"], s["v_scale"])
    return _pool_outputs(s)


def _values(codes, scales):
    """Rows of a cache as 32-bit numbers."""
    if scales is None:
        return codes.float()
    return codes.view(torch.float8_e4m3fn).float() * torch.exp2(scales.float() - 127)[..., None]


def _plain_read(s):
    case = s["case"]
    pos, seq = s["pos"].long(), s["seq"].long()
    page, off = s["table"][seq, pos // case["page"]].long(), pos % case["page"]
    out = []
    for n in ("k", "v"):
        sc = s[n + "_scale"]
        out.append(_values(s[n][page, :, off], None if sc is None else sc[page, :, off]).to(_TYPES[case["output"]]))
    return out


def _plain_attend(s):
    case = s["case"]
    b, h, hk, page = case["seqs"], case["h"], case["hk"], case["page"]
    table = s["table"].long().clamp(min=0)
    wide = table.shape[1] * page
    rows = []
    for n in ("k", "v"):
        sc = s[n + "_scale"]
        x = _values(s[n][table], None if sc is None else sc[table])  # [b, pages, hk, page, d]
        rows.append(x.permute(0, 2, 1, 3, 4).reshape(b, hk, wide, -1))
    k, v = rows
    seen = torch.arange(wide, device="cuda")[None, :] < s["lengths"][:, None]
    v = torch.where(seen[:, None, :, None], v, 0)
    q = s["q"].float().reshape(b, hk, h // hk, -1)
    x = (q @ k.transpose(-1, -2)) * s["scale"]
    x = torch.where(seen[:, None, None, :], x, float("-inf"))
    top = x.amax(-1, keepdim=True)
    top = torch.where(top == float("-inf"), 0, top)
    p = torch.exp(x - top)
    total = p.sum(-1, keepdim=True)
    o = torch.where(total > 0, (p @ v) / total, 0)
    lse = torch.log(total) + top
    return [o.reshape(b, h, -1).to(s["q"].dtype), lse.reshape(b, h)]


def _plain_sample(s):
    """In 64 bits: the borders of top-p and of the drawn interval decide whole numbers."""
    x = s["logits"].double()
    x = torch.where(x.isnan(), float("-inf"), x)
    t, p = s["temperature"].double()[:, None], s["top_p"].double()[:, None]
    greedy = ~(t > 0)
    best, at = x.max(1, keepdim=True)
    w = torch.exp((x - best) / torch.where(greedy, 1, t))
    order = torch.sort(x, dim=1, descending=True, stable=True).indices
    ws = w.gather(1, order)
    rank = torch.arange(x.shape[1], device="cuda")[None, :]
    k = torch.where(s["top_k"] > 0, s["top_k"], x.shape[1])[:, None]
    keep = (rank < k) & (x.gather(1, order) > float("-inf"))
    ws = torch.where(keep, ws, 0)
    before = torch.cumsum(ws, 1) - ws
    keep &= (p >= 1) | (rank == 0) | (before < p * ws.sum(1, keepdim=True))
    keep &= (rank == 0) | (ws >= s["min_p"].double()[:, None])
    kept = torch.where(greedy[:, 0], 1, keep.sum(1))
    w = torch.where(torch.zeros_like(keep).scatter(1, order, keep), w, 0)
    c = torch.cumsum(w, 1)
    total = c[:, -1:]
    token = (c <= s["u"].double()[:, None] * total).sum(1, keepdim=True)
    first = (x == best).int().argmax(1, keepdim=True)  # the lowest index of the largest logit
    token = torch.where(greedy, first, token)
    prob = torch.where(greedy, 1, w.gather(1, token) / total)
    return [token[:, 0].int(), prob[:, 0].float(), kept.int()]


_PLAIN = {"append": _plain_append, "read": _plain_read, "attend": _plain_attend, "sample": _plain_sample}


def run(state):
    return _run_own(state) if own else _PLAIN[state["case"]["op"]](state)


# ---- from the definitions, in 64 bits --------------------------------------------------------------
def _two(e):
    """2^e exactly, from the bits of a double."""
    return ((e.to(torch.int64) + 1023) << 52).view(torch.float64)


def _e4m3_values(codes, scales):
    """The numbers that bytes stand for: sign, 4 bits of exponent (bias 7), 3 of mantissa."""
    c = codes.to(torch.int64)
    e, m = (c >> 3) & 15, (c & 7).double()
    v = torch.where(e > 0, (1 + m / 8) * _two(e - 7), m / 8 * 2.0 ** -6)
    v = torch.where(c > 127, -v, v)
    return v if scales is None else v * _two(scales.to(torch.int64) - 127)[..., None]


def _e4m3_round(x):
    """To the nearest number of 4 significant bits (steps of 2^-9 below 2^-6), ties to the even one."""
    e = torch.floor(torch.log2(x.abs().clamp(min=1e-300)))
    e = e - (_two(e) > x.abs()).double() + (_two(e + 1) <= x.abs()).double()
    step = _two(e.clamp(min=-6) - 3)
    return torch.round(x / step) * step


def _exact_append(s):
    case = s["case"]
    if case["packed"]:
        n = case["hk"] * case["d"]
        new = [s["qkv"][:, n:2 * n].reshape(-1, case["hk"], case["d"]), s["qkv"][:, 2 * n:].reshape(-1, case["hk"], case["d"])]
    else:
        new = [s["k_new"], s["v_new"]]
    pos, seq, table = s["pos"].cpu().numpy(), s["seq"].cpu().numpy(), s["table"].cpu().numpy()
    take = np.nonzero(pos >= 0)[0]
    row = table[seq[take], pos[take] // case["page"]].astype(np.int64) * case["page"] + pos[take] % case["page"]
    row, take = torch.from_numpy(row).cuda(), torch.from_numpy(take).cuda()
    pools, scales = [], []
    for x, name in zip(new, ("k", "v")):
        pool, x = s[name], x.double()[take]
        old = pool.double() if case["cache"] != "e4m3" else _e4m3_values(pool, None)
        flat = old.permute(0, 2, 1, 3).reshape(-1, case["hk"], pool.shape[-1]).clone()  # rows in the order of the positions
        if case["cache"] == "e4m3":
            a = x.abs().amax(-1).clamp(min=1e-300)
            e = torch.ceil(torch.log2(a / 448))
            e = e + (a > 448 * _two(e)).double() - (a <= 448 * _two(e - 1)).double()
            e = e.clamp(min=-126)
            x = _e4m3_round(x / _two(e)[..., None])
            sc = s[name + "_scale"].permute(0, 2, 1).reshape(-1, case["hk"]).clone()
            sc[row] = (e + 127).to(torch.uint8)
            scales.append(sc.reshape(pool.shape[0], case["page"], case["hk"]).permute(0, 2, 1).contiguous())
        flat[row] = x
        pools.append(flat.reshape(pool.shape[0], case["page"], case["hk"], -1).permute(0, 2, 1, 3).contiguous())
    return pools + scales


def _sequence(s, b, n):
    """K and V of sequence b's first n tokens in 64 bits, [hk, n, d]."""
    case = s["case"]
    out = []
    for name in ("k", "v"):
        pages = s["table"][b, : -(-n // case["page"])].long()
        x = s[name].index_select(0, pages)
        sc = s[name + "_scale"]
        x = x.double() if sc is None else _e4m3_values(x, sc.index_select(0, pages))
        out.append(x.transpose(0, 1).flatten(1, 2)[:, :n])
    return out


def _exact_read(s):
    seq = s["seq"].cpu().numpy()
    parts = [_sequence(s, b, int((seq == b).sum())) for b in range(s["case"]["seqs"])]
    return [torch.cat([p[i].transpose(0, 1) for p in parts]) for i in (0, 1)]


def _exact_attend(s):
    case, outs, lses = s["case"], [], []
    group = case["h"] // case["hk"]
    for b, n in enumerate(s["lengths"].cpu().tolist()):
        if n == 0:
            outs.append(torch.zeros((case["h"], case["dv"]), device="cuda", dtype=torch.float64))
            lses.append(torch.full((case["h"],), float("-inf"), device="cuda", dtype=torch.float64))
            continue
        k, v = _sequence(s, b, n)
        heads = []
        for i in range(case["hk"]):
            x = s["q"][b, i * group:(i + 1) * group].double() @ k[i].T * s["scale"]
            z = torch.logsumexp(x, 1)
            heads.append((torch.exp(x - z[:, None]) @ v[i], z))
        outs.append(torch.cat([o for o, _ in heads]))
        lses.append(torch.cat([z for _, z in heads]))
    return [torch.stack(outs), torch.stack(lses)]


def _exact_sample(s):
    x = s["logits"].double().cpu().numpy()
    t, k, p, m, u = (s[n].double().cpu().numpy() for n in ("temperature", "top_k", "top_p", "min_p", "u"))
    out = []
    for i in range(x.shape[0]):
        if t[i] <= 0:
            out.append((int(np.argmax(x[i])), 1.0, 1))
            continue
        order = np.argsort(-x[i], kind="stable")
        order = order[x[i][order] > -np.inf]
        if k[i] > 0:
            order = order[: int(k[i])]
        w = np.exp((x[i][order] - x[i][order[0]]) / t[i])
        if p[i] < 1:
            before = np.concatenate([[0.0], np.cumsum(w)[:-1]])
            w = w[: max(1, int(np.sum(before < p[i] * w.sum())))]
        w = w[: max(1, int(np.sum(w >= m[i])))]
        order = order[: len(w)]
        by = np.argsort(order)
        c = np.cumsum(w[by])
        j = min(int(np.searchsorted(c, u[i] * c[-1], side="right")), len(w) - 1)
        out.append((int(order[by[j]]), w[by[j]] / c[-1], len(w)))
    tok, prob, kept = zip(*out)
    return [np.array(tok, np.int32), np.array(prob), np.array(kept, np.int32)]


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "read": _exact_read, "attend": _exact_attend, "sample": _exact_sample}[case["op"]](s)


if __name__ == "__main__":
    for c in listed() + [dict(draw(random.Random(i)), name=f"drawn {i}") for i in range(6)]:
        print(c["name"], {k: f"{v:.3g}" for k, v in work(c).items()})
