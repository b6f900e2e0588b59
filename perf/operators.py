"""What the prompt-cache operators cost: attention of packed texts over a cached prompt that all of them share, and the
operations on the cache's pages (store, fork, free + compact + copy).

`run` makes one pass of a case's operator: with `own` the calls a program makes of `abstracts_search_amd.prompt_cache`,
without it the same result from elementary torch operations in 32 bits.  Shapes: n_layers x n_kv_heads x head_dim of an
encoder, pages of 64 tokens [n_pages, n_layers, n_kv_heads, 2 (K, V), 64, head_dim]; texts packed back to back."""
import math

import numpy as np
import torch

own = False

PAGE = 64
DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16}


def listed():
    att, store, fork, turn = "attention", "store", "fork", "turnover"
    return [
        # one prompted query of a search box (a short instruction in front of ten tokens): nothing but latency
        dict(name="one_query", kind=att, dtype="bf16", heads=12, kv_heads=2, dim=128, prompt=37, texts=1, q_lo=10, q_hi=10, past_lo=0, past_hi=0, causal=True),
        # one new token for each of 64 texts, each with up to 200 tokens of its own behind a prompt of 2048
        dict(name="single_tokens", kind=att, dtype="f16", heads=32, kv_heads=8, dim=128, prompt=2048, texts=64, q_lo=1, q_hi=1, past_lo=0, past_hi=200, causal=True),
        # four single tokens over a very long prompt: the cache is streamed once, the work has to be split along it
        dict(name="single_long", kind=att, dtype="bf16", heads=32, kv_heads=8, dim=128, prompt=65500, texts=4, q_lo=1, q_hi=1, past_lo=0, past_hi=31, causal=True),
        # a full encode pass (about 32 k tokens of abstracts) behind an instruction with a few examples
        dict(name="texts", kind=att, dtype="bf16", heads=12, kv_heads=2, dim=128, prompt=400, texts=128, q_lo=8, q_hi=500, past_lo=0, past_hi=0, causal=True),
        # texts behind thousands of tokens of examples: bound by the matrix cores
        dict(name="examples", kind=att, dtype="f16", heads=32, kv_heads=8, dim=128, prompt=4096, texts=48, q_lo=30, q_hi=512, past_lo=0, past_hi=0, causal=True),
        # every head with its own keys, head dim 64, ragged texts from one token on that see each other's both sides
        dict(name="both_sides", kind=att, dtype="bf16", heads=16, kv_heads=16, dim=64, prompt=1000, texts=24, q_lo=1, q_hi=333, past_lo=0, past_hi=0, causal=False),
        # a short instruction's keys and values of all layers put into the cache; thousands of tokens of examples likewise
        dict(name="store_instruction", kind=store, dtype="bf16", layers=28, kv_heads=2, dim=128, prompt=37),
        dict(name="store_examples", kind=store, dtype="bf16", layers=28, kv_heads=2, dim=128, prompt=4000),
        # four variants begun from one instruction; two hundred of them from a page of examples
        dict(name="fork_few", kind=fork, dtype="bf16", layers=28, kv_heads=2, dim=128, prompt=100, kids=4),
        dict(name="fork_many", kind=fork, dtype="f16", layers=28, kv_heads=2, dim=128, prompt=1000, kids=200),
        # a prompt leaves, the one above it moves down and is copied: a small cache, and one of 200-page prompts
        dict(name="turnover_small", kind=turn, dtype="bf16", layers=28, kv_heads=2, dim=128, prompt=500),
        dict(name="turnover_large", kind=turn, dtype="bf16", layers=28, kv_heads=2, dim=128, prompt=12800),
    ]


def draw(rng):
    def log(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    kind = rng.choice(["attention", "attention", "attention", "store", "fork", "turnover"])
    c = dict(kind=kind, dtype=rng.choice(["bf16", "f16"]))
    if kind == "attention":
        heads, kv = rng.choice([(12, 2), (32, 8), (16, 16), (4, 2), (28, 4), (64, 8)])
        c.update(heads=heads, kv_heads=kv, dim=rng.choice([64, 128]), causal=rng.random() < 0.8)
        if rng.random() < 0.4:                                   # single tokens with a past of their own
            c.update(prompt=log(1, 65000), texts=log(1, 128), q_lo=1, q_hi=1, past_lo=0, past_hi=log(1, 300))
        else:
            c.update(prompt=log(1, 4096), texts=log(1, 64), q_lo=log(1, 30), past_lo=0, past_hi=rng.choice([0, 0, 45]))
            c.update(q_hi=c["q_lo"] + log(1, 300))
            while work(c)["flops"] > 4e11:                       # never more than the largest listed one
                c["prompt"], c["texts"] = max(1, c["prompt"] // 2), max(1, c["texts"] // 2)
    else:
        c.update(layers=rng.choice([2, 12, 28]), kv_heads=rng.choice([2, 4]), dim=rng.choice([64, 128]))
        c.update(prompt=log(2, 2500 if kind == "turnover" else 3900 if kind == "store" else 2000))
        if kind == "fork":
            c.update(kids=log(1, 90))
            c["prompt"] += c["prompt"] % PAGE == 0               # the last page is partly filled: it is what a fork copies
    return c


def lengths(c):
    """[(new tokens, keys of its own)] of every text: spread over the case's ranges, the same for every seed"""
    got = []
    for i in range(c["texts"]):
        u, w = (i * 0.6180339887 + 0.5) % 1.0, (i * 0.7548776662 + 0.5) % 1.0
        q = c["q_lo"] + int(u * (c["q_hi"] - c["q_lo"] + 1))
        got.append((q, q + c["past_lo"] + int(w * (c["past_hi"] - c["past_lo"] + 1))))
    return got


def work(case):
    c = case
    if c["kind"] == "attention":
        lens = lengths(c)
        nq, nk = sum(q for q, _ in lens), sum(k for _, k in lens)
        pairs = sum(q * (c["prompt"] + k) - (q * (q - 1) // 2 if c["causal"] else 0) for q, k in lens)
        return {"bytes": 2 * c["dim"] * (2 * nq * c["heads"] + 2 * (nk + c["prompt"]) * c["kv_heads"]), "flops": 4 * c["dim"] * c["heads"] * pairs}
    token = c["layers"] * c["kv_heads"] * 2 * c["dim"] * 2       # bytes of one token's keys and values
    if c["kind"] == "store":
        return {"bytes": 2 * c["prompt"] * token, "flops": 0}
    if c["kind"] == "fork":
        return {"bytes": (1 + c["kids"]) * (c["prompt"] % PAGE) * token, "flops": 0}
    return {"bytes": 4 * c["prompt"] * token, "flops": 0}        # moved once, copied once


def inputs(c, seed):
    """the tensors of a case, from the seed alone"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    dt = DTYPES[c["dtype"]]

    def normal(*shape, scale=1.0):
        return (torch.randn(shape, generator=g, device="cuda") * scale).to(dt)

    if c["kind"] == "attention":
        lens = lengths(c)
        nq, nk = sum(q for q, _ in lens), sum(k for _, k in lens)
        kv, d, layers = c["kv_heads"], c["dim"], 2
        return dict(q=normal(nq, c["heads"], d, scale=1.5), k=normal(nk, kv, d), v=normal(nk, kv, d),
                    pk=normal(layers, c["prompt"], kv, d), pv=normal(layers, c["prompt"], kv, d))
    shape = (c["layers"], c["prompt"], c["kv_heads"], c["dim"])
    return dict(pk=normal(*shape), pv=normal(*shape))


def prepare(case, seed):
    c = case
    s = dict(case=c, **inputs(c, seed))
    layers, n, kv, d = s["pk"].shape
    n_pages = -(-n // PAGE)
    total = {"attention": n_pages, "store": n_pages, "fork": n_pages + c.get("kids", 0), "turnover": 2 * n_pages}[c["kind"]]
    if c["kind"] == "attention":
        lens = lengths(c)
        s["cu_q"] = torch.tensor(np.cumsum([0] + [q for q, _ in lens]), dtype=torch.int32, device="cuda")
        s["cu_k"] = torch.tensor(np.cumsum([0] + [k for _, k in lens]), dtype=torch.int32, device="cuda")
        s["q_max"], s["k_max"] = max(q for q, _ in lens), max(k for _, k in lens)
    if own:
        from abstracts_search_amd.prompt_cache import PromptCache
        cache = s["cache"] = PromptCache(layers, kv, d, total, dtype=s["pk"].dtype, max_entries=c.get("kids", 0) + 4)
        if c["kind"] != "store":
            s["entry"] = cache.new()
            cache.extend(s["entry"], s["pk"], s["pv"])
        if c["kind"] == "turnover":                              # the prompt that leaves lies below the one that stays
            s["low"], s["entry"] = s["entry"], cache.copy(s["entry"])
    else:
        s["pages"] = torch.zeros((total, layers, kv, 2, PAGE, d), dtype=s["pk"].dtype, device="cuda")
        s["table"] = torch.arange(n_pages, device="cuda")
        if c["kind"] != "store":
            put(s["pages"], s["table"], s["pk"], s["pv"])
        if c["kind"] == "turnover":
            s["pages"][n_pages:] = s["pages"][:n_pages]
    return s


def put(pages, table, k, v):
    """tokens 0 .. n - 1 of k, v [layers, n, kv, d] into the pages of `table`"""
    j = torch.arange(k.shape[1], device=k.device)
    pages[table[j // PAGE], :, :, 0, j % PAGE] = k.transpose(0, 1)
    pages[table[j // PAGE], :, :, 1, j % PAGE] = v.transpose(0, 1)


def run(state):
    s = state
    return (run_own if own else run_plain)(s["case"]["kind"], s)


def run_own(kind, s):
    if kind == "attention":
        return s["cache"].attention(s["entry"], 1, s["q"], s["k"], s["v"], s["cu_q"], s["cu_k"], causal=s["case"]["causal"])
    cache = s["cache"]
    if kind == "store":
        e = cache.new()
        cache.extend(e, s["pk"], s["pv"])
        table = cache.table(e)
        cache.free(e)
        return {"pages": cache.pages, "table": np.array(table)}
    if kind == "fork":
        kids = cache.fork(s["entry"], s["case"]["kids"])
        tables = [cache.table(e) for e in kids]
        cache.free(kids)
        return {"pages": cache.pages, "table": np.array(tables)}
    cache.free(s["low"])                                         # the lower prompt leaves,
    cache.compact()                                              # the other one moves down to its place
    s["low"], s["entry"] = s["entry"], cache.copy(s["entry"])    # and is copied to where it was
    return {"pages": cache.pages, "table": np.array([cache.table(s["low"]), cache.table(s["entry"])])}


def run_plain(kind, s):
    if kind == "attention":
        return plain_attention(s)
    pages, table, n = s["pages"], s["table"], s["pk"].shape[1]
    if kind == "store":
        put(pages, table, s["pk"], s["pv"])
        return {"pages": pages, "table": table}
    if kind == "fork":
        kids, used = s["case"]["kids"], n % PAGE
        new = table.numel() + torch.arange(kids, device="cuda")
        pages[new, :, :, :, :used] = pages[table[-1], :, :, :, :used]
        return {"pages": pages, "table": torch.cat([table[:-1].expand(kids, -1), new[:, None]], 1)}
    m = table.numel()
    pages[table] = pages[table + m]
    pages[table + m] = pages[table]
    return {"pages": pages, "table": torch.stack([table, table + m])}


def plain_attention(s):
    c, cu_q, cu_k = s["case"], s["cu_q"], s["cu_k"]
    kv, d, prompt = c["kv_heads"], c["dim"], c["prompt"]
    g, n, lq, lk = c["heads"] // kv, c["texts"], s["q_max"], s["k_max"]
    layer = s["pages"][s["table"], 1].float()                    # the prompt's pages -> [kv, prompt, d]
    layer = layer.permute(1, 2, 0, 3, 4).reshape(kv, 2, -1, d)[:, :, :prompt]
    pk, pv = layer[:, 0], layer[:, 1]
    # the packed texts, padded to [texts, longest, ...]
    tq = torch.arange(s["q"].shape[0], device="cuda", dtype=torch.int32)
    tk = torch.arange(s["k"].shape[0], device="cuda", dtype=torch.int32)
    sq, sk = torch.searchsorted(cu_q[1:], tq, right=True), torch.searchsorted(cu_k[1:], tk, right=True)
    q = torch.zeros((n, lq, kv, g, d), device="cuda")
    k, v = torch.zeros((n, lk, kv, d), device="cuda"), torch.zeros((n, lk, kv, d), device="cuda")
    q[sq, tq - cu_q[sq]] = s["q"].float().view(-1, kv, g, d)
    k[sk, tk - cu_k[sk]], v[sk, tk - cu_k[sk]] = s["k"].float(), s["v"].float()
    q = q.permute(2, 0, 1, 3, 4).reshape(kv, n, lq * g, d) * (1.0 / math.sqrt(d))
    k, v = k.permute(2, 0, 1, 3).contiguous(), v.permute(2, 0, 1, 3).contiguous()   # [kv, texts, longest, d]
    with_prompt = torch.matmul(q.reshape(kv, n * lq * g, d), pk.transpose(1, 2).contiguous()).view(kv, n, lq, g, prompt)
    with_own = torch.matmul(q, k.transpose(2, 3).contiguous()).view(kv, n, lq, g, lk)
    lens_q, lens_k = (cu_q[1:] - cu_q[:-1]).view(n, 1, 1), (cu_k[1:] - cu_k[:-1]).view(n, 1, 1)
    i, j = torch.arange(lq, device="cuda").view(1, lq, 1), torch.arange(lk, device="cuda").view(1, 1, lk)
    seen = (j < lens_k).expand(n, lq, lk)
    if c["causal"]:
        seen = seen & (j <= i + lens_k - lens_q)
    with_own = with_own.masked_fill(~seen[None, :, :, None], -math.inf)
    m = torch.maximum(with_prompt.amax(-1, keepdim=True), with_own.amax(-1, keepdim=True))
    ep, eo = torch.exp(with_prompt - m), torch.exp(with_own - m)
    total = ep.sum(-1, keepdim=True) + eo.sum(-1, keepdim=True)
    o = torch.matmul(ep.view(kv, n * lq * g, prompt), pv.contiguous()).view(kv, n, lq, g, d)
    o = o + torch.matmul(eo.view(kv, n, lq * g, lk), v).view(kv, n, lq, g, d)
    o = (o / total).permute(1, 2, 0, 3, 4).reshape(n, lq, kv * g, d)
    return o[sq, tq - cu_q[sq]].to(s["q"].dtype)


def exact(case, seed):
    """the definitions in 64 bits, text by text and page by page"""
    c, x = case, inputs(case, seed)
    if c["kind"] == "attention":
        if work(c)["flops"] > 2e12:
            return None
        pk, pv = x["pk"][1].double(), x["pv"][1].double()
        rep, out, a, b = c["heads"] // c["kv_heads"], [], 0, 0
        for nq, nk in lengths(c):
            keys = torch.cat([pk, x["k"][b:b + nk].double()]).repeat_interleave(rep, 1).permute(1, 2, 0).contiguous()
            vals = torch.cat([pv, x["v"][b:b + nk].double()]).repeat_interleave(rep, 1).transpose(0, 1).contiguous()
            score = torch.bmm(x["q"][a:a + nq].double().transpose(0, 1).contiguous(), keys) / math.sqrt(c["dim"])
            if c["causal"]:
                hidden = torch.ones(nq, nk, dtype=torch.bool, device="cuda").triu(nk - nq + 1)
                score[:, :, c["prompt"]:][:, hidden] = -math.inf
            out.append(torch.bmm(torch.softmax(score, -1), vals).transpose(0, 1))
            a, b = a + nq, b + nk
        return torch.cat(out)
    n = c["prompt"]
    m, used = -(-n // PAGE), n % PAGE
    total = {"store": m, "fork": m + c.get("kids", 0), "turnover": 2 * m}[c["kind"]]
    pages = torch.zeros((total, c["layers"], c["kv_heads"], 2, PAGE, c["dim"]), dtype=torch.float64, device="cuda")
    for p in range(m):
        rows = min(PAGE, n - p * PAGE)
        for which, t in enumerate((x["pk"], x["pv"])):
            pages[p, :, :, which, :rows] = t[:, p * PAGE:p * PAGE + rows].transpose(1, 2).double()
    if c["kind"] == "store":
        return {"pages": pages, "table": np.arange(m)}
    if c["kind"] == "turnover":
        pages[m:] = pages[:m]
        return {"pages": pages, "table": np.arange(2 * m).reshape(2, m)}
    for kid in range(c["kids"]):
        pages[m + kid, :, :, :, :used] = pages[m - 1, :, :, :, :used]
    return {"pages": pages, "table": np.array([list(range(m - 1)) + [m + kid] for kid in range(c["kids"])])}
