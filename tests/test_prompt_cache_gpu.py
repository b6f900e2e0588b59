"""GPU tests of the prompt cache (csrc/prompt_kernels.h through prompt_cache.PromptCache): the attention of packed texts behind
a cached prompt against the formula in 64 bits, and the operations on the cache's pages against a host model of them.

Tolerance of the attention, element by element, from the roundings it makes.  With w_j = p_j / sum p (the exact weights):
  * a probability enters the product with V rounded to the tensors' type: off by at most half a step, h = finfo.eps / 2, of
    itself, so the output by h sum w |v|;
  * the output is rounded once: h |o|;
  * scores, exponentials, sums and accumulators are f32.  A score of magnitude s (sum of |q k| products x scale) is off by at
    most ~hd 2^-24 s, which moves its weight by that much: with the inputs below s < 200 and hd <= 128, 2^-24 x 128 x 200 = 1.6e-3
    at the very worst, where every rounding goes the same way; the bound used is 4e-4 sum w |v| (a quarter of that);
  * f16 holds 2^7 p: a probability below 2^-25 2^-7 of the largest is lost: at most 2^-32 |v| for each key (below the f32 term)."""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
BF, HF = torch.bfloat16, torch.float16


@pytest.fixture(scope="module")
def pc():
    import abstracts_search_amd.prompt_cache as m
    return m


def reference(q, pk, pv, k, v, cu_q, cu_k, causal, scale=None):
    """(o, sum w |v|) in 64 bits; rows that see nothing are zero"""
    hd, rep = q.shape[2], q.shape[1] // pk.shape[1]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    b = torch.zeros_like(o)
    for i in range(len(cu_q) - 1):
        a0, a1, k0, k1 = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
        nq, nk = a1 - a0, k1 - k0
        if not nq:
            continue
        kk = torch.cat([pk.double(), k[k0:k1].double()]).repeat_interleave(rep, 1)
        vv = torch.cat([pv.double(), v[k0:k1].double()]).repeat_interleave(rep, 1)
        P = pk.shape[0]
        for h in range(q.shape[1]):
            for t in range(nq):
                n = P + (min(max(nk - nq + t + 1, 0), nk) if causal else nk)
                if not n:
                    continue
                w = torch.softmax((kk[:n, h] @ q[a0 + t, h].double()) * scale, 0)
                o[a0 + t, h] = w @ vv[:n, h]
                b[a0 + t, h] = w @ vv[:n, h].abs()
    return o, b


def reference_many(q, pk, pv, k, v, cu_q, cu_k, causal, scale=None):
    """the same by whole matrices (long cases)"""
    hd, rep, P = q.shape[2], q.shape[1] // pk.shape[1], pk.shape[0]
    scale = 1.0 / math.sqrt(hd) if scale is None else scale
    o = torch.zeros(q.shape, dtype=torch.float64, device=q.device)
    b = torch.zeros_like(o)
    for i in range(len(cu_q) - 1):
        a0, a1, k0, k1 = cu_q[i], cu_q[i + 1], cu_k[i], cu_k[i + 1]
        nq, nk = a1 - a0, k1 - k0
        if not nq or not P + nk:
            continue
        kk = torch.cat([pk.double(), k[k0:k1].double()]).repeat_interleave(rep, 1)
        vv = torch.cat([pv.double(), v[k0:k1].double()]).repeat_interleave(rep, 1)
        s = torch.bmm(q[a0:a1].double().transpose(0, 1).contiguous(), kk.permute(1, 2, 0).contiguous()) * scale
        if causal:
            s[:, :, P:].masked_fill_(torch.ones(nq, nk, dtype=torch.bool, device=q.device).triu(nk - nq + 1), -math.inf)
        w = torch.softmax(s, -1)
        sees = P + (torch.arange(nk - nq + 1, nk + 1, device=q.device).clamp(0, nk) if causal else torch.full((nq,), nk, device=q.device))
        w = torch.where((sees == 0).view(1, nq, 1), torch.zeros_like(w), w)
        o[a0:a1] = torch.bmm(w, vv.transpose(0, 1).contiguous()).transpose(0, 1)
        b[a0:a1] = torch.bmm(w, vv.abs().transpose(0, 1).contiguous()).transpose(0, 1)
    return o, b


def close(out, o, b, what=""):
    h = torch.finfo(out.dtype).eps / 2
    err = (out.double() - o).abs()
    tol = (h + 4e-4) * b + h * o.abs() * (1 + h) + 1e-7
    bad = ~(err <= tol)
    assert not bad.any(), (what, int(bad.sum()), bad.nonzero()[:5].tolist(), float(err[bad].max()), float((err / tol)[bad].max()))


def make(pc, dtype, heads, kv, hd, prompt, lens, past=None, layers=2, layer=1, seed=0, scramble=True):
    """a cache with a prompt in scattered pages, and packed texts"""
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, generator=g, device="cuda").to(dtype)
    cache = pc.PromptCache(layers, kv, hd, -(-prompt // 64) * 2 + 6, dtype=dtype, max_entries=8)
    pk, pv = r(layers, prompt, kv, hd), r(layers, prompt, kv, hd)
    e = cache.new()
    if scramble:                                              # two entries grow in turn, one of them leaves: every other page
        other = cache.new()
        for p0 in range(0, prompt, 64):
            cache.extend(e, pk[:, p0:p0 + 64], pv[:, p0:p0 + 64])
            cache.extend(other, pk[:, :1].expand(-1, 64, -1, -1), pv[:, :1].expand(-1, 64, -1, -1))
        cache.free(other)
    else:
        cache.extend(e, pk, pv)
    past = past or [0] * len(lens)
    cu_q = np.cumsum([0] + list(lens)).tolist()
    cu_k = np.cumsum([0] + [n + p for n, p in zip(lens, past)]).tolist()
    q, k, v = r(cu_q[-1], heads, hd) * 1.5, r(cu_k[-1], kv, hd), r(cu_k[-1], kv, hd)
    return cache, e, pk[layer], pv[layer], q, k, v, cu_q, cu_k


def dev(cu):
    return torch.tensor(cu, dtype=torch.int32, device="cuda")


CASES = [
    # dtype heads kv hd prompt lens past causal
    (BF, 12, 2, 128, 37, [10], None, True),
    (BF, 4, 2, 64, 1, [1], None, True),
    (HF, 8, 8, 64, 64, [1, 1, 1], [0, 5, 64], True),
    (BF, 7, 1, 128, 65, [3, 0, 17, 1, 0], [0, 4, 2, 9, 0], True),
    (HF, 16, 2, 128, 130, [64, 65, 63], None, True),
    (BF, 6, 3, 64, 0, [5, 33, 1, 70], None, True),
    (BF, 6, 3, 64, 0, [5, 33, 1, 70], [3, 0, 0, 64], False),
    (HF, 5, 5, 128, 63, [2, 90], [61, 40], True),
    (BF, 40, 1, 128, 128, [3, 9], [0, 1], True),              # a group of 40 heads: a token spans several tiles of rows
    (HF, 28, 4, 128, 200, [1] * 40, list(range(40)), True),
    (BF, 64, 8, 64, 257, [1] * 9 + [0] * 3 + [2], [0] * 12 + [7], False),
    (BF, 2, 2, 128, 5, [129, 1, 255], [0, 300, 0], True),
]


@pytest.mark.parametrize("dtype,heads,kv,hd,prompt,lens,past,causal", CASES)
def test_attention_vs_formula(pc, dtype, heads, kv, hd, prompt, lens, past, causal):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, heads, kv, hd, prompt, lens, past)
    out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k), causal=causal)
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, causal)
    close(out, o, b)


def test_the_two_references_agree(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 5, [3, 0, 6], [0, 2, 4])
    for causal in (True, False):
        a, b = reference(q, pk, pv, k, v, cu_q, cu_k, causal), reference_many(q, pk, pv, k, v, cu_q, cu_k, causal)
        assert torch.allclose(a[0], b[0], rtol=1e-12, atol=1e-12) and torch.allclose(a[1], b[1], rtol=1e-12, atol=1e-12)


def test_more_queries_than_keys_leaves_rows_empty(pc):
    """causal, aligned at the end: with 2 keys for 5 queries the first three see no key of their own; without a prompt they are zero"""
    for prompt in (0, 3):
        cache, e, pk, pv, q, _, _, cu_q, _ = make(pc, BF, 4, 2, 64, prompt, [5, 4, 3])
        cu_k = [0, 2, 2, 5]
        k, v = torch.randn(5, 2, 64, device="cuda").to(BF), torch.randn(5, 2, 64, device="cuda").to(BF)
        out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
        o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
        close(out, o, b)
        if not prompt:
            assert (out[:3] == 0).all() and (out[5:9] == 0).all() and (out[3:5] != 0).any()


def test_no_own_keys_one_text_and_default_bounds(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, HF, 6, 2, 64, 70, [21])
    none = torch.zeros(0, 2, 64, dtype=HF, device="cuda")
    o, b = reference_many(q, pk, pv, none, none, [0, 21], [0, 0], True)
    close(cache.attention(e, 1, q), o, b)
    close(cache.attention(e, 1, q, none, none), o, b)
    o, b = reference_many(q, pk, pv, k, v, [0, 21], [0, 21], True)
    close(cache.attention(e, 1, q, k, v), o, b)
    close(cache.attention(e, 1, q, k, v, dev([0, 21])), o, b)
    o, b = reference_many(q, pk, pv, k, v, [0, 21], [0, 21], True, scale=0.3)
    close(cache.attention(e, 1, q, k, v, scale=0.3), o, b)
    assert cache.attention(e, 1, q[:0]).shape == (0, 6, 64)


@pytest.mark.parametrize("causal", [True, False])
def test_strided_views_of_a_fused_projection(pc, causal):
    """q, k and v as slices of one [tokens, (heads + 2 kv) hd] buffer; out a slice too; odd strides are copied inside the call"""
    heads, kv, hd, prompt, lens = 6, 2, 64, 77, [19, 1, 40]
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, heads, kv, hd, prompt, lens)
    T = cu_q[-1]
    fused = torch.cat([q, k, v], 1).contiguous()
    big = torch.full((T, 2 * heads, hd), 7.0, dtype=BF, device="cuda")
    fq, fk, fv = fused[:, :heads], fused[:, heads:heads + kv], fused[:, heads + kv:]
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, causal)
    got = cache.attention(e, 1, fq, fk, fv, dev(cu_q), dev(cu_k), causal=causal, out=big[:, heads:])
    close(got, o, b)
    assert (big[:, :heads] == 7).all()
    odd = torch.zeros(T, heads, hd + 1, dtype=BF, device="cuda")[:, :, 1:]      # rows of 65 elements, 2 bytes off
    odd.copy_(q)
    turned = k.permute(1, 0, 2).contiguous().permute(1, 0, 2)                   # heads outermost
    last = v.permute(0, 2, 1).contiguous().permute(0, 2, 1)                     # the last axis strided
    assert torch.equal(cache.attention(e, 1, odd, turned, last, dev(cu_q), dev(cu_k), causal=causal), got)


def test_rows_behind_the_last_text(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 6, 2, 128, 90, [30, 5])
    pad = torch.randn(9, 6, 128, device="cuda").to(BF)
    padk = torch.full((9, 2, 128), float("nan"), dtype=BF, device="cuda")
    q2, k2, v2 = torch.cat([q, pad]), torch.cat([k, padk]), torch.cat([v, padk])
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    out = cache.attention(e, 1, q2, k2, v2, dev(cu_q), dev(cu_k))
    close(out[:35], o, b)
    assert (out[35:] == 0).all()
    held = torch.full_like(q2, 3.0)
    cache.attention(e, 1, q2, k2, v2, dev(cu_q), dev(cu_k), out=held)
    assert torch.equal(held[:35], out[:35]) and (held[35:] == 3).all()


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("heads,kv,hd,prompt,lens", [(12, 2, 128, 70, [9, 30, 64, 1, 50]), (4, 4, 64, 0, [3, 1, 1, 20])])
def test_what_is_masked_may_hold_anything(pc, dtype, heads, kv, hd, prompt, lens):
    """infinities and NaN in the keys and values of later tokens and of other texts leave every row as it was; the rows that
    do see them get what the formula gives"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, heads, kv, hd, prompt, lens)
    clean = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
    k2, v2 = k.clone(), v.clone()
    for i, x in ((1, float("nan")), (3, float("inf")), (len(lens) - 1, float("-inf"))):
        at = cu_k[i + 1] - 1                                    # a text's last key: seen by its last query alone
        v2[at] = x
        k2[at] = -x
    out = cache.attention(e, 1, q, k2, v2, dev(cu_q), dev(cu_k))
    hit = torch.zeros(cu_q[-1], dtype=torch.bool, device="cuda")
    for i in (1, 3, len(lens) - 1):
        hit[cu_q[i + 1] - 1] = True
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    close(out[~hit], o[~hit], b[~hit])
    close(clean, o, b)
    assert torch.isnan(out[cu_q[2] - 1]).all()                  # (NaN keys and values)
    # a key of the type's lowest value, and one that is -inf in every product, weigh nothing
    low = torch.finfo(dtype).min
    k3, q3 = k.clone(), q.abs() + 0.01
    k3[cu_k[1] - 1], k3[cu_k[2] - 1] = low, float("-inf")
    out = cache.attention(e, 1, q3, k3, v, dev(cu_q), dev(cu_k))
    o, b = reference_many(q3, pk, pv, k3, v, cu_q, cu_k, True)
    ok = ~torch.isnan(o).any(-1).any(-1)                        # (a text whose only key is -inf has no softmax: NaN on both sides)
    close(out[ok], o[ok], b[ok])
    assert torch.isnan(out[~ok]).all()


@pytest.mark.parametrize("prompt,lens", [(300, [40, 3, 60]), (2000, [1, 1, 1])])
def test_prompts_that_hold_no_numbers(pc, prompt, lens):
    """infinities and NaN that rows do see: those rows are not finite, the others right"""
    for what, where in ((math.nan, "v"), (math.inf, "v"), (math.nan, "k")):
        cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 8, 2, 128, prompt, lens)
        o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
        bad = (pv if where == "v" else pk)[None, prompt - 7:prompt - 6].clone()
        bad[..., 1, 5] = what                                 # key head 1, dim 5
        other = (pk if where == "v" else pv)[None, prompt - 7:prompt - 6]
        cache.write(e, bad if where == "k" else other, bad if where == "v" else other, prompt - 7, layer=1)
        v[cu_k[1] - 1] = math.nan                             # and a text's last value: only its last token sees it
        out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
        last = cu_q[1] - 1
        keep = [t for t in range(cu_q[-1]) if t != last]
        close(out[keep][:, :4], o[keep][:, :4], b[keep][:, :4])
        assert out[last].isnan().all()
        if where == "k":
            assert out[:, 4:].isnan().all()
        else:                                                 # (an infinity stays one behind a masked NaN)
            assert (out[keep][:, 4:, 5].isnan() if what != what else out[keep][:, 4:, 5] == what).all()
            dims = [d for d in range(128) if d != 5]
            close(out[keep][:, 4:][..., dims], o[keep][:, 4:][..., dims], b[keep][:, 4:][..., dims])


def test_extreme_scores(pc):
    """scores far apart (a one-hot softmax), all equal, and a maximum that grows all along the prompt"""
    for dtype in (BF, HF):
        cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, 4, 2, 64, 300, [10, 70], scramble=False)
        for scale in (0.0, 4.0):
            o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True, scale=scale)
            out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k), scale=scale)
            # (scale 4: scores up to ~200: 32 x the f32 term of the ordinary scale, see the tolerance above)
            h = torch.finfo(dtype).eps / 2
            assert ((out.double() - o).abs() <= (h + 1.6e-3) * b + h * o.abs() * (1 + h) + 1e-7).all()
        ramp = torch.linspace(0.01, 3, 300, device="cuda")[:, None, None].expand(300, 2, 64).to(dtype)
        grow = cache.new()
        cache.extend(grow, ramp.expand(2, 300, 2, 64), pv.expand(2, 300, 2, 64))
        qq = torch.ones_like(q)
        o, b = reference_many(qq, ramp, pv, k, v, cu_q, cu_k, True)
        close(cache.attention(grow, 1, qq, k, v, dev(cu_q), dev(cu_k)), o, b)


def test_long_prompt_few_rows_and_many(pc):
    """single tokens over a long prompt (the work is split along it), and enough rows to fill the chip"""
    for dtype, heads, kv, hd, prompt, lens, past in ((BF, 32, 8, 128, 20001, [1, 1, 1], [0, 31, 2]), (HF, 12, 2, 128, 9000, [7], None),
                                                     (BF, 16, 16, 64, 1000, [200, 1, 333, 64], None), (HF, 12, 2, 128, 400, [500, 77, 300, 90, 512], None)):
        cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, heads, kv, hd, prompt, lens, past, scramble=False)
        for causal in (True, False):
            o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, causal)
            out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k), causal=causal)
            close(out, o, b, (heads, prompt, causal))
            assert torch.equal(out, cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k), causal=causal))   # the same bits every time


def test_more_texts_than_a_table_in_shared_memory(pc):
    lens = [(i * 7) % 3 for i in range(3000)]
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 20, lens)
    out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
    g = torch.Generator().manual_seed(1)
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    close(out, o, b)


def test_bounds_that_are_no_bounds_stay_inside(pc):
    """cu arrays are device data nobody checks: wrong ones give wrong rows, not reads outside (texts past the end are cut)"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [30, 20])
    for cq, ck in (([0, 30, 90], [0, 30, 90]), ([0, 30, 50], [0, 1 << 30, 1 << 30]), ([0, 30, 50], [-5, 30, -7]), ([5, 3, 50], [0, 30, 50])):
        out = cache.attention(e, 1, q, k, v, dev(cq), dev(ck))
        assert out.shape == q.shape
    torch.cuda.synchronize()


# ---------------------------------------------------------------------------------------------------------------
# pages
# ---------------------------------------------------------------------------------------------------------------
class Model:
    """what the entries hold, on the host"""

    def __init__(self):
        self.kv = {}

    def check(self, pc, cache):
        held = {}
        for e, (k, v) in self.kv.items():
            assert cache.length(e) == k.shape[1]
            t = cache.table(e)
            assert len(t) == -(-k.shape[1] // 64) and all(0 <= p < cache.n_pages for p in t)
            for i, p in enumerate(t):
                rows = min(64, k.shape[1] - 64 * i)
                page = cache.pages[p]
                assert torch.equal(page[:, :, 0, :rows].transpose(1, 2).cpu(), k[:, 64 * i:64 * i + rows]), (e, i)
                assert torch.equal(page[:, :, 1, :rows].transpose(1, 2).cpu(), v[:, 64 * i:64 * i + rows]), (e, i)
                held.setdefault(p, []).append((e, rows))
        for p, who in held.items():                             # only full pages are shared
            assert len(who) == 1 or all(r == 64 for _, r in who)
        assert cache.used_pages == len(held)


@pytest.mark.parametrize("dtype,layers,kv,hd", [(BF, 3, 2, 64), (HF, 1, 5, 128)])
def test_pages_against_a_model(pc, dtype, layers, kv, hd):
    """two hundred operations in a fixed random order; after each, every entry holds what it should"""
    rng = np.random.default_rng(3)
    g = torch.Generator(device="cuda").manual_seed(2)
    cache, m = pc.PromptCache(layers, kv, hd, 40, dtype=dtype, max_entries=12), Model()
    full = 0
    for step in range(200):
        op = rng.choice(["new", "extend", "extend", "fork", "copy", "free", "compact", "resize", "write"])
        live = sorted(m.kv)
        e = int(rng.choice(live)) if live else None
        try:
            if op == "new" or e is None:
                n = cache.new()
                assert n not in m.kv
                m.kv[n] = (torch.zeros(layers, 0, kv, hd, dtype=dtype),) * 2
            elif op == "extend":
                n = int(rng.choice([0, 1, 5, 63, 64, 65, 200]))
                k, v = (torch.randn(layers, n, kv, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
                cache.extend(e, k, v)
                m.kv[e] = tuple(torch.cat([a, b.cpu()], 1) for a, b in zip(m.kv[e], (k, v)))
            elif op == "fork":
                kids = cache.fork(e, int(rng.integers(0, 4)))
                assert not set(kids) & set(m.kv) and len(set(kids)) == len(kids)
                for c in kids:
                    m.kv[c] = m.kv[e]
            elif op == "copy":
                c = cache.copy(e)
                m.kv[c] = m.kv[e]
                assert not set(cache.table(c)) & set(cache.table(e))
            elif op == "free":
                cache.free(e)
                del m.kv[e]
            elif op == "compact":
                cache.compact()
                assert all(p < cache.used_pages for x in m.kv for p in cache.table(x))
            elif op == "resize":
                cache.resize(max(1, cache.used_pages, int(rng.integers(20, 50))))
                assert all(p < cache.used_pages for x in m.kv for p in cache.table(x))
            elif op == "write":
                n = m.kv[e][0].shape[1]
                if n % 64:                                      # the last, partly filled page is the entry's own
                    s = n - n % 64
                    k, v = (torch.randn(1, n - s, kv, hd, generator=g, device="cuda").to(dtype) for _ in range(2))
                    cache.write(e, k, v, s, layer=layers - 1)
                    kk, vv = m.kv[e][0].clone(), m.kv[e][1].clone()
                    kk[layers - 1, s:], vv[layers - 1, s:] = k[0].cpu(), v[0].cpu()
                    m.kv[e] = (kk, vv)
        except RuntimeError as err:                             # a full pool or list of entries refuses and changes nothing
            assert "free" in str(err) or "max_entries" in str(err), err
            full += 1
            cache.free([x for x in live[::2]])
            for x in live[::2]:
                del m.kv[x]
        m.check(pc, cache)
    assert full >= 2


def test_pages_are_handed_out_lowest_first_and_shared(pc):
    cache = pc.PromptCache(1, 2, 64, 12)
    t = torch.randn(1, 130, 2, 64, device="cuda").to(BF)
    a = cache.new()
    cache.extend(a, t, t)
    kids = cache.fork(a, 3)
    assert cache.table(a) == [0, 1, 2] and [cache.table(x) for x in kids] == [[0, 1, 3], [0, 1, 4], [0, 1, 5]]
    cache.free([a, kids[1]])
    assert cache.used_pages == 4
    b = cache.new()
    cache.extend(b, t[:, :100], t[:, :100])
    assert cache.table(b) == [2, 4]
    cache.free(kids[0])
    assert cache.compact() == 1 and sorted(sum((cache.table(x) for x in (kids[2], b)), [])) == [0, 1, 2, 3, 4]
    assert cache.compact() == 0
    with pytest.raises(RuntimeError, match="free"):
        cache.reserve(b, 64 * 10)
    assert cache.length(b) == 100


def test_strided_keys_and_values_are_stored(pc):
    cache = pc.PromptCache(2, 2, 64, 8)
    e = cache.new()
    x = torch.randn(2, 70, 3, 2, 64, device="cuda").to(BF)
    cache.extend(e, x[:, :, 1], x[:, :, 2])                     # slices of a fused buffer
    p = cache.pages[cache.table(e)].transpose(0, 1).transpose(1, 2)
    assert torch.equal(cache.pages[0][:, :, 0].transpose(1, 2), x[:, :64, 1]) and torch.equal(cache.pages[1][:, :, 1, :6].transpose(1, 2), x[:, 64:, 2])
    odd = torch.randn(2, 5, 2, 65, device="cuda").to(BF)[..., 1:]
    cache.extend(e, odd, odd)
    assert torch.equal(cache.pages[1][:, :, 0, 6:11].transpose(1, 2), odd)


def test_more_pages_than_a_launch_carries(pc):
    """prompts of more than 896 pages, forks of more than 320 entries, copies and moves of more than 480 pages: several launches each"""
    cache = pc.PromptCache(1, 1, 64, 4000, max_entries=800)
    g = torch.Generator(device="cuda").manual_seed(4)
    n = 64 * 1000 + 7
    k, v = (torch.randn(1, n, 1, 64, generator=g, device="cuda").to(BF) for _ in range(2))
    low, e = cache.new(), cache.new()
    cache.extend(low, k[:, :64 * 900], v[:, :64 * 900])
    cache.extend(e, k[:, :5], v[:, :5])
    cache.extend(e, k[:, 5:], v[:, 5:])                          # 1001 pages, the first one begun
    kids = cache.fork(e, 700)
    cache.free(low)
    assert cache.compact() == 900 and cache.used_pages == 1701

    def holds(x):
        t = torch.tensor(cache.table(x), device="cuda")
        return [cache.pages[t, 0, 0, w].reshape(-1, 64)[:n] for w in (0, 1)]

    for x in (e, kids[0], kids[319], kids[320], kids[699], cache.copy(kids[5])):
        assert torch.equal(holds(x)[0], k[0, :, 0]) and torch.equal(holds(x)[1], v[0, :, 0])
    q = torch.randn(3, 2, 64, generator=g, device="cuda").to(BF)
    none = torch.zeros(0, 1, 64, dtype=BF, device="cuda")
    o, b = reference_many(q, k[0], v[0], none, none, [0, 3], [0, 0], True)
    for x in (e, kids[650]):
        close(cache.attention(x, 0, q), o, b)
    cache.resize(3000)
    assert torch.equal(holds(kids[650])[0], k[0, :, 0])
    close(cache.attention(kids[650], 0, q), o, b)


def test_offsets_beyond_32_bits(pc):
    """a pool of 5 GiB: entries behind the first 4 GiB (bytes, and 2^31 elements)"""
    layers, kv, hd = 16, 4, 128                                  # 2 MiB a page
    cache = pc.PromptCache(layers, kv, hd, 2600)
    low = cache.new()
    cache.reserve(low, 64 * 2300)                                # 4.6 GiB
    g = torch.Generator(device="cuda").manual_seed(9)
    k, v = (torch.randn(layers, 200, kv, hd, generator=g, device="cuda").to(BF) for _ in range(2))
    e = cache.new()
    cache.extend(e, k, v)
    assert min(cache.table(e)) == 2300
    kid = cache.fork(e)[0]
    q = torch.randn(9, 8, hd, generator=g, device="cuda").to(BF)
    none = torch.zeros(0, kv, hd, dtype=BF, device="cuda")
    for x in (e, kid, cache.copy(e)):
        for layer in (0, layers - 1):
            o, b = reference_many(q, k[layer], v[layer], none, none, [0, 9], [0, 0], True)
            close(cache.attention(x, layer, q), o, b)
    cache.free(low)
    assert cache.compact() == cache.used_pages
    close(cache.attention(kid, layers - 1, q), o, b)


def test_nothing_to_see_and_broadcast_operands(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 6, 3, 64, 0, [4, 9])
    assert (cache.attention(e, 1, q) == 0).all()
    none = torch.zeros(0, 3, 64, dtype=BF, device="cuda")
    assert (cache.attention(e, 1, q, none, none, dev(cu_q), dev([0, 0, 0]), causal=False) == 0).all()
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 6, 3, 64, 66, [4, 9])
    k1, v1 = k[:, :1].expand(-1, 3, -1), v[:, :1].expand(-1, 3, -1)              # one key head for all: stride 0
    o, b = reference_many(q, pk, pv, k1, v1, cu_q, cu_k, True)
    close(cache.attention(e, 1, q, k1, v1, dev(cu_q), dev(cu_k)), o, b)
    q1 = q[:, :1].expand(-1, 6, -1)
    o, b = reference_many(q1, pk, pv, k, v, cu_q, cu_k, True)
    close(cache.attention(e, 1, q1, k, v, dev(cu_q), dev(cu_k)), o, b)
    own = q.clone()                                              # the output in q's place
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    cache.attention(e, 1, own, k, v, dev(cu_q), dev(cu_k), out=own)
    close(own, o, b)


@pytest.mark.parametrize("prompt,first", [(0, 0), (1000, 0), (0, 9)])
def test_split_keys_and_rows_without_any(pc, prompt, first):
    """few rows and many keys of their own: the keys are split, and the join has to know which rows see nothing, belong to no text,
    or were done again (what is masked holds no numbers)"""
    lens, past = [1] * 9 + [0, 30, 1] + [1] * 9, [300, 0, 7, 64, 1, 130, 0, 500, 2, 0, -20, -1] + [90] * 9
    lens, past, at = lens[first:], past[first:], 10 - first   # (from the tenth on: too few keys to split)
    if first:
        lens, past = lens[:3], past[:3]
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 8, 2, 128, prompt, lens, past)
    assert first or cu_k[-1] > 1000
    # text `at`: 30 queries on 10 keys, the first 20 of which see none of them; the one behind it: no key at all
    v[cu_k[at] + 5:cu_k[at + 1]] = math.nan                       # .. and the rows before the 26th see none of these
    tail = 3                                                  # rows of no text
    qq = torch.cat([q, q[:tail]])
    out = torch.full_like(qq, 7.0)
    cache.attention(e, 1, qq, k, v, dev(cu_q), dev(cu_k), out=out)
    assert (out[-tail:] == 7.0).all()
    fresh = cache.attention(e, 1, qq, k, v, dev(cu_q), dev(cu_k))
    assert (fresh[-tail:] == 0).all() and torch.equal(fresh[:-tail].isnan(), out[:-tail].isnan())
    assert torch.equal(fresh[:-tail].nan_to_num(), out[:-tail].nan_to_num())
    r0, r1 = cu_q[at] + 25, cu_q[at + 1]
    assert out[r0:r1].isnan().all()
    if not prompt:
        assert (out[cu_q[at]:cu_q[at] + 20] == 0).all() and (out[cu_q[at + 1]:cu_q[at + 2]] == 0).all()
    v[cu_k[at] + 5:cu_k[at + 1]] = 0
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    keep = torch.ones(q.shape[0], dtype=torch.bool, device="cuda")
    keep[r0:r1] = False
    close(out[:-tail][keep], o[keep], b[keep])


@pytest.mark.parametrize("prompt,front,n", [(0, 5, 3), (70, 5, 3), (70, 200, 3), (0, 33, 400)])
def test_rows_in_front_of_the_first_text(pc, prompt, front, n):
    """bounds that begin behind 0: the rows and keys in front belong to no text"""
    lens = [2, n, 40]
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, HF, 6, 3, 64, prompt, lens, [0, 9, 1])
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    wide = lambda t, m: torch.cat([torch.full_like(t[:1], math.nan).expand(m, -1, -1), t])
    qq, kk, vv = wide(q, front), wide(k, 11), wide(v, 11)
    out = torch.full_like(qq, 7.0)
    bounds = dev([c + front for c in cu_q]), dev([c + 11 for c in cu_k])
    cache.attention(e, 1, qq, kk, vv, *bounds, out=out)
    assert (out[:front] == 7.0).all()
    close(out[front:], o, b)
    fresh = cache.attention(e, 1, qq, kk, vv, *bounds)
    assert (fresh[:front] == 0).all() and torch.equal(fresh[front:], out[front:])


@pytest.mark.parametrize("dtype", [BF, HF])
def test_both_forms_of_the_probabilities(pc, dtype):
    """few rows keep the probabilities in two parts: the error is the output's rounding alone; many rows keep one part"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, 8, 2, 128, 500, [300, 212, 88])
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))                   # 2400 rows a key head
    close(out, o, b)
    few = cache.attention(e, 1, q[:60], k[:180], v[:180], dev([0, 21, 60]), dev([0, 30, 180]))   # 240
    o2, b2 = reference_many(q[:60], pk, pv, k[:180], v[:180], [0, 21, 60], [0, 30, 180], True)
    h = torch.finfo(dtype).eps / 2                               # (and h^2 b of what the second part leaves)
    assert ((few.double() - o2).abs() <= h * o2.abs() * (1 + h) + (h * h + 4e-4) * b2 + 1e-7).all()


# ---------------------------------------------------------------------------------------------------------------
# streams, graphs, refusals
# ---------------------------------------------------------------------------------------------------------------
def test_a_captured_pass_follows_its_inputs_and_moved_pages(pc):
    """two graphs over one cache, replayed in turn with eager work between; a page move in between is followed"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 12, 2, 128, 5000, [1, 1, 9])
    _, _, _, _, q2, k2, v2, cu_q2, cu_k2 = make(pc, BF, 12, 2, 128, 70, [40, 3], seed=5)
    args = [(q, k, v, dev(cu_q), dev(cu_k)), (q2, k2, v2, dev(cu_q2), dev(cu_k2))]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for a in args:
            cache.attention(e, 1, *a)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for a in args:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(cache.attention(e, 1, *a))
        graphs.append(g)
    for rep in range(4):
        for a, g, o in zip(args, graphs, outs):
            a[0].mul_(-0.9)
            g.replay()
            want = cache.attention(e, 1, *a)
            torch.cuda.synchronize()
            assert torch.equal(o, want), rep
        if rep == 1:
            assert cache.compact() > 0
    with pytest.raises(RuntimeError, match="captured"):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.fork(e)
    torch.cuda.synchronize()


def test_another_stream_and_freed_pages(pc):
    """an entry read on a side stream is freed and its pages refilled at once: the reader still sees what was there"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 32, 8, 128, 8000, [40, 60], scramble=False)
    want = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    cq, ck = dev(cu_q), dev(cu_k)
    with torch.cuda.stream(side):
        outs = [cache.attention(e, 1, q, k, v, cq, ck) for _ in range(8)]
    cache.free(e)
    f = cache.new()
    z = torch.zeros(2, 8000, 8, 128, dtype=BF, device="cuda")
    cache.extend(f, z, z)
    torch.cuda.synchronize()
    assert all(torch.equal(o, want) for o in outs)


def test_pages_given_up_on_several_streams(pc):
    """two forks on streams of their own share a page: whoever gives it up first may still read it when the other's stream takes
    the page for something else, so that stream waits"""
    cache = pc.PromptCache(1, 1, 64, 4, max_entries=6)
    home, s1, s2 = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()
    kv = torch.randn(1, 64, 1, 64, device="cuda", dtype=BF)
    parent = cache.new()
    cache.extend(parent, kv, kv)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        a = cache.fork(parent)[0]
    with torch.cuda.stream(s2):
        b = cache.fork(parent)[0]
    assert cache.table(a) == cache.table(b) == [0]
    cache.free(parent)
    q = torch.randn(1, 2, 64, device="cuda", dtype=BF)
    torch.cuda.synchronize()
    with torch.cuda.stream(s1):
        torch.cuda._sleep(20_000_000)                         # ~10 ms of s1 before it reads
        out = cache.attention(a, 0, q)
        cache.free(a)
        read = torch.cuda.Event()
        read.record()
    with torch.cuda.stream(s2):
        cache.free(b)
        c = cache.new()
        cache.extend(c, kv * 0, kv * 0)
        assert cache.table(c) == [0] and read.query()         # the host came back behind s1's reading
    torch.cuda.synchronize()
    w = torch.softmax(kv[0, :, 0].double() @ q[0].double().t() / 8, 0)
    o, m = w.t() @ kv[0, :, 0].double(), w.t() @ kv[0, :, 0].double().abs()
    close(out, o[None], m[None])
    # the same with a page that is moved: what a's stream reads stays until it is done
    cache.free(c)
    low = cache.new()
    cache.extend(low, kv, kv)
    with torch.cuda.stream(s2):
        up = cache.new()
        cache.extend(up, kv, kv)
        assert cache.table(up) == [1]
        with torch.cuda.stream(s1):
            x = cache.fork(up)[0]
            y = cache.fork(up)[0]
        cache.free(up)
        cache.free(x)                                         # (another stream's: waits)
    with torch.cuda.stream(s1):
        z = cache.fork(y)[0]
        cache.free(y)
        torch.cuda._sleep(20_000_000)
        out = cache.attention(z, 0, q)
    cache.free(low)
    assert cache.compact() == 1 and cache.table(z) == [0]
    with torch.cuda.stream(s1):
        again = cache.attention(z, 0, q)
    torch.cuda.synchronize()
    assert torch.equal(out, again)
    close(out, o[None], m[None])
    assert home == torch.cuda.current_stream()


def test_refusals(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [5])
    bad = [
        (ValueError, dict(q=q[0])), (ValueError, dict(q=q.half())), (ValueError, dict(q=q.cpu())), (ValueError, dict(q=q[..., :32])),
        (RuntimeError, dict(q=torch.zeros(5, 3, 64, dtype=BF, device="cuda"))), (ValueError, dict(k=k[:4])), (ValueError, dict(v=None)),
        (ValueError, dict(k=k[:, :1])), (ValueError, dict(cu_q=dev(cu_q).long())), (ValueError, dict(cu_q=dev([0]), cu_k=dev([0]))),
        (ValueError, dict(cu_q=None)), (ValueError, dict(cu_k=torch.tensor(cu_k, dtype=torch.int32))), (ValueError, dict(out=q.float())),
        (ValueError, dict(out=torch.empty(5, 4, 65, dtype=BF, device="cuda")[..., :64])), (ValueError, dict(scale=float("nan"))),
        (ValueError, dict(scale=-1.0)), (RuntimeError, dict(entry=e + 1)), (RuntimeError, dict(entry=-1)), (RuntimeError, dict(layer=2)),
        (RuntimeError, dict(layer=-1)), (ValueError, dict(q=q.clone().requires_grad_())),
    ]
    for kind, change in bad:
        a = dict(entry=e, layer=1, q=q, k=k, v=v, cu_q=dev(cu_q), cu_k=dev(cu_k))
        a.update(change)
        with pytest.raises(kind):
            cache.attention(**a)
    with torch.no_grad():
        assert cache.attention(e, 1, q.clone().requires_grad_(), k, v, dev(cu_q)).shape == q.shape
    t = torch.zeros(2, 3, 2, 64, dtype=BF, device="cuda")
    for kind, f in ((RuntimeError, lambda: cache.write(e, t, t, 68)), (RuntimeError, lambda: cache.write(e, t, t, -1)), (RuntimeError, lambda: cache.write(e, t, t, 0, layer=1)),
                    (ValueError, lambda: cache.extend(e, t[:1], t[:1])), (ValueError, lambda: cache.extend(e, t, t[:, :2])), (ValueError, lambda: cache.extend(e, t.half(), t.half())),
                    (RuntimeError, lambda: cache.free([e, e])), (RuntimeError, lambda: cache.free(99)), (ValueError, lambda: cache.fork(e, -1)),
                    (RuntimeError, lambda: cache.fork(e, 99)), (RuntimeError, lambda: cache.reserve(e, -1)), (RuntimeError, lambda: cache.resize(1)),
                    (ValueError, lambda: cache.resize(0)), (RuntimeError, lambda: cache.length(77))):
        with pytest.raises(kind):
            f()
    kid = cache.fork(e)[0]
    with pytest.raises(RuntimeError, match="share"):
        cache.write(kid, t, t, 0)
    cache.write(kid, t, t, 66)
    small = pc.PromptCache(1, 2, 64, 4, max_tokens=100)
    x = small.new()
    with pytest.raises(RuntimeError, match="at most 100"):
        small.reserve(x, 101)
    small.reserve(x, 100)
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)    # nothing of this has changed the prompt
    close(cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k)), o, b)


# ---------------------------------------------------------------------------------------------------------------
# calls at the edges
# ---------------------------------------------------------------------------------------------------------------
class OpenCapture:
    """another thread captures a stream in global mode while the body runs; `ended`: what hipStreamEndCapture returned"""

    def __init__(self, blocking=False):
        self.blocking = blocking

    def __enter__(self):
        import ctypes
        import threading
        hip, V = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
        self.leave, opened, side = threading.Event(), threading.Event(), torch.cuda.Stream().cuda_stream
        if self.blocking:
            made = V()
            assert hip.hipStreamCreate(ctypes.byref(made)) == 0
            side = made.value

        def run():
            self.began = hip.hipStreamBeginCapture(V(side), 0)
            opened.set()
            self.leave.wait(60)
            self.ended = hip.hipStreamEndCapture(V(side), ctypes.byref(V()))
            hip.hipGetLastError()

        self.thread = threading.Thread(target=run, daemon=True)
        self.thread.start()
        assert opened.wait(60) and self.began == 0
        return self

    def __exit__(self, *exc):
        self.leave.set()
        self.thread.join()


def test_captures_of_other_threads_are_left_alone(pc):
    """whatever waits for the device, allocates or clears works beside a capture in another thread, waits in earnest, and lets it be
    (torch's own allocator does not: what it hands out inside was held before)"""
    cache = pc.PromptCache(1, 1, 64, 4, max_entries=4)
    kv, q = torch.randn(1, 64, 1, 64, device="cuda", dtype=BF), torch.randn(1, 2, 64, device="cuda", dtype=BF)
    side, nothing, got = torch.cuda.Stream(), kv * 0, [torch.empty_like(q) for _ in range(3)]

    def read_elsewhere(e, out):                               # from here on whoever takes e's pages has to wait for `side`
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            torch.cuda._sleep(20_000_000)
            cache.attention(e, 0, q, out=out)

    low, e = cache.new(), cache.new()
    for x in (low, e):
        cache.extend(x, kv, kv)
    want = cache.attention(e, 0, q)
    read_elsewhere(e, got[0])
    torch.zeros((6, 1, 1, 2, 64, 64), dtype=BF, device="cuda")
    torch.cuda.synchronize()
    with OpenCapture() as c:
        read_elsewhere(e, got[0])
        cache.free(low)
        assert cache.compact() == 1 and cache.table(e) == [0]                     # waits for `side`
        read_elsewhere(e, got[1])
        cache.resize(6)
        read_elsewhere(e, got[2])
        cache.free(e)
        e = cache.new()
        cache.extend(e, nothing, nothing)
        raw = pc.c_void_p()                                                        # (pages that the library allocates and clears)
        pc._check(pc._Lib.get().mi_prompt_cache_create(pc.ctypes.byref(pc._Cfg(1, 1, 64, 1, 4, 2, 0)), 0, None, pc.ctypes.byref(raw)))
        pc._check(pc._Lib.get().mi_prompt_cache_resize(raw, None, 9, None))
        pc._check(pc._Lib.get().mi_prompt_cache_destroy(raw))
    assert c.ended == 0
    torch.cuda.synchronize()
    with OpenCapture(blocking=True) as c:                                          # (beside which the null stream may not be used)
        pc._check(pc._Lib.get().mi_prompt_cache_create(pc.ctypes.byref(pc._Cfg(1, 1, 64, 1, 4, 2, 0)), 0, None, pc.ctypes.byref(raw)))
        pc._check(pc._Lib.get().mi_prompt_cache_resize(raw, None, 9, side.cuda_stream))
        pc._check(pc._Lib.get().mi_prompt_cache_destroy(raw))
    assert c.ended == 0
    assert all(torch.equal(x, want) for x in got)
    assert (cache.pages[cache.table(e)[0]] == 0).all()


@pytest.mark.parametrize("captured", [False, True])
def test_a_page_that_was_shared_is_written_behind_its_readers(pc, captured):
    """a fork reads on a stream of its own and is freed there; its parent then writes the page that both held, eagerly or in a graph:
    behind the fork's reading"""
    cache = pc.PromptCache(1, 1, 64, 4, max_entries=6)
    kv, q = torch.randn(1, 64, 1, 64, device="cuda", dtype=BF), torch.randn(1, 2, 64, device="cuda", dtype=BF)
    nothing, out, side = kv * 0, torch.empty_like(q), torch.cuda.Stream()
    parent = cache.new()
    cache.extend(parent, kv, kv)
    want = cache.attention(parent, 0, q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kid = cache.fork(parent)[0]
        torch.cuda._sleep(20_000_000)                         # ~10 ms of this stream before it reads
        cache.attention(kid, 0, q, out=out)
        cache.free(kid)
        read = torch.cuda.Event()
        read.record()
    if captured:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            cache.write(parent, nothing, nothing, 0)
        for _ in range(3):
            g.replay()
    else:
        cache.write(parent, nothing, nothing, 0)
        assert read.query()                                   # the host came back behind the reading
    torch.cuda.synchronize()
    assert torch.equal(out, want)
    assert (cache.pages[0] == 0).all()


@pytest.mark.parametrize("length,at,n", [(200, 64, 10), (200, 0, 64), (128, 70, 5), (192, 10, 150), (130, 128, 2), (64, 0, 0)])
def test_a_captured_write_changes_its_own_entry_alone(pc, length, at, n):
    """forks taken between a graph's capture and its replays keep what they held: the pages the graph writes are theirs, not shared"""
    cache = pc.PromptCache(2, 1, 64, 40, max_entries=12)
    g = torch.Generator(device="cuda").manual_seed(length)
    new = lambda m: torch.randn(2, m, 1, 64, generator=g, device="cuda").to(BF)
    k, v, k2, v2 = new(length), new(length), new(n), new(n)
    e = cache.new()
    cache.extend(e, k, v)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cache.write(e, k2, v2, at)
    held = lambda x: [cache.pages[torch.tensor(cache.table(x), device="cuda")][:, :, 0, w].transpose(0, 1).reshape(2, -1, 64)[:, :length] for w in (0, 1)]
    same = lambda x, kk, vv: torch.equal(held(x)[0], kk[:, :, 0]) and torch.equal(held(x)[1], vv[:, :, 0])
    kids = cache.fork(e, 3) + cache.fork(e)
    grandkid = cache.fork(kids[0])[0]
    full, first = length // 64, at // 64 if n else 64
    for x in kids:                                            # what lies in front of the graph's pages is shared
        assert cache.table(x)[:min(full, first)] == cache.table(e)[:min(full, first)]
        assert not set(cache.table(x)[min(full, first):]) & set(cache.table(e))
    assert cache.table(grandkid)[:full] == cache.table(kids[0])[:full]
    for rep in range(3):
        graph.replay()
        kk, vv = k.clone(), v.clone()
        kk[:, at:at + n], vv[:, at:at + n] = k2, v2
        assert same(e, kk, vv) and all(same(x, k, v) for x in [*kids, grandkid]), rep
        k2.mul_(-1.5)
        if rep == 1:
            cache.compact()
    copy = cache.copy(e)
    assert set(cache.table(cache.fork(copy)[0])) & set(cache.table(copy)) == set(cache.table(copy)[:full])
    cache.free([e, copy, *kids])
    assert same(grandkid, k, v)
    again = cache.new()                                       # the entry's number used again: nothing of the graph's is left
    cache.extend(again, k, v)
    assert cache.table(cache.fork(again)[0])[:full] == cache.table(again)[:full]


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("prompt,lens", [(37, [10]), (100, [3, 1]), (2000, [1, 1, 1]), (300, [90, 40]), (64, [5])])
def test_an_infinity_in_the_prompts_last_value(pc, dtype, prompt, lens):
    """a page's rows behind the prompt's end weigh nothing, whatever the last token's value is: a row that sees an infinity gets it,
    with and without own keys, few rows and many, split or not"""
    for what in (math.inf, -math.inf, math.nan):
        cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, 8, 2, 128, prompt, lens)
        o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
        none = torch.zeros(0, 2, 128, dtype=dtype, device="cuda")
        o2, b2 = reference_many(q, pk, pv, none, none, cu_q, [0] * len(cu_q), True)
        bad = pv[None, prompt - 1:].clone()
        bad[..., 1, 5] = what                                 # key head 1, dim 5
        cache.write(e, pk[None, prompt - 1:].contiguous(), bad, prompt - 1, layer=1)
        dims = [d for d in range(128) if d != 5]
        for out, oo, bb in ((cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k)), o, b), (cache.attention(e, 1, q, None, None, dev(cu_q)), o2, b2)):
            close(out[:, :4], oo[:, :4], bb[:, :4])
            close(out[:, 4:][..., dims], oo[:, 4:][..., dims], bb[:, 4:][..., dims])
            assert (out[:, 4:, 5].isnan() if what != what else out[:, 4:, 5] == what).all(), what


@pytest.mark.parametrize("dtype", [BF, HF])
@pytest.mark.parametrize("prompt,lens,past", [(0, [30], None), (70, [9, 64, 5], None), (0, [90, 110], None), (2000, [1, 1], [70, 3])])
def test_an_infinity_among_the_own_values(pc, dtype, prompt, lens, past):
    """rows that see it get it (its probability is held exactly by one rounding, by both, or by none), the rows before it keep their
    values"""
    for what in (math.inf, -math.inf):
        for back in (1, 2, 4):                                # the text's last key, and ones that more of its rows see
            cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, dtype, 8, 2, 128, prompt, lens, past)
            o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
            at = cu_k[1] - back
            v[at, 1, 5] = what                                # key head 1, dim 5 of the first text
            out = cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k))
            sees = torch.zeros(q.shape, dtype=torch.bool, device="cuda")
            sees[max(0, cu_q[1] - back):cu_q[1], 4:, 5] = True
            assert (out[sees] == what).all(), (what, back)
            close(out[~sees], o[~sees], b[~sees])


class Between:
    """the library, with `what()` called once before or behind a function: another thread's call in that place"""

    def __init__(self, cache, name, what, before=False):
        self.lib, self.name, self.what, self.before = cache._lib, name, what, before

    def __getattr__(self, name):
        f = getattr(self.lib, name)
        if name != self.name or self.what is None:
            return f

        def call(*a):
            what, self.what = self.what, None
            if self.before:
                what()
            rc = f(*a)
            if not self.before:
                what()
            return rc
        return call


def test_a_prompt_that_grows_between_two_calls_of_one_attention(pc):
    """the workspace is asked for, another thread extends the entry: the attention of the longer prompt needs more of it, now and in
    the calls that follow"""
    _, _, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 8, 2, 128, 200, [2, 1])
    cache = pc.PromptCache(2, 2, 128, 200)
    e = cache.new()
    cache.extend(e, pk.expand(2, -1, -1, -1), pv.expand(2, -1, -1, -1))
    g = torch.Generator(device="cuda").manual_seed(3)
    k2, v2 = (torch.randn(2, 9000, 2, 128, generator=g, device="cuda").to(BF) for _ in range(2))
    cache._lib = Between(cache, "mi_prompt_attention_workspace", lambda: cache.extend(e, k2, v2))
    o, b = reference_many(q, torch.cat([pk, k2[1]]), torch.cat([pv, v2[1]]), k, v, cu_q, cu_k, True)
    for _ in range(3):
        close(cache.attention(e, 1, q, k, v, dev(cu_q), dev(cu_k)), o, b)


def test_forks_of_a_parent_that_grows_and_of_pages_that_move(pc):
    """the forks' tables are the forks', whatever another thread does to the parent or the pool before fork comes back"""
    for length in (64, 100, 200):
        cache = pc.PromptCache(1, 1, 64, 40)
        kv = torch.randn(1, 300, 1, 64, device="cuda").to(BF)
        low, e = cache.new(), cache.new()
        cache.extend(low, kv[:, :70], kv[:, :70])
        cache.extend(e, kv[:, :length], kv[:, :length])

        def ask(x):                                           # the library's own answer
            t, n = (pc.c_int32 * 40)(), pc.c_int32()
            pc._check(pc._Lib.get().mi_prompt_cache_entry(cache._h, x, pc.ctypes.byref(n), t, 40))
            return t[:-(-n.value // 64)]

        cache._lib = Between(cache, "mi_prompt_cache_entry", lambda: cache.extend(e, kv, kv), before=True)
        kids = cache.fork(e, 3)
        assert [cache.table(x) for x in kids] == [ask(x) for x in kids]
        assert [cache.length(x) for x in kids] == [length] * 3
        cache._lib = Between(cache, "mi_prompt_cache_fork", lambda: (cache.free(low), cache.compact()))
        kids += cache.fork(kids[0], 2)
        assert [cache.table(x) for x in kids] == [ask(x) for x in kids]

        class Late(dict):                                     # .. and where the move comes just before the tables are noted
            def update(self, known):
                cache.free(kids[1])
                cache.compact()
                super().update(known)

        cache._tables = Late(cache._tables)
        kids += cache.fork(kids[0], 2)
        del kids[1]
        assert [cache.table(x) for x in kids] == [ask(x) for x in kids]


@pytest.mark.parametrize("tokens,heads", [(1, 6), (1, 1), (5, 1), (2, 6)])
def test_axes_of_length_one_with_odd_strides(pc, tokens, heads):
    """one token, or one head, cut from a padded buffer: a stride that nothing is reached by may be anything"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, heads, 1, 64, 70, [tokens])
    odd = lambda t: torch.nn.functional.pad(torch.cat([t, t]).flatten(1), (0, 4))[:, :t[0].numel()].unflatten(1, t.shape[1:])[:len(t)]
    one = lambda t: t.contiguous().as_strided(t.shape, (t.stride(0), 5, 1)) if t.shape[1] == 1 else t
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    for cut in (odd, one):
        q1, k1, v1 = cut(q), cut(k), cut(v)
        assert torch.equal(q1, q) and (cut is one or q1.stride(0) % 8)
        close(cache.attention(e, 1, q1, k1, v1), o, b)
        out = one(torch.zeros_like(q)) if tokens > 1 else odd(torch.zeros_like(q))
        assert cache.attention(e, 1, q1, k1, v1, out=out) is out
        close(out, o, b)


def test_an_output_that_is_broadcast_is_refused(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [3])
    for out in (torch.zeros_like(q[:1]).expand(3, -1, -1), torch.zeros_like(q[:, :1]).expand(-1, 4, -1)):
        with pytest.raises(ValueError, match="broadcast"):
            cache.attention(e, 1, q, k, v, out=out)
    one = torch.zeros_like(q[:1, :1]).expand(1, 1, 64)
    cache2, e2, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 1, 1, 64, 70, [1])
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    close(cache2.attention(e2, 1, q, k, v, out=one), o, b)


def test_gradients_are_refused_not_lost(pc):
    """tensors that need one, forward-mode tangents, and an output that a backward pass has saved"""
    import torch.autograd.forward_ad as forward
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [3])
    want = cache.attention(e, 1, q, k, v)
    t = torch.randn(2, 5, 2, 64, device="cuda").to(BF)
    leaf = lambda x: x.clone().requires_grad_()
    for f in (lambda: cache.extend(e, leaf(t), t), lambda: cache.extend(e, t, leaf(t)), lambda: cache.write(e, leaf(t), t, 65), lambda: cache.write(e, t, leaf(t) * 2, 65),
              lambda: cache.attention(e, 1, leaf(q), k, v), lambda: cache.attention(e, 1, q, leaf(k), v), lambda: cache.attention(e, 1, q, k, leaf(v)),
              lambda: cache.attention(e, 1, q, k, v, out=leaf(q)), lambda: torch.func.vjp(lambda x: cache.attention(e, 1, x, k, v), q)):
        with pytest.raises(ValueError, match="gradient"):
            f()
    with torch.no_grad(), forward.dual_level():
        dual = lambda x: forward.make_dual(x, torch.ones_like(x))
        for f in (lambda: cache.extend(e, dual(t), t), lambda: cache.write(e, t, dual(t), 65), lambda: cache.attention(e, 1, dual(q), k, v),
                  lambda: cache.attention(e, 1, q, k, dual(v))):
            with pytest.raises(ValueError, match="tangent"):
                f()
        assert torch.equal(cache.attention(e, 1, q, k, v), want)
    with pytest.raises(ValueError, match="tangent"):
        torch.func.jvp(lambda x: cache.attention(e, 1, x, k, v), (q,), (q,))
    assert cache.length(e) == 70
    out, w = torch.zeros_like(q), leaf(q)
    loss = (out * w).sum()
    cache.attention(e, 1, q, k, v, out=out)
    with pytest.raises(RuntimeError, match="inplace"):
        loss.backward()
    for mode in (torch.no_grad, torch.inference_mode):
        with mode():
            assert torch.equal(cache.attention(e, 1, leaf(q), k, v, out=torch.empty_like(q)), want)
    with torch.no_grad():
        cache.extend(e, leaf(t), t)
    assert cache.length(e) == 75


def test_the_per_thread_stream_is_another_one_in_every_thread(pc):
    """a page that one thread gives up on its per-thread stream, where it is still read, and another takes on its own: the same
    handle, not the same stream"""
    import threading
    cache = pc.PromptCache(1, 1, 64, 1, max_entries=1)
    kv, q = torch.randn(1, 64, 1, 64, device="cuda", dtype=BF), torch.randn(1, 2, 64, device="cuda", dtype=BF)
    nothing, out, steps, done = kv * 0, torch.empty_like(q), [], [threading.Event(), threading.Event()]
    e = cache.new()
    cache.extend(e, kv, kv)
    want = cache.attention(e, 0, q)
    cache.free(e)
    torch.cuda.synchronize()

    def first():
        with torch.cuda.stream(torch.cuda.ExternalStream(2)):     # hipStreamPerThread
            x = cache.new()
            cache.extend(x, kv, kv)
            torch.cuda._sleep(20_000_000)
            cache.attention(x, 0, q, out=out)
            cache.free(x)
            steps.append(torch.cuda.Event())
            steps[0].record()
        done[0].set()
        done[1].wait(60)                                      # (the thread and its stream live until the other is done)

    def second():
        done[0].wait(60)
        with torch.cuda.stream(torch.cuda.ExternalStream(2)):
            x = cache.new()
            cache.extend(x, nothing, nothing)
            steps.append(steps[0].query())
        done[1].set()

    ts = [threading.Thread(target=f) for f in (first, second)]
    [t.start() for t in ts]
    [t.join() for t in ts]
    torch.cuda.synchronize()
    assert steps[1] is True and torch.equal(out, want) and (cache.pages == 0).all()


def test_numbers_beyond_32_bits_are_refused(pc):
    """ctypes would cut them: reserve(e, 2^32 + 5) was five tokens, write(start=2^32) the first one"""
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [3])
    want, big = cache.attention(e, 1, q, k, v), 1 << 32
    t = torch.zeros(2, 3, 2, 64, dtype=BF, device="cuda")
    for f in (lambda: cache.reserve(e, big + 5), lambda: cache.reserve(e + big, 5), lambda: cache.write(e, t, t, big), lambda: cache.write(e, t, t, 0, layer=big),
              lambda: cache.write(e + big, t, t, 0), lambda: cache.extend(e + big, t, t), lambda: cache.fork(e + big), lambda: cache.copy(e - big),
              lambda: cache.free(e + big), lambda: cache.free([e, e - big]), lambda: cache.resize(big + 40), lambda: cache.length(e + big), lambda: cache.table(e + big)):
        with pytest.raises(ValueError, match="int32"):
            f()
    with pytest.raises(RuntimeError, match="max_entries"):
        cache.fork(e, 1 << 40)
    for entry, layer in ((e + big, 1), (e, 1 + big), (e - big, 1)):
        with pytest.raises(RuntimeError, match="no entry"):
            cache.attention(entry, layer, q, k, v)
    assert cache.length(e) == 70 and torch.equal(cache.attention(e, 1, q, k, v), want)
    many = k[:1, :, :].as_strided((2 ** 31 - 8, 2, 64), (0, 64, 1))
    with pytest.raises(RuntimeError, match="2\\^31 keys"):
        cache.attention(e, 1, q, many, many, dev([0, 3]), dev([0, 3]))


def test_a_captured_write_waits_for_the_readers_of_a_page_that_was_shared(pc):
    """with the reading still under way when the write is captured (torch's own capture would have waited for it)"""
    import ctypes
    hip, V = ctypes.CDLL("libamdhip64.so"), ctypes.c_void_p
    cache = pc.PromptCache(1, 1, 64, 4, max_entries=6)
    kv, q = torch.randn(1, 64, 1, 64, device="cuda", dtype=BF), torch.randn(1, 2, 64, device="cuda", dtype=BF)
    nothing, out, side, s = kv * 0, torch.empty_like(q), torch.cuda.Stream(), torch.cuda.Stream()
    parent = cache.new()
    cache.extend(parent, kv, kv)
    want = cache.attention(parent, 0, q)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        kid = cache.fork(parent)[0]
        torch.cuda._sleep(20_000_000)
        cache.attention(kid, 0, q, out=out)
        cache.free(kid)
        read = torch.cuda.Event()
        read.record()
    graph, exe = V(), V()
    assert hip.hipStreamBeginCapture(V(s.cuda_stream), 2) == 0
    with torch.cuda.stream(s):
        cache.write(parent, nothing, nothing, 0)
        done = read.query()
    assert hip.hipStreamEndCapture(V(s.cuda_stream), ctypes.byref(graph)) == 0 and done
    assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, ctypes.c_size_t(0)) == 0
    for _ in range(3):
        assert hip.hipGraphLaunch(exe, V(s.cuda_stream)) == 0
        torch.cuda.synchronize()
        assert torch.equal(out, want) and (cache.pages[0] == 0).all()
        cache.pages[0] = 1
    assert hip.hipGraphExecDestroy(exe) == 0 and hip.hipGraphDestroy(graph) == 0


def test_the_library_refuses_an_output_whose_rows_are_the_same_memory(pc):
    cache, e, pk, pv, q, k, v, cu_q, cu_k = make(pc, BF, 4, 2, 64, 70, [3])
    out = torch.zeros_like(q)
    for o_token, o_head, ok in ((256, 64, True), (0, 64, False), (256, 0, False)):
        a = pc._ATTN.pack(e, 1, 4, 3, 3, 1, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), 256, 64, 128, 64, 128, 64, o_token, o_head, 0, 0, 1, 0.125, 0, 0, 0, 0)
        rc = pc._Lib.get().mi_prompt_attention(cache._h, a, None)
        assert (rc == 0) == ok and (ok or b"same memory" in pc._Lib.get().mi_enc_last_error())
    o, b = reference_many(q, pk, pv, k, v, cu_q, cu_k, True)
    torch.cuda.synchronize()
    close(out, o, b)


def test_several_threads_on_one_cache(pc):
    """four threads store, fork, read, copy, write and free prompts on streams of their own while a fifth moves pages: every output is
    what its prompt gives"""
    import threading
    cache = pc.PromptCache(2, 2, 64, 120, max_entries=100, max_tokens=64 * 20)
    rng = np.random.default_rng(5)
    g = torch.Generator(device="cuda").manual_seed(5)
    kv = [[torch.randn(2, n, 2, 64, generator=g, device="cuda").to(BF) for _ in range(2)] for n in (1, 63, 64, 130, 200, 320, 700)]
    q = torch.randn(5, 4, 64, generator=g, device="cuda").to(BF)
    own = [torch.randn(5, 2, 64, generator=g, device="cuda").to(BF) for _ in range(2)]
    want = []
    for k, v in kv:
        e = cache.new()
        cache.extend(e, k, v)
        want.append(cache.attention(e, 1, q, *own))
        cache.free(e)
    torch.cuda.synchronize()
    outs, errors, stop = [], [], threading.Event()

    def run(seed):
        r = np.random.default_rng(seed)
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                held = []
                for _ in range(150):
                    op = r.integers(0, 6)
                    try:
                        if op < 2 or not held:
                            i, e = int(r.integers(0, len(kv))), cache.new()
                            held.append((e, i))
                            k, v = kv[i]
                            half = k.shape[1] // 2
                            cache.extend(e, k[:, :half], v[:, :half])
                            cache.extend(e, k[:, half:], v[:, half:])
                        else:
                            e, i = held[int(r.integers(0, len(held)))]
                            if op == 2:
                                held += [(c, i) for c in cache.fork(e, int(r.integers(1, 4)))]
                            elif op == 3:
                                held.append((cache.copy(e), i))
                            elif op == 4:
                                k, v = kv[i]
                                last = (k.shape[1] - 1) // 64 * 64
                                if k.shape[1] % 64:                   # (the same tokens once more, in the page that is the entry's own)
                                    cache.write(e, k[:, last:], v[:, last:], last)
                            else:
                                held.remove((e, i))
                                cache.free(e)
                    except RuntimeError as err:                   # a full pool: half of what is held goes
                        assert "free" in str(err) or "max_entries" in str(err), err
                        bad = [h for h in held if cache.length(h[0]) != kv[h[1]][0].shape[1]]
                        gone = bad + [h for h in held if h not in bad][::2]
                        cache.free([e for e, _ in gone])
                        held = [h for h in held if h not in gone]
                        continue
                    for e, i in held[-2:]:
                        outs.append((i, cache.attention(e, 1, q, *own)))
                cache.free([e for e, _ in held])
        except Exception as err:                                  # pragma: no cover
            errors.append(err)

    def move():
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not stop.is_set():
                    cache.compact()
                    if rng.random() < 0.2:
                        try:
                            cache.resize(int(rng.integers(120, 140)))
                        except RuntimeError as err:               # (fewer than are used)
                            assert "in use" in str(err), err
        except Exception as err:                                  # pragma: no cover
            errors.append(err)

    ts = [threading.Thread(target=run, args=(s,)) for s in range(4)]
    mover = threading.Thread(target=move)
    [t.start() for t in ts + [mover]]
    [t.join() for t in ts]
    stop.set()
    mover.join()
    torch.cuda.synchronize()
    assert not errors, errors
    assert len(outs) > 500 and all(torch.equal(o, want[i]) for i, o in outs)
    assert cache.used_pages == 0
