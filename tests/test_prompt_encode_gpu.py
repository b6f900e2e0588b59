"""GPU tests of encoding behind a cached prompt (SentenceTransformer.cache_prompt -> mi_encoder_encode_prompted): the embeddings
of prompt + text against the fp32 oracle (cosine within 1e-3, the encoder's bound) and against the uncached path, through every
regime of token counts the encoder has."""
from dataclasses import replace

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def st():
    import abstracts_search_amd.sentence_transformers as m
    return m


@pytest.fixture(autouse=True)
def cached_whatever_it_costs(st, monkeypatch):
    monkeypatch.setattr(st.SentenceTransformer, "prompt_break_even", (0, 0, 0))


@pytest.fixture(scope="module")
def tiny():
    from oracle import encoder_oracle as E
    cfg = replace(E.TINY, causal=True, max_seq_len=400)
    return cfg, E.synth_weights(cfg, 11)


def oracle_encode(cfg, W, toks):
    from oracle import encoder_oracle as E
    cu = np.concatenate([[0], np.cumsum([len(t) for t in toks])])
    return E.encode(cfg, W, np.concatenate(toks), cu, True).numpy()


def same(a, b, cos):
    assert np.isfinite(a).all() and np.isfinite(b).all()
    c = (a * b).sum(1) / np.maximum(np.linalg.norm(a, axis=1) * np.linalg.norm(b, axis=1), 1e-30)
    assert c.min() > 1 - cos, c.min()


@pytest.mark.parametrize("prompt_len", [1, 7, 63, 64, 65, 200])
@pytest.mark.parametrize("lens", [[1], [9], [30], [17, 1, 20], [1] * 40, [60, 3, 90], [120, 77, 150, 31]])
def test_prompted_against_the_oracle(st, tiny, prompt_len, lens):
    cfg, W = tiny
    rng = np.random.default_rng(prompt_len * 100 + len(lens))
    prompt = rng.integers(0, cfg.vocab_size, prompt_len).tolist()
    toks = [prompt + rng.integers(0, cfg.vocab_size, n).tolist() for n in lens]
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    plain = model.encode_tokens(toks, normalize_embeddings=True)
    raw = model.encode_tokens(toks)
    p0 = st.debug_counter("prompted_passes")
    assert model.cache_prompt(prompt) == prompt_len
    e = model.encode_tokens(toks, normalize_embeddings=True)
    assert st.debug_counter("prompted_passes") == p0 + 2         # the prompt's own pass and one for the texts
    ref = oracle_encode(cfg, W, toks)
    same(e, ref, 1e-3)
    same(e, plain, 1e-3)
    same(model.encode_tokens(toks), raw, 1e-3)
    assert np.allclose(np.linalg.norm(model.encode_tokens(toks), axis=1), np.linalg.norm(raw, axis=1), rtol=2e-2)
    assert np.array_equal(e, model.encode_tokens(toks, normalize_embeddings=True))     # the same bits every time
    model.drop_prompts()
    p1 = st.debug_counter("prompted_passes")
    assert np.array_equal(plain, model.encode_tokens(toks, normalize_embeddings=True))
    assert st.debug_counter("prompted_passes") == p1


def test_few_texts_behind_a_short_prompt_go_without_it(st, tiny, monkeypatch):
    """where a pass over all tokens costs no more than one over the texts' own, the cache is not used (and the result is the plain one's)"""
    cfg, W = tiny
    monkeypatch.undo()
    assert st.SentenceTransformer.prompt_break_even == (48, 64, 384)
    rng = np.random.default_rng(4)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    ids = lambda n: rng.integers(0, cfg.vocab_size, n).tolist()
    short, long = ids(20), ids(100)
    #                  texts             used
    for prompt, lens, cached in ((short, [11], False), (short, [28], False), (short, [29], True), (short, [15] * 8, False), (short, [60], True),
                                 (short, [14] * 16, True), (long, [5], True), (long, [65], False), (long, [64], True), (long, [60] * 6, True)):
        toks = [prompt + ids(n) for n in lens]
        plain = model.encode_tokens(toks, normalize_embeddings=True)
        model.cache_prompt(prompt)
        p0 = st.debug_counter("prompted_passes")
        got = model.encode_tokens(toks, normalize_embeddings=True)
        assert st.debug_counter("prompted_passes") == p0 + cached, (len(prompt), lens)
        same(got, plain, 1e-3)
        assert cached or np.array_equal(got, plain)
        model.drop_prompts()
    # groups of either kind in one call, results in their places
    model.cache_prompt(short)
    model.cache_prompt(long)
    toks = [short + ids(10), ids(30), long + ids(7), ids(3), long + ids(2)]
    p0 = st.debug_counter("prompted_passes")
    same(model.encode_tokens(toks, normalize_embeddings=True), oracle_encode(cfg, W, toks), 1e-3)
    assert st.debug_counter("prompted_passes") == p0 + 1


@pytest.mark.parametrize("knob", [None, "MI_NO_FEW", "MI_NO_FEW_QKV8", "MI_NO_ROPE_FUSE"])
def test_prompted_at_the_real_width(st, knob, monkeypatch):
    """two layers of stella's width, causal: the query-time path, the few-hundred-token tiles and the many-token slab GEMMs (whose
    Q and K leave with their rotary pairs interleaved), one prompt computed by one of them and read by all"""
    if knob:
        monkeypatch.setenv(knob, "1")
    cfg = dict(st.STELLA_EN_1_5B_V5, vocab_size=2048, n_layers=2, causal=True, max_seq_len=700)
    g = torch.Generator(device="cuda").manual_seed(5)
    H, I, hd = cfg["hidden"], cfg["intermediate"], cfg["head_dim"]
    qc, kc = cfg["n_heads"] * hd, cfg["n_kv_heads"] * hd
    rnd = lambda shape, scale: (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()
    W = {"embed_tokens.weight": rnd((2048, H), 0.3), "norm.weight": torch.ones(H, device="cuda"), "dense.weight": rnd((1024, H), H ** -0.5),
         "dense.bias": torch.zeros(1024, device="cuda")}
    for l in range(2):
        p = f"layers.{l}."
        W.update({p + "input_layernorm.weight": torch.ones(H, device="cuda"), p + "post_attention_layernorm.weight": torch.ones(H, device="cuda"),
                  p + "self_attn.q_proj.weight": rnd((qc, H), H ** -0.5), p + "self_attn.q_proj.bias": rnd((qc,), 0.3),
                  p + "self_attn.k_proj.weight": rnd((kc, H), H ** -0.5), p + "self_attn.k_proj.bias": rnd((kc,), 0.3),
                  p + "self_attn.v_proj.weight": rnd((kc, H), H ** -0.5), p + "self_attn.v_proj.bias": rnd((kc,), 0.1),
                  p + "self_attn.o_proj.weight": rnd((H, qc), qc ** -0.5), p + "mlp.gate_proj.weight": rnd((I, H), H ** -0.5),
                  p + "mlp.up_proj.weight": rnd((I, H), H ** -0.5), p + "mlp.down_proj.weight": rnd((H, I), I ** -0.5)})
    model = st.SentenceTransformer(config=cfg, weights=W)
    rng = np.random.default_rng(6)
    for prompt_len in (20, 130, 333):                             # computed by the query-time path, by the mid and by the slab tiles
        prompt = rng.integers(0, 2048, prompt_len).tolist()
        batches = [[rng.integers(0, 2048, int(n)).tolist() for n in lens] for lens in
                   ([12], [40], [8, 20, 9], rng.integers(5, 60, 12), rng.integers(30, 300, 60))]
        plain = [model.encode_tokens([prompt + t for t in b], normalize_embeddings=True) for b in batches]
        model.cache_prompt(prompt)
        for b, want in zip(batches, plain):
            same(model.encode_tokens([prompt + t for t in b], normalize_embeddings=True), want, 2e-4)
        model.drop_prompts()


def test_prompts_that_begin_alike_and_texts_without_one(st, tiny):
    """prompts that extend each other (shared pages), texts behind each, behind none, and one that is a cached prompt itself"""
    cfg, W = tiny
    rng = np.random.default_rng(3)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    a = rng.integers(0, cfg.vocab_size, 100).tolist()
    b, c = a + rng.integers(0, cfg.vocab_size, 70).tolist(), a + rng.integers(0, cfg.vocab_size, 28).tolist()
    other = rng.integers(0, cfg.vocab_size, 30).tolist()
    text = lambda n: rng.integers(0, cfg.vocab_size, n).tolist()
    toks = [b + text(10), other + text(4), a + text(50), c + text(3), a, b, other, c + text(150), [5], b + text(1), a[:40]]
    ref = oracle_encode(cfg, W, toks)
    for order in ([a, b, c, other], [b, other, a, c], [c, b, a]):
        for p in order:
            model.cache_prompt(p)
        model.cache_prompt(order[0])                              # again: nothing to do
        for bs in (None, 2):
            same(model.encode_tokens(toks, normalize_embeddings=True, batch_size=bs), ref, 1e-3)
        model.drop_prompts()
    # many prompts: the pool grows, and what is cached stays right
    grown = [a + text(60 + i) for i in range(30)]
    for p in grown:
        model.cache_prompt(p)
    toks = [p + text(5) for p in grown]
    same(model.encode_tokens(toks, normalize_embeddings=True), oracle_encode(cfg, W, toks), 1e-3)


def test_prompted_on_other_streams_and_threads(st, tiny):
    import threading
    cfg, W = tiny
    rng = np.random.default_rng(8)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    prompt = rng.integers(0, cfg.vocab_size, 150).tolist()
    work = [[prompt + rng.integers(0, cfg.vocab_size, int(n)).tolist() for n in rng.integers(1, 90, 6)] for _ in range(4)]
    model.cache_prompt(prompt)
    want = [model.encode_tokens(w, normalize_embeddings=True) for w in work]
    got, errors = [None] * 4, []

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(5):
                    got[i] = model.encode_tokens(work[i], normalize_embeddings=True)
        except Exception as e:                                    # pragma: no cover
            errors.append(e)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    for k in range(6):                                            # prompts come meanwhile, and the pool grows
        model_ids = rng.integers(0, cfg.vocab_size, 350).tolist()
        n = st.c_int32()
        a = np.asarray(model_ids, np.int32)
        st._check(st._Lib.get().mi_encoder_cache_prompt(model._h, len(a), a.ctypes.data, st.ctypes.byref(n), None))
        if k % 2:
            st._check(st._Lib.get().mi_encoder_drop_prompt(model._h, n.value))
    [t.join() for t in ts]
    assert not errors, errors
    for g, w in zip(got, want):
        assert np.array_equal(g, w)


def test_encode_with_a_prompt_string(st, tiny):
    """encode(prompt_name=..) on a model with a tokenizer: the cached prompt is found behind the string, also where the tokenizer
    appends its own token to every text"""
    from tokenizers import Tokenizer, models, pre_tokenizers
    cfg, W = tiny
    words = ["[UNK]", "Instruct", ":", "find", "papers", "Query", "a", "0", "The", "(", "x"] + [f"w{i}" for i in range(40)] + ["</s>"]
    tk = Tokenizer(models.WordLevel({w: i for i, w in enumerate(words)}, unk_token="[UNK]"))
    tk.pre_tokenizer = pre_tokenizers.Whitespace()
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W, tokenizer=tk, prompts={"q": "Instruct: find papers\nQuery: "})
    model._host_tok.eos_id = words.index("</s>")
    texts = ["w1 w2", "w3", "w9 w9 w9 w30 a"]
    plain = model.encode(texts, prompt_name="q", normalize_embeddings=True)
    assert model.cache_prompt(prompt_name="q") == 6
    p0 = st.debug_counter("prompted_passes")
    same(model.encode(texts, prompt_name="q", normalize_embeddings=True), plain, 1e-3)
    assert st.debug_counter("prompted_passes") == p0 + 1
    one = model.encode("w1 w2", prompt_name="q", normalize_embeddings=True)
    assert np.array_equal(one, plain[0]) or (one * plain[0]).sum() > 1 - 1e-3
    same(model.encode(texts, normalize_embeddings=True), oracle_encode(cfg, W, model.tokenize(texts)), 1e-3)


def test_refusals(st, tiny):
    cfg, W = tiny
    two = replace(cfg, causal=False)
    both = st.SentenceTransformer(config=two.to_dict(), weights=W)
    with pytest.raises(ValueError, match="causal"):
        both.cache_prompt([1, 2, 3])
    lib, n, a = st._Lib.get(), st.c_int32(), np.asarray([1, 2, 3], np.int32)
    assert lib.mi_encoder_cache_prompt(both._h, 3, a.ctypes.data, st.ctypes.byref(n), None) != 0 and b"causal" in lib.mi_enc_last_error()
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    for bad in ([], [1] * 400):
        with pytest.raises(ValueError):
            model.cache_prompt(bad)
    with pytest.raises(RuntimeError, match="out of range"):
        model.cache_prompt([1, cfg.vocab_size])
    with pytest.raises(ValueError, match="not found"):
        model.cache_prompt(prompt_name="nope")
    model.cache_prompt([1] * 390)
    h = next(iter(model._cached_prompts.values()))
    out, ids = torch.empty(1, 64, device="cuda"), np.ones(11, np.int32)
    run = lambda handle, ids: lib.mi_encoder_encode_prompted(model._h, handle, 1, ids.ctypes.data, np.asarray([0, len(ids)], np.int32).ctypes.data, 1,
                                                              out.data_ptr(), None, None)
    assert run(h, ids) != 0 and b"longer than max_seq_len" in lib.mi_enc_last_error()
    assert run(h + 1, ids[:3]) != 0 and b"no such cached prompt" in lib.mi_enc_last_error()
    assert run(h, ids[:10]) == 0
    assert lib.mi_encoder_drop_prompt(model._h, h + 1) != 0
    model.load_weights({"norm.weight": W["norm.weight"]})         # (drops the prompts)
    assert run(h, ids[:3]) != 0 and not model._cached_prompts
    torch.cuda.synchronize()


def test_prompts_come_and_go_beside_a_capture(st, tiny):
    """another thread's open capture neither stops a prompt from being cached or dropped nor ends; what is dropped leaves the pool (of
    512 entries: a third round would find it full)"""
    from test_prompt_cache_gpu import OpenCapture
    cfg, W = tiny
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    model.cache_prompt([1, 2, 3])
    side = torch.cuda.Stream()
    for _ in range(3):
        for i in range(255):
            model.cache_prompt([5, i % 50, i // 50])
        with torch.cuda.stream(side):                         # read on another stream: its pages are waited for
            model.encode_tokens([[5, 0, 0, 7, 9], [5, 1, 0, 3]])
        with OpenCapture() as c:
            model.drop_prompts()
            model.cache_prompt([1, 2, 3])
        assert c.ended == 0
    assert np.isfinite(model.encode_tokens([[1, 2, 3, 4]])).all()


def test_prompts_come_and_go_while_others_encode(st, tiny):
    """cache_prompt and drop_prompts on one thread, encode_tokens on four: every encode answers, with the prompt's tokens where the prompt
    has gone meanwhile"""
    import threading
    cfg, W = tiny
    rng = np.random.default_rng(12)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    ids = lambda n: rng.integers(0, cfg.vocab_size, int(n)).tolist()
    prompts = [ids(n) for n in (5, 30, 64, 100, 150)]
    prompts += [prompts[3] + ids(20), prompts[1] + ids(1)]
    work = [[prompts[(i + j) % 7] + ids(rng.integers(1, 60)) for j in range(7)] for i in range(4)]
    want = [model.encode_tokens(w, normalize_embeddings=True) for w in work]
    got, errors, stop = [[] for _ in work], [], threading.Event()

    def run(i):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                while not stop.is_set() or not got[i]:
                    got[i].append(model.encode_tokens(work[i], normalize_embeddings=True))
        except Exception as e:                                    # pragma: no cover
            errors.append(e)

    ts = [threading.Thread(target=run, args=(i,)) for i in range(4)]
    [t.start() for t in ts]
    try:
        for k in range(40):
            for p in prompts[k % 3:]:
                model.cache_prompt(p)
            for n in range(20):                                   # (many at a time: the table of prompts changes under every lookup)
                model.cache_prompt([n, k % 50, 1, 2])
            if k % 2:
                model.drop_prompts()
    finally:
        stop.set()
        [t.join() for t in ts]
    assert not errors, errors
    for g, w in zip(got, want):
        assert g
        for e in g:
            same(e, w, 1e-3)


def test_two_threads_cache_the_same_prompt(st, tiny):
    """one of them runs it, and dropping the prompts drops all there are"""
    import threading
    cfg, W = tiny
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    p0 = st.debug_counter("prompted_passes")
    for k in range(10):
        ts = [threading.Thread(target=model.cache_prompt, args=([k, 1, 2, 3],)) for _ in range(4)]
        [t.start() for t in ts]
        [t.join() for t in ts]
    assert st.debug_counter("prompted_passes") == p0 + 10
    handles = list(model._cached_prompts.values())
    model.drop_prompts()
    assert len(handles) == 10 and not model._cached_prompts
    for h in handles:
        assert st._Lib.get().mi_encoder_drop_prompt(model._h, h) != 0


def test_a_prompt_the_library_dropped_is_encoded_in_full(st, tiny):
    cfg, W = tiny
    rng = np.random.default_rng(2)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    prompt = rng.integers(0, cfg.vocab_size, 80).tolist()
    toks = [prompt + rng.integers(0, cfg.vocab_size, n).tolist() for n in (3, 40, 9, 1)] + [[4, 5]]
    plain = model.encode_tokens(toks, normalize_embeddings=True)
    model.cache_prompt(prompt)
    st._check(st._Lib.get().mi_encoder_drop_prompt(model._h, next(iter(model._cached_prompts.values()))))
    for bs in (None, 2):
        same(model.encode_tokens(toks, normalize_embeddings=True, batch_size=bs), plain, 1e-3)
    assert not model._cached_prompts
    model.cache_prompt(prompt)
    p0 = st.debug_counter("prompted_passes")
    same(model.encode_tokens(toks, normalize_embeddings=True), plain, 1e-3)
    assert st.debug_counter("prompted_passes") == p0 + 1
    model.load_weights({})                                        # (nothing is loaded: the library would have kept them)
    assert not model._cached_prompts
    for _ in range(2):                                            # (of 256 prompts)
        for i in range(200):
            model.cache_prompt([7, i % 60, i // 60])
        model.load_weights({})


def test_a_prompt_cached_while_weights_load_is_of_the_new_ones(st, tiny):
    """through the C entries: whatever prompt is left when both threads are done gives what its tokens give"""
    import threading
    cfg, W = tiny
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    lib, E = st._Lib.get(), torch.from_numpy(np.asarray(W["embed_tokens.weight"], np.float32))
    E = [E.contiguous(), (E * 1.5).contiguous()]
    shape = (st.c_int64 * 2)(*E[0].shape)
    handles, errors = {}, []

    def load():
        for i in range(60):
            if lib.mi_encoder_load_tensor(model._h, b"embed_tokens.weight", E[i % 2].data_ptr(), 0, shape, 2):
                errors.append(lib.mi_enc_last_error())

    t = threading.Thread(target=load)
    t.start()
    k = 0
    while t.is_alive() or k < 5:
        a, n = np.asarray([1 + k % 50, 2, 3 + k // 50], np.int32), st.c_int32()
        if lib.mi_encoder_cache_prompt(model._h, 3, a.ctypes.data, st.ctypes.byref(n), None):
            errors.append(lib.mi_enc_last_error())
            break
        handles[n.value] = a.tolist()
        k += 1
    t.join()
    assert not errors, errors
    left = 0
    for h, p in handles.items():
        toks = [p + [9, 4, 7], p + [3]]
        out, ids = torch.empty(2, 64, device="cuda"), np.asarray([9, 4, 7, 3], np.int32)
        if lib.mi_encoder_encode_prompted(model._h, h, 2, ids.ctypes.data, np.asarray([0, 3, 4], np.int32).ctypes.data, 1, out.data_ptr(), None, None):
            assert b"no such cached prompt" in lib.mi_enc_last_error()
            continue
        torch.cuda.synchronize()
        left += 1
        same(out.cpu().numpy(), model.encode_tokens(toks, normalize_embeddings=True), 1e-3)
    assert left


@pytest.mark.parametrize("pass_tokens", [0, 1000])
def test_many_prompts_in_one_call(st, tiny, monkeypatch, pass_tokens):
    """thirty prompts with a text each: in a pass apiece behind their pages, or together with their tokens; the same either way"""
    cfg, W = tiny
    monkeypatch.setattr(st.SentenceTransformer, "prompt_pass_tokens", pass_tokens)
    rng = np.random.default_rng(21)
    model = st.SentenceTransformer(config=cfg.to_dict(), weights=W)
    ids = lambda n: rng.integers(0, cfg.vocab_size, n).tolist()
    base = ids(100)
    prompts = [base + ids(60 + i) for i in range(30)]
    toks = [p + ids(5) for p in prompts] + [prompts[3] + ids(30), ids(12)]
    for p in prompts:
        model.cache_prompt(p)
    p0 = st.debug_counter("prompted_passes")
    same(model.encode_tokens(toks, normalize_embeddings=True), oracle_encode(cfg, W, toks), 1e-3)
    assert st.debug_counter("prompted_passes") == p0 + (0 if pass_tokens else 30)
