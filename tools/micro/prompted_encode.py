"""What a cached prompt buys: a causal model of stella_en_1.5B_v5's shape (synthetic weights), texts behind a prompt, encoded with
the prompt's tokens in every text and behind the cached prompt; what passes cost by their tokens; several prompts in one call.
python tools/micro/prompted_encode.py"""
import os
import sys
import time

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.dirname(os.path.abspath(__file__)))))
import numpy as np
import torch

import abstracts_search_amd.sentence_transformers as st

cfg = dict(st.STELLA_EN_1_5B_V5, causal=True, max_seq_len=5000)
model = st.SentenceTransformer(config=cfg)
g = torch.Generator(device="cuda").manual_seed(7)
rnd = lambda shape, scale: (torch.randn(shape, generator=g, device="cuda") * scale).bfloat16()
H, I = cfg["hidden"], cfg["intermediate"]
qc, kc = cfg["n_heads"] * cfg["head_dim"], cfg["n_kv_heads"] * cfg["head_dim"]
one = torch.ones(H, device="cuda")
model.load_weights({"embed_tokens.weight": rnd((cfg["vocab_size"], H), 0.3), "norm.weight": one, "dense.weight": rnd((cfg["dense_out"], H), H ** -0.5),
                    "dense.bias": torch.zeros(cfg["dense_out"], device="cuda")})
for l in range(cfg["n_layers"]):
    p = f"layers.{l}."
    model.load_weights({p + "input_layernorm.weight": one, p + "post_attention_layernorm.weight": one,
                        p + "self_attn.q_proj.weight": rnd((qc, H), H ** -0.5), p + "self_attn.q_proj.bias": rnd((qc,), 0.1),
                        p + "self_attn.k_proj.weight": rnd((kc, H), H ** -0.5), p + "self_attn.k_proj.bias": rnd((kc,), 0.1),
                        p + "self_attn.v_proj.weight": rnd((kc, H), H ** -0.5), p + "self_attn.v_proj.bias": rnd((kc,), 0.1),
                        p + "self_attn.o_proj.weight": rnd((H, qc), qc ** -0.5), p + "mlp.gate_proj.weight": rnd((I, H), H ** -0.5),
                        p + "mlp.up_proj.weight": rnd((I, H), H ** -0.5), p + "mlp.down_proj.weight": rnd((H, I), I ** -0.5)})
rng = np.random.default_rng(1)
ids = lambda n: rng.integers(0, cfg["vocab_size"], n).tolist()


def ms(f, n):
    for _ in range(3):
        f()
    torch.cuda.synchronize()
    t = time.perf_counter()
    for _ in range(n):
        f()
    torch.cuda.synchronize()
    return (time.perf_counter() - t) / n * 1e3


def forced(f, attrs=dict(prompt_break_even=(0, 0, 0), prompt_pass_tokens=0)):
    """f() with every text behind its cached prompt, whatever that costs"""
    for k, v in attrs.items():
        setattr(model, k, v)
    try:
        return f()
    finally:
        for k in attrs:
            delattr(model, k)


print("what a forward pass takes, by its tokens (texts x tokens each: ms)")
print("  " + ", ".join(f"{n} x {l}: {ms(lambda b=[ids(l) for _ in range(n)]: model.encode_tokens(b, as_tensor=True), 10):.2f}" for n, l in
                      ((1, 20), (1, 31), (2, 24), (2, 35), (3, 50), (3, 100), (10, 100), (20, 100), (50, 100), (100, 100), (300, 100))), flush=True)
print("texts behind one prompt: with its tokens, behind the cached prompt, and what encode_tokens takes (the cache or not)")
for prompt_len, texts, text_len, reps in ((20, 1, 11, 50), (30, 1, 11, 50), (24, 8, 15, 30), (32, 16, 15, 30), (20, 16, 15, 30), (60, 4, 40, 30), (200, 1, 60, 30),
                                          (200, 1, 100, 30), (400, 1, 11, 50), (400, 16, 15, 30), (400, 128, 220, 5), (4000, 16, 15, 5), (4000, 64, 220, 3)):
    prompt = ids(prompt_len)
    batch = [prompt + ids(text_len) for _ in range(texts)]
    run = lambda: model.encode_tokens(batch, normalize_embeddings=True, as_tensor=True)
    plain, ref = ms(run, reps), run()
    t = time.perf_counter()
    model.cache_prompt(prompt)
    once = (time.perf_counter() - t) * 1e3
    cached, got = forced(lambda: (ms(run, reps), run()))
    print(f"prompt {prompt_len:5d}, {texts:4d} texts of {text_len:4d} tokens: {plain:9.3f} ms, {cached:9.3f} ms ({plain / cached:6.2f}x; caching it {once:.1f} ms), {ms(run, reps):9.3f} ms, "
          f"cosine >= {float((ref * got).sum(1).min()):.6f}", flush=True)
    model.drop_prompts()
print("several prompts of 160 tokens in one call: likewise")
for prompts, each, text_len in ((2, 1, 5), (2, 4, 15), (4, 1, 5), (4, 4, 15), (10, 1, 5), (10, 8, 60), (30, 1, 5), (30, 4, 15), (30, 8, 60)):
    base = ids(100)
    heads = [base + ids(60) for _ in range(prompts)]
    batch = [p + ids(text_len) for p in heads for _ in range(each)]
    run = lambda: model.encode_tokens(batch, normalize_embeddings=True, as_tensor=True)
    plain = ms(run, 10)
    for p in heads:
        model.cache_prompt(p)
    print(f"{prompts:3d} prompts, {each} texts of {text_len:3d} behind each: {plain:9.3f} ms, {forced(lambda: ms(run, 10)):9.3f} ms, {ms(run, 10):9.3f} ms", flush=True)
    model.drop_prompts()
prompt = ids(20)
batch = [prompt + ids(11) for _ in range(40)]
run = lambda: model.encode_tokens(batch, batch_size=1, normalize_embeddings=True, as_tensor=True)
plain = ms(run, 5)
model.cache_prompt(prompt)
print(f"40 queries of 31 tokens one at a time: {plain:.2f} ms, {forced(lambda: ms(run, 5)):.2f} ms, {ms(run, 5):.2f} ms")
