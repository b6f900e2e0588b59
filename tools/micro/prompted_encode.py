"""What a cached prompt buys: a causal model of stella_en_1.5B_v5's shape (synthetic weights), texts behind a prompt, encoded with
the prompt's tokens in every text and behind the cached prompt.   python tools/micro/prompted_encode.py"""
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


for prompt_len, texts, text_len, reps in ((20, 1, 11, 50), (30, 1, 11, 50), (400, 1, 11, 50), (20, 16, 15, 30), (400, 16, 15, 30), (400, 128, 220, 5), (4000, 16, 15, 5), (4000, 64, 220, 3)):
    prompt = ids(prompt_len)
    batch = [prompt + ids(text_len) for _ in range(texts)]
    run = lambda: model.encode_tokens(batch, normalize_embeddings=True, as_tensor=True)
    plain, ref = ms(run, reps), run()
    t = time.perf_counter()
    model.cache_prompt(prompt)
    once = (time.perf_counter() - t) * 1e3
    cached, got = ms(run, reps), run()
    print(f"prompt {prompt_len:5d}, {texts:4d} texts of {text_len:4d} tokens: {plain:9.3f} ms, behind the cached prompt {cached:9.3f} ms ({plain / cached:6.2f}x; caching it {once:.1f} ms), "
          f"cosine >= {float((ref * got).sum(1).min()):.6f}", flush=True)
    model.drop_prompts()
