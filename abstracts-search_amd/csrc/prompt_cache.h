// prompt_cache.h -- what encoder.hip uses of prompt_cache.hip besides the C ABI.
#pragma once
#include <cstdint>

#include "../../include/mi_encoder.h"
#include "common.h"

namespace mi {

// the encoder's own operand forms (PromptArgs: vt, inter, frag), and an entry that is being filled
struct PromptForms {
    bool vt = false, inter = false;
    void *frag = nullptr;
    int frag_mt = 0;
    int prompt_tokens = -1;      // attend to this many of the entry's tokens (-1: all)
};
int64_t prompt_attention_workspace(mi_prompt_cache *c, const mi_prompt_attn &a);
void prompt_attention(mi_prompt_cache *c, const mi_prompt_attn &a, const PromptForms &f, void *stream);
// K rows (k_inter: rotary pairs interleaved) and V^T columns of an encoder pass -> tokens start .. of an entry, one layer
void prompt_cache_write_vt(mi_prompt_cache *c, int32_t entry, int32_t layer, int32_t start, int32_t n, const void *k, int64_t k_token, bool k_inter,
                           const void *vt, int64_t ldvt, void *stream);

}  // namespace mi
