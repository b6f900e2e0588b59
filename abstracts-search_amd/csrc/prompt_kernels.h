// prompt_kernels.h -- gfx950 kernels of the prompt cache (include/mi_encoder.h): the attention of packed texts over a
// cached prompt that all of them stand behind, and the operations on the cache's pages.
//
// Pages: [page][layer][key head][K, V][64 tokens][head dim], bf16 or f16.  One (page, layer, key head) is one contiguous run of
// 64 K rows and 64 V rows (32 KiB at head dim 128): the attention reads whole runs, a page is copied as one run.
//
// Attention.  For key head kvh the query rows are (token, head of the group) pairs, token first: row r = token r / G, head
// kvh G + r % G (G = query heads per key head).  Every row sees all P prompt keys and the keys [lo, hi) of its own text:
//     o = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),   s_j = scale log2(e) (q . k_j),   m >= all s_j so far
// with m, the sum and o held in f32 and carried over the keys in one pass.  Rows of different texts share everything about the
// prompt, so a tile of rows is cut from the packed tokens wherever texts begin or end: the prompt part needs no mask at all.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace mipc {

constexpr int PC_PAGE = 64;

typedef unsigned short bf16_t;            // 16-bit words of either type
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));

// two f32 -> packed bf16, round to nearest even (v_cvt_pk_bf16_f32)
__device__ __forceinline__ unsigned pack2(float lo, float hi) {
    const f32x2_t v = {lo, hi};
    return __builtin_bit_cast(unsigned, __builtin_convertvector(v, bf16x2_t));
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off);
    return v;
}

struct TBf16 {
    static constexpr int dtype = 1;
    __device__ static float up(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
    __device__ static unsigned pack(float lo, float hi) { return pack2(lo, hi); }
    __device__ static unsigned short down(float v) { return (unsigned short)(pack2(v, v) & 0xffffu); }
    // probabilities are rounded to the values' type for the product with V (relative error 2^-9 each, the denominator sums the
    // f32 values); bf16 has f32's exponents
    static constexpr float shift = 0.f;
};
struct TF16 {
    static constexpr int dtype = 2;
    __device__ static float up(unsigned short b) { return (float)__builtin_bit_cast(_Float16, b); }
    __device__ static unsigned pack(float lo, float hi) {
        typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
        const f32x2_t v = {lo, hi};
        return __builtin_bit_cast(unsigned, __builtin_convertvector(v, f16x2_t));
    }
    __device__ static unsigned short down(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
    // f16 loses what is below 2^-25: the probabilities are held as 2^7 p (p <= 1), so that a long tail of small ones keeps its
    // weight; the factor cancels in o / sum
    static constexpr float shift = 7.f;
};

struct PromptArgs {
    const bf16_t *q, *k, *v;
    bf16_t *out;
    int64_t q_token, q_head, k_token, k_head, v_token, v_head, o_token, o_head;
    const bf16_t *pages;                 // first page, at the layer's offset
    int64_t page_stride;                 // elements from page to page
    const int32_t *table;
    int P;                               // prompt tokens
    int n_tokens, n_keys, n_texts;
    const int32_t *cu_q, *cu_k;
    int n_heads, n_kv, G;
    int causal, zero_rest;
    float scale2;                        // scale * log2(e)
    // the encoder's own buffers: V^T [n_kv * hd][v_token] instead of rows (vt), Q and K with the rotary pairs interleaved while the
    // pages hold them in the weights' order (inter), the output as operand fragments of the next product (frag, frag_mt tiles)
    int vt, inter;
    bf16_t *frag;
    int frag_mt;
};

// the text of token t, and the keys [lo, hi) of its own that it sees; t behind the last text: false.  Whatever the two arrays
// hold, the result stays inside [0, n_keys].
__device__ __forceinline__ bool prompt_own_range(const PromptArgs &a, int t, int &lo, int &hi) {
    int q0 = 0, q1 = a.n_tokens, k0 = 0, k1 = a.n_keys;
    if (a.cu_q) {
        int i = 0, n = a.n_texts;                             // the last text with cu_q[i] <= t
        while (n > 1) {
            const int half = n >> 1;
            if (a.cu_q[i + half] <= t) i += half;
            n -= half;
        }
        q0 = a.cu_q[i]; q1 = a.cu_q[i + 1];
        k0 = min(max(a.cu_k[i], 0), a.n_keys);
        k1 = min(max(a.cu_k[i + 1], k0), a.n_keys);
    }
    lo = k0;
    // (64 bits: whatever the arrays hold)
    hi = a.causal ? (int)min(max((int64_t)k1 - q1 + t + 1, (int64_t)k0), (int64_t)k1) : k1;
    return t >= q0 && t < q1;
}

// ---------------------------------------------------------------------------------------------------------------------
// One row by one wave: lanes over the keys of a step for the scores, over the head's dims for the output.  Sees exactly the
// row's keys, so nothing that is masked is ever read.  64 keys cost ~1 us: the plain form of the kernels below, and what they
// fall back to for rows where a masked value that is no number would have entered a product (0 x inf).
// ---------------------------------------------------------------------------------------------------------------------
template <class T, int HD>
__device__ void prompt_row(const PromptArgs &a, int token, int head, int64_t p0, int64_t p1, int64_t lo, int64_t hi, float *qs /* [HD] of this wave */,
                           float (&o)[HD / 64], float &m, float &l) {
    constexpr int DPL = HD / 64;
    const int lane = threadIdx.x & 63, kvh = head / a.G;
    m = -__builtin_huge_valf();
    l = 0.f;
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = 0.f;
    for (int part = 0; part < 2; ++part) {                    // the prompt's keys, then the text's own
        const bf16_t *qp = a.q + token * a.q_token + head * a.q_head;
#pragma unroll
        for (int e = 0; e < DPL; ++e) {
            const int d = lane * DPL + e;
            const int src = part == 0 && a.inter ? (d < HD / 2 ? 2 * d : 2 * (d - HD / 2) + 1) : d;
            qs[d] = T::up(qp[src]);
        }
        __builtin_amdgcn_wave_barrier();
        const int64_t b0 = part ? lo : p0, b1 = part ? hi : p1;
        for (int64_t b = b0; b < b1; b += 64) {
            const int n = (int)(b1 - b < 64 ? b1 - b : 64);
            const int64_t key = b + (lane < n ? lane : n - 1);
            const bf16_t *kp, *vp = nullptr;
            if (part == 0) kp = a.pages + a.table[key / PC_PAGE] * a.page_stride + ((int64_t)kvh * 2 * PC_PAGE + key % PC_PAGE) * HD;
            else kp = a.k + key * a.k_token + kvh * a.k_head;
            float s = 0.f;
            for (int d = 0; d < HD; d += 8) {
                const uint4 w = *reinterpret_cast<const uint4 *>(kp + d);
                const unsigned u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s = fmaf(qs[d + 2 * j], T::up((unsigned short)(u[j] & 0xffffu)), s);
                    s = fmaf(qs[d + 2 * j + 1], T::up((unsigned short)(u[j] >> 16)), s);
                }
            }
            s *= a.scale2;
            if (lane >= n) s = -__builtin_huge_valf();
            float mx = s;
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
            const float mn = fmaxf(m, mx), ms = mn == -__builtin_huge_valf() ? 0.f : mn;
            const float alpha = m == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(m - ms);
            const float p = __builtin_amdgcn_exp2f(s - ms + T::shift);
            l = l * alpha + wave_sum(p);
            m = mn;
#pragma unroll
            for (int e = 0; e < DPL; ++e) o[e] *= alpha;
            for (int i = 0; i < n; ++i) {
                const float pi = __shfl(p, i);
                const int64_t kk = b + i;
                if (part == 0) vp = a.pages + a.table[kk / PC_PAGE] * a.page_stride + (((int64_t)kvh * 2 + 1) * PC_PAGE + kk % PC_PAGE) * HD + lane * DPL;
                else if (!a.vt) vp = a.v + kk * a.v_token + kvh * a.v_head + lane * DPL;
                else vp = a.v + ((int64_t)kvh * HD + lane * DPL) * a.v_token + kk;
                const int64_t vs = part && a.vt ? a.v_token : 1;
#pragma unroll
                for (int e = 0; e < DPL; ++e) o[e] = fmaf(pi, T::up(vp[e * vs]), o[e]);
            }
        }
        __builtin_amdgcn_wave_barrier();
    }
}

template <class T, int HD>
__global__ void __launch_bounds__(256) prompt_row_kernel(PromptArgs a) {
    constexpr int DPL = HD / 64;
    __shared__ float qs[4][HD];
    const int w = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int64_t row = (int64_t)blockIdx.x * 4 + w;
    if (row >= (int64_t)a.n_tokens * a.n_heads) return;
    const int token = (int)(row / a.n_heads), head = (int)(row % a.n_heads);
    int lo, hi;
    float o[DPL], m, l;
    const bool live = prompt_own_range(a, token, lo, hi);
    if (!live && !a.zero_rest) return;
    if (live) prompt_row<T, HD>(a, token, head, 0, a.P, lo, hi, qs[w], o, m, l);
    bf16_t *op = a.out + token * a.o_token + head * a.o_head + lane * DPL;
#pragma unroll
    for (int e = 0; e < DPL; ++e) op[e] = live && (a.P > 0 || hi > lo) ? T::down(o[e] / l) : 0;   // (0 / 0 where every score is -inf, as the formula has it)
}

// ---------------------------------------------------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------------------------------------------------
// page numbers into an entry's table (they travel as kernel arguments: stream order is all that a later reader needs)
struct PcTableArgs {
    int32_t *dst;
    int n;
    int32_t val[960];
};
__global__ void __launch_bounds__(256) pc_table_kernel(PcTableArgs a) {
    for (int i = threadIdx.x; i < a.n; i += 256) a.dst[i] = a.val[i];
}

// keys and values of n tokens into the pages of an entry: a thread per (layer, token, key head, 8 dims) and K / V.
// k_inter: the source's dims are interleaved by rotary pair (2 f + h = pair f, half h); v_dim != 1: the source is V^T, elements
// v_dim apart.  Both only where the encoder stores a prompt, once.
struct PcWriteArgs {
    const bf16_t *k, *v;
    int64_t k_layer, k_token, k_head, v_layer, v_token, v_head, v_dim;
    bf16_t *pages;
    int64_t page_stride, layer_stride;
    const int32_t *table;
    int layer, n_layers, start, n, n_kv, hd, k_inter;
};
__global__ void __launch_bounds__(256) pc_write_kernel(PcWriteArgs a) {
    const int per = a.hd / 8;
    const int64_t total = (int64_t)a.n_layers * a.n * a.n_kv * per * 2;
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (i >= total) return;
    const int c = (int)(i % per);
    int64_t r = i / per;
    const int h = (int)(r % a.n_kv);
    r /= a.n_kv;
    const int t = (int)(r % a.n);
    r /= a.n;
    const int which = (int)(r & 1), l = (int)(r >> 1);
    const int pos = a.start + t;
    bf16_t *dst = a.pages + a.table[pos / PC_PAGE] * a.page_stride + (a.layer + l) * a.layer_stride +
                  (((int64_t)h * 2 + which) * PC_PAGE + pos % PC_PAGE) * a.hd + c * 8;
    const bf16_t *src = which ? a.v + l * a.v_layer + t * a.v_token + h * a.v_head : a.k + l * a.k_layer + t * a.k_token + h * a.k_head;
    if (which ? a.v_dim == 1 : !a.k_inter) {
        *reinterpret_cast<uint4 *>(dst) = *reinterpret_cast<const uint4 *>(src + c * 8);
        return;
    }
    const int64_t st = which ? a.v_dim : 2;
    src += which ? c * 8 * a.v_dim : (c * 8 < a.hd / 2 ? 2 * c * 8 : 2 * (c * 8 - a.hd / 2) + 1);
#pragma unroll
    for (int j = 0; j < 8; ++j) dst[j] = src[j * st];
}

// the first `rows` rows of every (layer, key head, K / V) of page src[j] -> page dst[j].  grid (blocks, jobs)
struct PcCopyArgs {
    const bf16_t *from;
    bf16_t *to;
    int64_t page_stride;                  // elements
    int segs, hd, rows;                   // segments of a page: layers x key heads x 2
    int32_t src[480], dst[480];
};
__global__ void __launch_bounds__(256) pc_copy_kernel(PcCopyArgs a) {
    const int per = a.rows * a.hd / 8;                        // 16-byte words of a segment
    const int64_t total = (int64_t)a.segs * per;
    const bf16_t *s = a.from + a.src[blockIdx.y] * a.page_stride;
    bf16_t *d = a.to + a.dst[blockIdx.y] * a.page_stride;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t off = (i / per * PC_PAGE * a.hd) + i % per * 8;
        *reinterpret_cast<uint4 *>(d + off) = *reinterpret_cast<const uint4 *>(s + off);
    }
}

// the tables of new entries that begin as `parent` does: its first `shared` pages, then (own[i] >= 0) one page of the entry's own
struct PcForkArgs {
    int32_t *tables;
    int64_t ld;
    int parent, shared, n;
    int32_t entry[480], own[480];
};
__global__ void __launch_bounds__(256) pc_fork_kernel(PcForkArgs a) {
    const int32_t *p = a.tables + a.parent * a.ld;
    int32_t *t = a.tables + a.entry[blockIdx.x] * a.ld;
    for (int i = threadIdx.x; i < a.shared; i += 256) t[i] = p[i];
    if (threadIdx.x == 0 && a.own[blockIdx.x] >= 0) t[a.shared] = a.own[blockIdx.x];
}

// page numbers src[j] -> dst[j] in every table (src ascending; words behind an entry's length may change too, nothing reads them)
struct PcRemapArgs {
    int32_t *tables;
    int64_t words;
    int n;
    int32_t src[480], dst[480];
};
__global__ void __launch_bounds__(256) pc_remap_kernel(PcRemapArgs a) {
    __shared__ int32_t src[480], dst[480];
    for (int i = threadIdx.x; i < a.n; i += 256) { src[i] = a.src[i]; dst[i] = a.dst[i]; }
    __syncthreads();
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < a.words; i += (int64_t)gridDim.x * 256) {
        const int32_t v = a.tables[i];
        int lo = 0, n = a.n;
        while (n > 1) {
            const int half = n >> 1;
            if (src[lo + half] <= v) lo += half;
            n -= half;
        }
        if (src[lo] == v) a.tables[i] = dst[lo];
    }
}

}  // namespace mipc
