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

typedef __attribute__((ext_vector_type(8))) __bf16 bf16x8;
typedef __attribute__((ext_vector_type(8))) _Float16 f16x8;
typedef __attribute__((ext_vector_type(4))) short i16x4;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

struct TBf16 {
    static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ static float up(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
    __device__ static unsigned pack(float lo, float hi) { return pack2(lo, hi); }
    __device__ static unsigned short down(float v) { return (unsigned short)(pack2(v, v) & 0xffffu); }
    // probabilities are rounded to the values' type for the product with V (relative error 2^-9 each, the denominator sums the
    // f32 values); bf16 has f32's exponents
    static constexpr float shift = 0.f;
};
struct TF16 {
    static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
    }
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
    // the tile kernel: keys split `splits` ways; partials o [splits][n_heads n_tokens][hd] and (m, sum) in f32 (splits > 1)
    int splits, tiles;
    float *part_o;
    float2 *part_ml;
};

// the text of token t, and the keys [lo, hi) of its own that it sees; t behind the last text: false.  Whatever the two arrays
// hold, the result stays inside [0, n_keys].
__device__ __forceinline__ bool prompt_own_range(const PromptArgs &a, const int *cu_q, const int *cu_k, int t, int &lo, int &hi) {
    int q0 = 0, q1 = a.n_tokens, k0 = 0, k1 = a.n_keys;
    if (a.cu_q) {
        int i = 0, n = a.n_texts;                             // the last text with cu_q[i] <= t
        while (n > 1) {
            const int half = n >> 1;
            if (cu_q[i + half] <= t) i += half;
            n -= half;
        }
        q0 = cu_q[i]; q1 = cu_q[i + 1];
        k0 = min(max(cu_k[i], 0), a.n_keys);
        k1 = min(max(cu_k[i + 1], k0), a.n_keys);
    }
    lo = k0;
    // (64 bits: whatever the arrays hold)
    hi = a.causal ? (int)min(max((int64_t)k1 - q1 + t + 1, (int64_t)k0), (int64_t)k1) : k1;
    return t >= q0 && t < q1;
}

// ---------------------------------------------------------------------------------------------------------------------
// One row by one wave: lanes over the keys of a step for the scores, over the head's dims for the output.  Sees exactly the
// row's keys, so nothing that is masked is ever read.  64 keys cost ~1 us: for the rows of the kernel
// below in which a masked value that is no number would have entered a product (0 x inf).
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

// ---------------------------------------------------------------------------------------------------------------------
// A tile of 32 NW rows of one key head by NW waves, the keys in chunks of 64 (a page, or 64 of the texts' own): K and V of a
// chunk arrive by LDS-DMA, double buffered, and serve every wave.  Computed transposed: S^T = K Q^T on 32x32x16 MFMAs leaves a
// lane 32 scores of ONE row (the other half of the chunk sits in lane ^ 32), so the softmax is in-lane but for one exchange.
// Which key a row position of S^T stands for is free: position m <-> key m with bits 2 and 3 exchanged; then registers
// 8 J .. 8 J + 7 hold keys 16 J + 8 (lane / 32) .. + 8, which is the B fragment of O^T += V^T P^T as it stands.  The A fragment V^T
// comes out of the row-major V tile by ds_read_b64_tr_b16 (a 16-lane group reads 4 keys x 16 dims, each lane gets one dim's 4 keys).
// Slots of 16 bytes are XORed inside the rows: K by the key bits that the 16 lanes of a read differ in, V so that the 4 rows of a
// transposing read fall on different banks.
//
// The running maximum is raised only when a row's scores pass it by 8 (in log2): p stays below 2^8, the sums are f32, and the
// rescaling of o leaves the steady state.
//
// A masked key has p = 0 exactly, and 0 x (inf or NaN in its V) would be NaN: a row whose result is no finite number is done again
// by prompt_row, which reads only what the row sees.
// ---------------------------------------------------------------------------------------------------------------------
__device__ __forceinline__ void dma16(const void *gptr, void *lds_wave_base) {   // 64 lanes x 16 bytes -> 1 KiB at lds_wave_base
    const unsigned m0v = __builtin_amdgcn_readfirstlane((unsigned)(size_t)(__attribute__((address_space(3))) void *)lds_wave_base);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off\n" ::"s"(m0v), "v"(gptr) : "memory");
}
__device__ __forceinline__ u32x2 lds_tr(const bf16_t *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)p));
}
__device__ __forceinline__ bool not_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) == 0x7f800000u; }

constexpr int PA_CU = 1024;               // texts whose bounds are kept in LDS

// four consecutive dims of one (token, head) of the output
template <class T, int HD>
__device__ __forceinline__ void prompt_store4(const PromptArgs &a, int token, int head, int d, float x, float y, float z, float w) {
    bf16_t *p = a.frag ? a.frag + ((((int64_t)head * (HD / 32) + d / 32) * a.frag_mt + (token >> 4)) * 64 + (d % 32) / 8 * 16 + (token & 15)) * 8 + d % 8
                       : a.out + token * a.o_token + head * a.o_head + d;
    *reinterpret_cast<uint2 *>(p) = make_uint2(T::pack(x, y), T::pack(z, w));
}

template <class T, int HD, int NW, bool VT>
__global__ void __launch_bounds__(64 * NW, 2) prompt_tile_kernel(PromptArgs a) {
    constexpr int KC = PC_PAGE, NKK = HD / 16, NDT = HD / 32, SL = HD / 8;      // keys of a chunk, MFMA steps over hd, output tiles, slots of a row
    constexpr int RPP = 64 / SL, PIECES = KC / RPP, PPW = PIECES / NW;            // rows of a 1-KiB piece, pieces of a K or V tile, of a wave
    constexpr int STG = 2 * KC * HD;
    static_assert(PIECES % NW == 0, "pieces divide over the waves");
    __shared__ __attribute__((aligned(16))) bf16_t smem[2 * STG];
    __shared__ int s_cu[2][PA_CU + 1];
    __shared__ float s_q[NW][HD];                                               // prompt_row's
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, half = lane >> 5;
    // blocks b, b + 8, .. run on one XCD: each XCD takes a contiguous eighth of the (key head, split, tile) sequence, whose members
    // share the key head's pages in its L2
    const int items = a.n_kv * a.splits * a.tiles, per = (items + 7) / 8;
    const int it = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (it >= items || (int)(blockIdx.x / 8) >= per) return;
    const int tile = it % a.tiles, split = it / a.tiles % a.splits, kvh = it / a.tiles / a.splits;
    const int rows = a.n_tokens * a.G, r0 = tile * 32 * NW;
    // bounds of the texts
    const bool in_lds = a.cu_q && a.n_texts <= PA_CU;
    if (in_lds) {
        for (int i = tid; i <= a.n_texts; i += 64 * NW) { s_cu[0][i] = a.cu_q[i]; s_cu[1][i] = a.cu_k[i]; }
        __syncthreads();
    }
    const int *cq = in_lds ? s_cu[0] : a.cu_q, *ck = in_lds ? s_cu[1] : a.cu_k;
    const int t_end = min(a.cu_q ? min(cq[a.n_texts], a.n_tokens) : a.n_tokens, (r0 + 32 * NW - 1) / a.G + 1);   // tokens of this tile that belong to texts
    const int row = r0 + 32 * w + li, token = min(row, rows - 1) / a.G, head = kvh * a.G + min(row, rows - 1) % a.G;
    int lo, hi, k0, k1, dummy;
    bool live = prompt_own_range(a, cq, ck, token, lo, hi) && row < rows;
    if (!prompt_own_range(a, cq, ck, r0 / a.G, k0, dummy) || !prompt_own_range(a, cq, ck, t_end - 1, dummy, k1)) k0 = k1 = 0;
    if (VT) k0 &= ~7;                                                           // V^T rows are read in 16-byte pieces
    if (k1 < k0) k1 = k0;
    // this workgroup's share of the chunks: nP of the prompt, then the texts' own
    const int nP = (a.P + KC - 1) / KC, n_all = nP + (k1 - k0 + KC - 1) / KC;
    const int c0 = (int)((int64_t)n_all * split / a.splits), c1 = (int)((int64_t)n_all * (split + 1) / a.splits);

    auto kswz = [](int key) { return SL == 16 ? key & 15 : (key & 3) | ((key >> 3) & 1) << 2; };
    auto vswz = [](int key) { return SL == 16 ? (key & 3) * 4 : ((key >> 1) & 1) * 4; };
    auto issue = [&](int c, int stage) {
        bf16_t *Ks = smem + stage * STG, *Vs = Ks + KC * HD;
        if (c < nP) {
            const bf16_t *pg = a.pages + a.table[c] * a.page_stride + (int64_t)kvh * 2 * KC * HD;
            const int last = min(a.P - c * KC, KC) - 1;                          // rows behind the prompt's end: its last one again (masked, and finite if the prompt is)
#pragma unroll
            for (int i = 0; i < PPW; ++i) {
                const int p = w * PPW + i, key = p * RPP + lane / SL, s = lane % SL, r = min(key, last);
                dma16(pg + r * HD + (s ^ kswz(key)) * 8, Ks + p * 512);
                dma16(pg + KC * HD + r * HD + (s ^ vswz(key)) * 8, Vs + p * 512);
            }
        } else {
            const int b = k0 + (c - nP) * KC;
#pragma unroll
            for (int i = 0; i < PPW; ++i) {
                const int p = w * PPW + i, key = p * RPP + lane / SL, s = lane % SL;
                const int64_t r = min(b + key, k1 - 1);
                dma16(a.k + r * a.k_token + kvh * a.k_head + (s ^ kswz(key)) * 8, Ks + p * 512);
                if (VT) {                                                        // 8 dims x 64 keys
                    const int d = p * 8 + (lane >> 3), sl = lane & 7;
                    dma16(a.v + ((int64_t)kvh * HD + d) * a.v_token + b + (sl ^ (d & 7)) * 8, Vs + p * 512);
                } else {
                    dma16(a.v + r * a.v_token + kvh * a.v_head + (s ^ vswz(key)) * 8, Vs + p * 512);
                }
            }
        }
    };
    // Q as B fragments: row li, dims 16 kk + 8 half .. (deint: from interleaved rotary pairs to the pages' order)
    u32x4 qf[NKK];
    auto load_q = [&](bool deint) {
        const bf16_t *qp = a.q + token * a.q_token + head * a.q_head;
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) {
            const int d = 16 * kk + 8 * half;
            if (!deint) {
                qf[kk] = *reinterpret_cast<const u32x4 *>(qp + d);
            } else {
                const int up = d >= HD / 2;
                const u32x4 x = *reinterpret_cast<const u32x4 *>(qp + 2 * (d - up * (HD / 2))), y = *reinterpret_cast<const u32x4 *>(qp + 2 * (d - up * (HD / 2)) + 8);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned u = j < 2 ? x[2 * j] : y[2 * j - 4], v = j < 2 ? x[2 * j + 1] : y[2 * j - 3];
                    qf[kk][j] = up ? (u >> 16) | (v & 0xffff0000u) : (u & 0xffffu) | (v << 16);
                }
            }
        }
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) asm volatile("" : "+v"(qf[kk]));        // (the wait for them sits here, not in the loop, where it would drain the DMA)
    };

    f32x16 o[NDT];
#pragma unroll
    for (int n = 0; n < NDT; ++n) o[n] = (f32x16)(0.f);
    float mrow = -__builtin_huge_valf(), lrow = 0.f;
    const int krow = (li & 0x13) | ((li & 4) << 1) | ((li & 8) >> 1);             // bits 2 and 3 exchanged
    const int kkey = kswz(krow);
    // transposing reads: lane (16 g + i) of a half addresses key 8 half + i / 4, dims 16 g + 4 (i % 4)
    const int vkey = 8 * half + ((lane & 15) >> 2), vslot = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vhalf = (lane & 1) * 4;

    auto compute = [&](int c, int stage) {
        const bf16_t *Ks = smem + stage * STG, *Vs = Ks + KC * HD;
        const bool own = c >= nP;
        const int b = own ? k0 + (c - nP) * KC : c * KC;
        // keys [l, h) of the chunk are this row's
        const int l = own ? max(lo - b, 0) : 0, h = !live ? 0 : min(own ? hi - b : a.P - b, KC);
        if (!__builtin_amdgcn_ballot_w64(l < h)) return;                        // (a wave none of whose rows sees the chunk)
        f32x16 s[2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            s[j] = (f32x16)(0.f);
            const bf16_t *kb = Ks + (32 * j + krow) * HD;
#pragma unroll
            for (int kk = 0; kk < NKK; ++kk) s[j] = T::mfma(*reinterpret_cast<const u32x4 *>(kb + (((2 * kk + half) ^ kkey) * 8)), qf[kk], s[j]);
        }
        if (__builtin_amdgcn_ballot_w64(l > 0 || h < KC)) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int key = 32 * j + 16 * (r >> 3) + 8 * half + (r & 7);
                    if (key < l || key >= h) s[j][r] = -__builtin_huge_valf();
                }
        }
        float mx = fmaxf(s[0][0], s[1][0]);
#pragma unroll
        for (int r = 1; r < 16; ++r) mx = fmaxf(fmaxf(mx, s[0][r]), s[1][r]);
        const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
        mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.scale2;
        if (__builtin_amdgcn_ballot_w64(mx > mrow + 8.f)) {
            const float mn = fmaxf(mrow, mx);
            const float alpha = mrow == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(mrow - mn);
            mrow = mn;
            lrow *= alpha;
#pragma unroll
            for (int n = 0; n < NDT; ++n) o[n] *= alpha;
        }
        const float sub = (mrow == -__builtin_huge_valf() ? 0.f : mrow) - T::shift;
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], a.scale2, -sub));
                lrow += s[j][r];
            }
#pragma unroll
        for (int J = 0; J < 4; ++J) {
            u32x4 pf;
#pragma unroll
            for (int e = 0; e < 4; ++e) pf[e] = T::pack(s[J >> 1][8 * (J & 1) + 2 * e], s[J >> 1][8 * (J & 1) + 2 * e + 1]);
#pragma unroll
            for (int n = 0; n < NDT; ++n) {
                u32x4 vf;
                if (VT && own) {
                    vf = *reinterpret_cast<const u32x4 *>(Vs + (32 * n + li) * KC + (((2 * J + half) ^ (li & 7)) * 8));
                } else {
                    const bf16_t *vp = Vs + (16 * J + vkey) * HD + vhalf;
                    const u32x2 x = lds_tr(vp + ((4 * n + vslot) ^ vswz(vkey)) * 8), y = lds_tr(vp + 4 * HD + ((4 * n + vslot) ^ vswz(vkey + 4)) * 8);
                    vf = (u32x4){x[0], x[1], y[0], y[1]};
                }
                o[n] = T::mfma(vf, pf, o[n]);
            }
        }
    };

    if (c0 < c1) {
        load_q(a.inter && c0 < nP);
        issue(c0, 0);
        for (int c = c0; c < c1; ++c) {
            if (a.inter && c == nP && c > c0) load_q(false);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");                     // own pieces of chunk c
            __syncthreads();                                                     // everyone's; chunk c - 1 is used up
            if (c + 1 < c1) issue(c + 1, (c + 1 - c0) & 1);
            compute(c, (c - c0) & 1);
        }
    }

    {
        const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(lrow), __float_as_uint(lrow), false, false);
        lrow = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    }
    bool bad = not_finite(lrow);
#pragma unroll
    for (int n = 0; n < NDT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) bad = bad || not_finite(o[n][r]);
    uint64_t redo = __builtin_amdgcn_ballot_w64(bad && live);
    redo = (redo | redo >> 32) & 0xffffffffu;
    const bool sees = a.P > 0 || hi > lo;
    const int64_t prow = ((int64_t)split * a.n_kv + kvh) * rows;                 // this split's partials of the key head
    if (row < rows && !(redo >> li & 1) && (live || a.zero_rest || a.splits > 1)) {
        if (a.splits > 1) {
            float *po = a.part_o + (prow + row) * HD;
#pragma unroll
            for (int n = 0; n < NDT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4 *>(po + 32 * n + 8 * q + 4 * half) = make_float4(o[n][4 * q], o[n][4 * q + 1], o[n][4 * q + 2], o[n][4 * q + 3]);
            if (!half) a.part_ml[prow + row] = make_float2(mrow, lrow);
        } else {
            const float inv = live && sees ? 1.0f / lrow : 0.f;                  // (0 x inf where every score is -inf: NaN, as 0 / 0)
#pragma unroll
            for (int n = 0; n < NDT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    prompt_store4<T, HD>(a, token, head, 32 * n + 8 * q + 4 * half, o[n][4 * q] * inv, o[n][4 * q + 1] * inv, o[n][4 * q + 2] * inv, o[n][4 * q + 3] * inv);
        }
    }
    while (redo) {
        const int i = __builtin_ctzll(redo);
        redo &= redo - 1;
        const int tk = __builtin_amdgcn_readlane(token, i), hd_ = __builtin_amdgcn_readlane(head, i), rr = __builtin_amdgcn_readlane(row, i);
        const int l_ = __builtin_amdgcn_readlane(lo, i), h_ = __builtin_amdgcn_readlane(hi, i);
        constexpr int DPL = HD / 64;
        float ro[DPL], m, l;
        const int64_t b0 = (int64_t)k0 + (int64_t)max(c0 - nP, 0) * KC, b1 = (int64_t)k0 + (int64_t)max(c1 - nP, 0) * KC;   // own keys of this split
        prompt_row<T, HD>(a, tk, hd_, min((int64_t)c0 * KC, (int64_t)a.P), min((int64_t)c1 * KC, (int64_t)a.P), max((int64_t)l_, b0), min((int64_t)h_, b1), s_q[w], ro, m, l);
#pragma unroll
        for (int e = 0; e < DPL; ++e) {
            const int d = lane * DPL + e;
            if (a.splits > 1) a.part_o[(prow + rr) * HD + d] = ro[e];
            else if (a.frag) a.frag[((((int64_t)hd_ * (HD / 32) + d / 32) * a.frag_mt + (tk >> 4)) * 64 + (d % 32) / 8 * 16 + (tk & 15)) * 8 + d % 8] = T::down(ro[e] / l);
            else a.out[tk * a.o_token + hd_ * a.o_head + d] = T::down(ro[e] / l);
        }
        if (a.splits > 1 && lane == 0) a.part_ml[prow + rr] = make_float2(m, l);
    }
}

// the splits' partials of a row -> the output: a wave per row, o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i in the splits' order
template <class T, int HD>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptArgs a) {
    constexpr int LPR = HD / 4;                                                  // lanes of a row, four dims each
    const int rows = a.n_tokens * a.G;
    const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) / LPR;
    if (i >= (int64_t)rows * a.n_kv) return;
    const int d = threadIdx.x % LPR * 4, kvh = (int)(i / rows), row = (int)(i % rows), token = row / a.G, head = kvh * a.G + row % a.G;
    int lo, hi;
    const bool live = prompt_own_range(a, a.cu_q, a.cu_k, token, lo, hi);
    if (!live && !a.zero_rest) return;
    float m = -__builtin_huge_valf(), l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    const int64_t n = (int64_t)rows * a.n_kv;
    for (int s = 0; s < a.splits; ++s) m = fmaxf(m, a.part_ml[s * n + i].x);
    const float sub = m == -__builtin_huge_valf() ? 0.f : m;
    for (int s = 0; s < a.splits; ++s) {
        const float2 ml = a.part_ml[s * n + i];
        const float4 x = *reinterpret_cast<const float4 *>(a.part_o + (s * n + i) * HD + d);
        const float f = __builtin_amdgcn_exp2f(ml.x - sub);
        l += f * ml.y;
        // (a split that saw no key of the row has zeros; its weight is 0 too)
        o.x += f * x.x; o.y += f * x.y; o.z += f * x.z; o.w += f * x.w;
    }
    const float inv = live && (a.P > 0 || hi > lo) ? 1.0f / l : 0.f;
    if (live) prompt_store4<T, HD>(a, token, head, d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    else prompt_store4<T, HD>(a, token, head, d, 0.f, 0.f, 0.f, 0.f);
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
