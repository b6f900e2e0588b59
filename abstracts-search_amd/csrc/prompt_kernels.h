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
#include <type_traits>
#include <utility>

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

// f(0), f(1), .. with the numbers as types: unrolled whatever the body's size
template <class F, int... I>
__device__ __forceinline__ void each_of(std::integer_sequence<int, I...>, F &&f) { (f(std::integral_constant<int, I>{}), ...); }
template <int N, class F>
__device__ __forceinline__ void each(F &&f) { each_of(std::make_integer_sequence<int, N>{}, f); }

struct TBf16 {
    static __device__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
    __device__ static float up(unsigned short b) { return __uint_as_float((unsigned)b << 16); }
    __device__ static unsigned pack(float lo, float hi) { return pack2(lo, hi); }
    __device__ static unsigned scaled(unsigned two, float f) { return pack(up((unsigned short)(two & 0xffffu)) * f, up((unsigned short)(two >> 16)) * f); }
    __device__ static unsigned short down(float v) { return (unsigned short)(pack2(v, v) & 0xffffu); }
    // probabilities are rounded to the values' type for the product with V (a relative error of up to 2^-8 each, the denominator sums the
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
    __device__ static unsigned scaled(unsigned two, float f) { return pack(up((unsigned short)(two & 0xffffu)) * f, up((unsigned short)(two >> 16)) * f); }
    __device__ static unsigned short down(float v) { return __builtin_bit_cast(unsigned short, (_Float16)v); }
    // f16 loses what is below 2^-25: the probabilities are held as 2^7 p, so that a long tail of small ones keeps its weight; the factor
    // cancels in o / sum.  p stays below 2^8 (the maximum may lag by that), so what is held below 2^15, half of f16's largest value
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
    float r_tiles, r_splits, r_G;        // 1 / tiles, ..
    float *part_o;
    float2 *part_ml;
};

// n / d for 0 <= n < 2^31, r = 1 / d: two approximations and a correction, a dozen instructions where a division is forty
__device__ __forceinline__ int quotient(int n, int d, float r) {
    int q = (int)((float)n * r);
    int rem = n - q * d;                                      // |rem| < 2^9 d
    const int more = (int)((float)rem * r);
    q += more;
    rem -= more * d;
    return q + (rem >= d) - (rem < 0);
}

// the text of token t, and the keys [lo, hi) of its own that it sees; t behind the last text: false.  Whatever the two arrays
// hold, the result stays inside [0, n_keys].
// (Ints: a pointer into global memory or into LDS -- one that may be either would be read by flat instructions, whose waits are for both)
template <class Ints>
__device__ __forceinline__ bool prompt_own_range(const PromptArgs &a, Ints cu_q, Ints cu_k, int t, int &lo, int &hi) {
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
// below in which a value that is no number has entered a product with a probability rounded to 0 or masked (0 x inf).
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
// A tile of 128 rows of one key head by four waves, the keys in chunks of 64 (a page, or 64 of the texts' own): K and V of a
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
// A masked key has p = 0 exactly (so have the rows behind the prompt's and the texts' end, which hold the last one again), a rounding may
// leave one of 0 or less, and 0 x (inf or NaN in V) would be NaN: a row whose result is no finite number is done again by prompt_row,
// which reads only what the row sees and keeps its probabilities in f32 -- unless its sum is NaN: the sum is over keys that the row
// sees, so every dim is NaN.  Slow where it is all rows: an infinity in V of a prompt of 4096 takes 13.1 k tokens from 1.05 to 294 ms, one
// in V of 400 32.7 k tokens from 0.2 to 39 (a NaN in the prompt's K costs nothing).
// ---------------------------------------------------------------------------------------------------------------------
typedef __attribute__((address_space(3))) bf16_t lds_t;
// 64 lanes x 16 bytes from base + the lane's offset -> 1 KiB at dst (the same in every lane)
__device__ __forceinline__ void dma16(const void *base, unsigned offset, lds_t *dst) {
    const unsigned m0v = __builtin_amdgcn_readfirstlane((unsigned)(size_t)dst);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2\n" ::"s"(m0v), "v"(offset), "s"(base) : "memory");
}
// a pointer that is the same in every lane, in scalar registers
__device__ __forceinline__ const bf16_t *uniform(const bf16_t *p) {
    const uint64_t u = reinterpret_cast<uint64_t>(p);
    return reinterpret_cast<const bf16_t *>((uint64_t)__builtin_amdgcn_readfirstlane((int)(u >> 32)) << 32 | (uint32_t)__builtin_amdgcn_readfirstlane((int)u));
}
__device__ __forceinline__ u32x2 lds_tr(const lds_t *p) {
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) i16x4 *)p));
}
__device__ __forceinline__ u32x4 lds_16(const lds_t *p) { return *(const __attribute__((address_space(3))) u32x4 *)p; }

constexpr int PA_WAVES = 4;               // waves of a workgroup: a tile of 128 rows
constexpr int PA_CU = 1023;               // texts whose bounds are kept in LDS

// four consecutive dims of one (token, head) of the output
template <class T, int HD>
__device__ __forceinline__ void prompt_store4(const PromptArgs &a, int token, int head, int d, float x, float y, float z, float w) {
    bf16_t *p = a.frag ? a.frag + ((((int64_t)head * (HD / 32) + d / 32) * a.frag_mt + (token >> 4)) * 64 + (d % 32) / 8 * 16 + (token & 15)) * 8 + d % 8
                       : a.out + token * a.o_token + head * a.o_head + d;
    *reinterpret_cast<uint2 *>(p) = make_uint2(T::pack(x, y), T::pack(z, w));
}

// the kernel's arguments once more, read from memory where they are used: the epilogues' share of them would otherwise sit in scalar
// registers all through the loop over the keys (120 of them spilled)
__device__ __forceinline__ const PromptArgs &args_again() {
    uint64_t p = (uint64_t)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PromptArgs *)(const __attribute__((address_space(4))) PromptArgs *)p;
}

// a wave's 32 rows: O^T tiles, the maxima and this half's sums -> the output, or this split's partials.  Prompt keys [p0, p1) and own
// keys [b0, b1) are what this workgroup went through.
template <class T, int HD>
__device__ __forceinline__ void prompt_finish(const f32x16 (&o)[HD / 32], float mrow, float lrow, int row, int token, int head, int lo, int hi,
                                              bool live, int split, int kvh, int64_t p0, int64_t p1, int64_t b0, int64_t b1, float *qs) {
    constexpr int NDT = HD / 32, DPL = HD / 64;
    const PromptArgs &a = args_again();
    const int lane = threadIdx.x & 63, li = lane & 31, half = lane >> 5, rows = a.n_tokens * a.G;
    const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(lrow), __float_as_uint(lrow), false, false);
    lrow = __uint_as_float(sw[0]) + __uint_as_float(sw[1]);
    const bool sees = live && (a.P > 0 || hi > lo);
    float zero = lrow * 0.f;                                                     // NaN if anything is no finite number
#pragma unroll
    for (int n = 0; n < NDT; ++n)
#pragma unroll
        for (int r = 0; r < 16; ++r) zero = __builtin_fmaf(o[n][r], 0.f, zero);
    const uint64_t bad = __builtin_amdgcn_ballot_w64(zero != 0.f && lrow == lrow && sees);
    unsigned redo = (unsigned)(bad | bad >> 32);
    const int64_t prow = ((int64_t)split * a.n_kv + kvh) * rows;                 // this split's partials of the key head
    if (row < rows && !(redo >> li & 1) && (live || a.zero_rest || a.splits > 1)) {
        if (a.splits > 1) {
            float *po = a.part_o + (prow + row) * HD + 4 * half;
#pragma unroll
            for (int n = 0; n < NDT; ++n)
#pragma unroll
                for (int q = 0; q < 4; ++q)
                    *reinterpret_cast<float4 *>(po + 32 * n + 8 * q) = make_float4(o[n][4 * q], o[n][4 * q + 1], o[n][4 * q + 2], o[n][4 * q + 3]);
            if (!half) a.part_ml[prow + row] = make_float2(mrow, !live ? -1.f : sees ? lrow : -2.f);   // (the same in every split: what the join does not have to look up)
        } else {
            const float inv = 1.0f / lrow;                  // (0 x inf where every score is -inf: NaN, as 0 / 0)
            // dims 32 n + 8 q + 4 half ..: rows of the output, or fragments (prompt_store4)
            bf16_t *po = (a.frag ? a.frag + (((int64_t)head * (HD / 32) * a.frag_mt + (token >> 4)) * 64 + (token & 15)) * 8 : a.out + token * a.o_token + head * a.o_head) + 4 * half;
            const int sn = a.frag ? a.frag_mt * 512 : 32, sq = a.frag ? 128 : 8;
#pragma unroll
            for (int n = 0; n < NDT; ++n, po += sn)
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    uint2 v = make_uint2(T::pack(o[n][4 * q] * inv, o[n][4 * q + 1] * inv), T::pack(o[n][4 * q + 2] * inv, o[n][4 * q + 3] * inv));
                    if (!sees) v = make_uint2(0u, 0u);
                    *reinterpret_cast<uint2 *>(po + q * sq) = v;
                }
        }
    }
    while (redo) {
        const int i = __builtin_ctz(redo);
        redo &= redo - 1;
        const int tk = __builtin_amdgcn_readlane(token, i), hd_ = __builtin_amdgcn_readlane(head, i), rr = __builtin_amdgcn_readlane(row, i);
        const int l_ = __builtin_amdgcn_readlane(lo, i), h_ = __builtin_amdgcn_readlane(hi, i);
        float ro[DPL], m, l;
        prompt_row<T, HD>(a, tk, hd_, min(p0, (int64_t)a.P), min(p1, (int64_t)a.P), max((int64_t)l_, b0), min((int64_t)h_, b1), qs, ro, m, l);
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

// TWO: the probabilities enter the product with V in two parts (what the type holds of them, and of the rest), which leaves the
// output's own rounding as the only one in 16 bits; one part costs another half step of the type on every output (error against 64
// bits 0.0023 instead of 0.0017 in bf16, 0.00029 instead of 0.00021 in f16).  Taken where a key head's rows are two tiles at most, which
// latency and the reading of the pages bound: 7 % longer than one part on ten tokens behind 37, 6 % on 64 single tokens of 32 heads behind
// 2048.  More rows are bound by the products: 25 % longer on 40 tokens of 64 heads behind 20 000, 32 % on 13.1 k behind 4096.
// Four waves also where one holds all the rows: the others bring their quarter of the keys in.  Workgroups of one and of two
// waves take 22 % and 16 % longer on ten tokens behind 37, 14 % and 10 % on four tokens behind 65 500, eight waves 5 % and 40 %.
// Two stages of LDS, so that two workgroups share a CU and overlap each other: four stages and one workgroup a CU took 1.7 times as
// long on four tokens behind 65 500 and 2 % longer on 13.1 k behind 4096, and four stages beside two workgroups (head dim 64) 4 %
// longer on 4 k tokens of 16 heads behind 1000.
// What bounds it, and what it takes with its join, launches included:
//   few rows, short prompt    latency: launch, arguments, bounds and Q, first page, two chunks, store; 8.9 us (10 tokens behind 37)
//   few rows, long prompt     reading the pages: 58 us for the 269 MB of 65 500 tokens (the kernel 46: 5.8 TB/s); 24 us for 64
//                             single tokens with pasts (35 MB) behind 2048, of which 5.7 for the partials of 16 splits
//   many rows                 matrix and vector work in turn: 1050 us for 13.1 k tokens of 32 heads of 128 behind 4096, 870 TFLOP/s, at the
//                             1.83 GHz of 2.4 that the power limit leaves, the matrix pipes busy 49 % of the cycles (products alone, without
//                             the exponentials, 652 us); head dim 64: the exponentials, 40 us for 4 k tokens of 16 heads behind 1000
template <class T, int HD, bool VT, bool TWO>
__global__ void __launch_bounds__(64 * PA_WAVES, 2) prompt_tile_kernel(PromptArgs a) {
    constexpr int NW = PA_WAVES, KC = PC_PAGE, NKK = HD / 16, NDT = HD / 32, SL = HD / 8;      // keys of a chunk, MFMA steps over hd, output tiles, slots of a row
    constexpr int RPP = 64 / SL, PIECES = KC / RPP, PPW = PIECES / NW;            // rows of a 1-KiB piece, pieces of a K or V tile, of a wave
    constexpr int STG = 2 * KC * HD, NS = 2;
    static_assert(PIECES % NW == 0, "pieces divide over the waves");
    __shared__ __attribute__((aligned(16))) bf16_t smem_[NS * STG];
    lds_t *const smem = (lds_t *)smem_;
    __shared__ int s_cu[2][PA_CU + 1];
    __shared__ float s_q[NW][HD];                                               // prompt_row's
    const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 31, half = lane >> 5;
    // blocks b, b + 8, .. run on one XCD: each XCD takes a contiguous eighth of the (key head, split, tile) sequence, whose members
    // share the key head's pages in its L2
    const int items = a.n_kv * a.splits * a.tiles, per = (items + 7) / 8;
    const int it = (int)(blockIdx.x % 8) * per + (int)(blockIdx.x / 8);
    if (it >= items || (int)(blockIdx.x / 8) >= per) return;
    const int part = quotient(it, a.tiles, a.r_tiles), kvh = quotient(part, a.splits, a.r_splits), tile = it - part * a.tiles, split = part - kvh * a.splits;
    const int rows = a.n_tokens * a.G, r0 = tile * 32 * NW;
    const int row = r0 + 32 * w + li, token = quotient(min(row, rows - 1), a.G, a.r_G), head = kvh * a.G + min(row, rows - 1) - token * a.G;
    // this workgroup's chunks 0 .. n - 1: its share of the prompt's pages, pages p0 .. p0 + np - 1, then of the 64-key pieces of its
    // texts' own keys [k0, k1), pieces o0 ..
    const int nP = (a.P + KC - 1) / KC;
    const int p0 = a.splits > 1 ? (int)((int64_t)nP * split / a.splits) : 0, np = (a.splits > 1 ? (int)((int64_t)nP * (split + 1) / a.splits) : nP) - p0;
    int k0 = 0, k1 = 0, o0 = 0;
    auto base_of = [&](int i) { return i < np ? (p0 + i) * KC : k0 + (o0 + i - np) * KC; };   // the chunk's first key

    auto swz = [](int key) { return SL == 16 ? (key & 3) << 2 | ((key >> 2) & 3) : ((key >> 1) & 1) << 2 | ((key >> 3) & 1) << 1 | (key & 1); };
    const bf16_t *const head_pages = a.pages + (int64_t)kvh * 2 * KC * HD;
    // the numbers of 64 pages, one in each lane (a number fetched for each chunk would be waited for with everything in flight)
    auto pages_from = [&](int i) { return a.table[min(p0 + i + lane, nP - 1)]; };
    int numbers = np > 0 ? pages_from(0) : 0;
    auto issue = [&](int i) {
        lds_t *Ks = smem + (i % NS) * STG, *Vs = Ks + KC * HD;
        // the base of a chunk is uniform, a lane adds 32 bits (the host bounds the strides)
        const bf16_t *kb, *vb;
        unsigned kt = HD * 2, vt = HD * 2;                                        // bytes from row to row
        int last = KC - 1;                                                       // rows behind the end: the last one again (masked, and finite if that one is)
        const bool own = i >= np;
        const int b = base_of(i);
        if (!own) {
            kb = head_pages + __builtin_amdgcn_readlane(numbers, i & 63) * a.page_stride;
            vb = kb + KC * HD;
            if ((i & 63) == 63) {
                numbers = pages_from(i + 1);
                asm volatile("" : "+v"(numbers));                                // (waited for here)
            }
            last = min(last, a.P - 1 - b);
        } else {
            kb = a.k + b * a.k_token + kvh * a.k_head;
            kt = (unsigned)a.k_token * 2;
            last = min(last, k1 - 1 - b);
            if (VT) vb = a.v + (int64_t)kvh * HD * a.v_token + b;
            else vb = a.v + b * a.v_token + kvh * a.v_head;
            vt = (unsigned)a.v_token * 2;
        }
        kb = uniform(kb);
        vb = uniform(vb);
#pragma unroll
        for (int e = 0; e < PPW; ++e) {                                          // (pieces dealt round the waves: a wave's pieces differ by whole multiples of the slot pattern)
            const int p = e * NW + w, key = p * RPP + lane / SL, r = min(key, last);
            const unsigned slot = (unsigned)((lane % SL) ^ swz(key)) * 16;
            dma16(kb, r * kt + slot, Ks + p * 512);
            if (VT && own) {                                                     // 8 dims x 64 keys
                const int d = p * 8 + (lane >> 3);
                dma16(vb, d * vt + (unsigned)((lane & 7) ^ (d & 7)) * 16, Vs + p * 512);
            } else {
                dma16(vb, r * vt + slot, Vs + p * 512);
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
    };
    auto pin_q = [&] {                                                           // (the wait for them sits here, not in the loop, where it would drain the DMA)
#pragma unroll
        for (int kk = 0; kk < NKK; ++kk) asm volatile("" : "+v"(qf[kk]));
    };

    // The first accesses of everything, one behind the other (each is a miss of 1 - 2 us): the texts' bounds, Q, the prompt's pages,
    // then the texts' own keys.
    const bool in_lds = a.cu_q && a.n_texts <= PA_CU;
    constexpr int CPT = (PA_CU + 1) / (64 * NW);                                 // bounds of a thread
    int b_q[CPT] = {}, b_k[CPT] = {};
    if (in_lds) {
#pragma unroll
        for (int e = 0; e < CPT; ++e) {
            const int i = tid + 64 * NW * e;
            if (i <= a.n_texts) { b_q[e] = a.cu_q[i]; b_k[e] = a.cu_k[i]; }
        }
    }
    load_q(a.inter && np > 0);
    if (in_lds) {
#pragma unroll
        for (int e = 0; e < CPT; ++e) {
            const int i = tid + 64 * NW * e;
            if (i <= a.n_texts) { s_cu[0][i] = b_q[e]; s_cu[1][i] = b_k[e]; }
        }
    }
    pin_q();                                                                     // (came in beside the bounds; the compiler's wait for them behind the first chunks would be one for these too)
    const int early = min(np, NS);
    for (int i = 0; i < early; ++i) issue(i);
    if (in_lds) asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // one search for all: lanes 0 .. 31 for their rows, lane 32 for the tile's first token that belongs to a text, the others for the last
    int lo, hi;
    bool live;
    const int t_last = quotient(min(r0 + 32 * NW, rows) - 1, a.G, a.r_G), t_first = quotient(r0, a.G, a.r_G);
    auto search = [&](auto cu_q, auto cu_k) {
        const int end = a.cu_q ? min(cu_q[a.n_texts] - 1, t_last) : t_last, begin = a.cu_q ? max(cu_q[0], t_first) : t_first;
        live = prompt_own_range(a, cu_q, cu_k, half ? (li ? end : begin) : token, lo, hi);
    };
    typedef const __attribute__((address_space(3))) int *lds_ints;
    if (in_lds) search((lds_ints)s_cu[0], (lds_ints)s_cu[1]);
    else search(a.cu_q, a.cu_k);
    const uint64_t found = __builtin_amdgcn_ballot_w64(live);
    k0 = __builtin_amdgcn_readlane(lo, 32);
    k1 = __builtin_amdgcn_readlane(hi, 33);
    if ((found >> 32 & 3) != 3) k0 = k1 = 0;
    lo = __builtin_amdgcn_permlane32_swap(lo, lo, false, false)[0];              // (the lower half's, in both)
    hi = __builtin_amdgcn_permlane32_swap(hi, hi, false, false)[0];
    live = (found >> li & 1) && row < rows;
    const bool wave_live = __builtin_amdgcn_ballot_w64(live) != 0;
    if (VT) k0 &= ~7;                                                           // V^T rows are read in 16-byte pieces
    k1 = max(k1, k0);
    const int nO = (k1 - k0 + KC - 1) / KC;
    o0 = a.splits > 1 ? (int)((int64_t)nO * split / a.splits) : 0;
    const int n = np + (a.splits > 1 ? (int)((int64_t)nO * (split + 1) / a.splits) : nO) - o0;
    for (int i = early; i < min(n, NS); ++i) issue(i);
    f32x16 o[NDT];
#pragma unroll
    for (int d = 0; d < NDT; ++d) o[d] = (f32x16)(0.f);
    float mrow = -__builtin_huge_valf(), lrow = 0.f;
    const int krow = (li & 0x13) | ((li & 4) << 1) | ((li & 8) >> 1);             // bits 2 and 3 exchanged
    const int kkey = swz(krow);
    // transposing reads: lane (16 g + i) of a half addresses key 8 half + i / 4, dims 16 g + 4 (i % 4)
    const int vkey = 8 * half + ((lane & 15) >> 2), vslot = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1), vhalf = (lane & 1) * 4;

    // what this wave has to do with chunk i: nothing, the plain product, or with a mask
    enum { SKIP = 0, FULL = 1, MASK = 2 };
    auto mode = [&](int i) {
        const int b = base_of(i);
        if (i < np) return !wave_live ? SKIP : b + KC <= a.P ? FULL : MASK;
        if (!__builtin_amdgcn_ballot_w64(live && lo < b + KC && hi > b)) return SKIP;
        return __builtin_amdgcn_ballot_w64(live && (lo > b || hi < b + KC)) ? MASK : FULL;
    };
    // A chunk is two tiles of 32 keys, each with its own online-softmax step, so that matrix and vector work of one wave overlap:
    //   S0 = K0 Q^T | S1 = K1 Q^T beside the exponentials of S0 | O += V0^T P0 beside those of S1 | O += V1^T P1
    // sched_barrier keeps the slots (a product, its share of the exponentials, the LDS reads of four products later) as written.
    auto product = [&](int i, int md) {
        const lds_t *Ks = smem + (i % NS) * STG, *Vs = Ks + KC * HD;
        constexpr int EPS = 16 / NKK;                                            // exponentials of a slot (both phases have NKK slots a tile)
        static_assert(2 * NDT == NKK, "as many products of V as of K");
        u32x4 kf[4], vf[4], pf[4], pr[TWO ? 4 : 1];                              // fragments in flight; probabilities, packed: keys 16 J + 8 half .., and their rest
        f32x16 s[2];
        const bool own = i >= np;
        const int b = base_of(i), l = own ? lo - b : 0, h = (own ? hi : a.P) - b;   // the row sees keys [l, h) of the chunk
        const unsigned from = (unsigned)(8 * half) - (unsigned)l, span = (unsigned)max(h - l, 0);
        auto read_k = [&](int f) { kf[f & 3] = lds_16(Ks + (krow + 32 * (f / NKK)) * HD + (((2 * (f % NKK) + half) ^ kkey) * 8)); };
        auto read_v = [&](int g) {
            const int J = g / NDT, n = g % NDT;
            if (VT && own) {
                vf[g & 3] = lds_16(Vs + (32 * n + li) * KC + (((2 * J + half) ^ (li & 7)) * 8));
            } else {
                const lds_t *vp = Vs + (16 * J + vkey) * HD + vhalf;
                const u32x2 x = lds_tr(vp + ((4 * n + vslot) ^ swz(vkey)) * 8), y = lds_tr(vp + 4 * HD + ((4 * n + vslot) ^ swz(vkey + 4)) * 8);
                vf[g & 3] = (u32x4){x[0], x[1], y[0], y[1]};
            }
        };
        float sub = 0.f, sum[2] = {0.f, 0.f};
        auto top = [&](auto J_) {                                                // mask, and the row's maximum
            constexpr int j = decltype(J_)::value;
            if (md == MASK) {
#pragma unroll
                for (int r = 0; r < 16; ++r) {                                   // (key - l as an unsigned number: one comparison for both ends)
                    const unsigned key = (unsigned)(32 * j + 16 * (r >> 3) + (r & 7)) + from;
                    s[j][r] = key < span ? s[j][r] : -__builtin_huge_valf();
                }
            }
            float mx = s[j][0];
#pragma unroll
            for (int r = 1; r < 16; ++r) mx = fmaxf(mx, s[j][r]);
            const u32x2 sw = __builtin_amdgcn_permlane32_swap(__float_as_uint(mx), __float_as_uint(mx), false, false);
            mx = fmaxf(__uint_as_float(sw[0]), __uint_as_float(sw[1])) * a.scale2;
            if (__builtin_amdgcn_ballot_w64(mx > mrow + 8.f)) {
                const float mn = fmaxf(mrow, ceilf(mx));                          // (whole numbers: the factor is a power of two, exact on what is rounded already)
                const float alpha = mrow == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(mrow - mn);
                mrow = mn;
                lrow *= alpha;
#pragma unroll
                for (int n = 0; n < NDT; ++n) o[n] *= alpha;
                if constexpr (j == 1) {
                    sum[0] *= alpha;
                    sum[1] *= alpha;
#pragma unroll
                    for (int q = 0; q < 2; ++q)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            pf[q][e] = T::scaled(pf[q][e], alpha);
                            if constexpr (TWO) pr[q][e] = T::scaled(pr[q][e], alpha);
                        }
                }
            }
            sub = (mrow == -__builtin_huge_valf() ? 0.f : mrow) - T::shift;
        };
        auto exps = [&](auto J_, int slot) {                                     // EPS of tile j's probabilities
            constexpr int j = decltype(J_)::value;
#pragma unroll
            for (int e = 0; e < EPS; ++e) {
                const int r = slot * EPS + e;
                s[j][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[j][r], a.scale2, -sub));
                sum[e & 1] += s[j][r];
                if (r & 1) {
                    unsigned two = T::pack(s[j][r - 1], s[j][r]);
                    asm volatile("" : "+v"(two), "+v"(sum[0]), "+v"(sum[1]));    // (here, not where it is used: the compiler sinks it past the products)
                    pf[2 * j + r / 8][r / 2 % 4] = two;
                    if constexpr (TWO) {
                        unsigned rest = T::pack(s[j][r - 1] - T::up((unsigned short)(two & 0xffffu)), s[j][r] - T::up((unsigned short)(two >> 16)));
                        asm volatile("" : "+v"(rest));
                        pr[2 * j + r / 8][r / 2 % 4] = rest;
                    }
                }
            }
        };
        s[0] = s[1] = (f32x16)(0.f);
#pragma unroll
        for (int f = 0; f < 4; ++f) read_k(f);
#pragma unroll
        for (int f = 0; f < NKK; ++f) {
            s[0] = T::mfma(kf[f & 3], qf[f], s[0]);
            read_k(f + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
        top(std::integral_constant<int, 0>{});
#pragma unroll
        for (int f = 0; f < NKK; ++f) {
            s[1] = T::mfma(kf[f & 3], qf[f], s[1]);
            if (f + 4 < NKK) read_k(NKK + f + 4);
            else read_v(f + 4 - NKK);
            exps(std::integral_constant<int, 0>{}, f);
            __builtin_amdgcn_sched_barrier(0);
        }
        top(std::integral_constant<int, 1>{});
#pragma unroll
        for (int g = 0; g < NKK; ++g) {
            o[g % NDT] = T::mfma(vf[g & 3], pf[g / NDT], o[g % NDT]);
            if constexpr (TWO) o[g % NDT] = T::mfma(vf[g & 3], pr[g / NDT], o[g % NDT]);
            read_v(g + 4);
            exps(std::integral_constant<int, 1>{}, g);
            __builtin_amdgcn_sched_barrier(0);
        }
        lrow += sum[0] + sum[1];
#pragma unroll
        for (int g = NKK; g < 2 * NKK; ++g) {
            o[g % NDT] = T::mfma(vf[g & 3], pf[g / NDT], o[g % NDT]);
            if constexpr (TWO) o[g % NDT] = T::mfma(vf[g & 3], pr[g / NDT], o[g % NDT]);
            if (g + 4 < 2 * NKK) read_v(g + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto landed = [&](int later) {                                               // own pieces of all but the last `later` chunks requested
        if (later) asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * PPW) : "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    };

    for (int i = 0; i < n; ++i) {
        if (i == np && i > 0 && a.inter) { load_q(false); pin_q(); }
        landed(i == 0 && n > 1);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");             // everyone's pieces; the chunk before is used up
        if (i > 0 && i + 1 < n) issue(i + 1);
        const int md = mode(i);
        if (md != SKIP) product(i, md);
    }
    prompt_finish<T, HD>(o, mrow, lrow, row, token, head, lo, hi, live, split, kvh, (int64_t)p0 * KC, (int64_t)(p0 + np) * KC,
                         (int64_t)k0 + (int64_t)o0 * KC, (int64_t)k0 + (int64_t)(o0 + n - np) * KC, s_q[w]);
}

// the splits' partials of a row -> the output: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.  HD / 4 lanes hold four dims each; PAR
// such groups take every PAR-th split of a row and meet in LDS, always in the same order.  One group up to 8 splits: all of its loads
// are in flight at once (128 single tokens take 6 % longer, their tiles included, with four groups); four beyond, where one would go
// through them as a chain (34 us at 64 splits, four 5.5) and eight are too many workgroups (64 single tokens behind 2048: 5 % longer).
// Bound by latency (5.5 us for 128 rows x 64 splits of 128 dims) and by the L2s' 17 MB of partials (5.7 us for 2048 rows x 16 splits: 3 TB/s).
template <class T, int HD, int PAR>
__global__ void __launch_bounds__(256) prompt_join_kernel(PromptArgs a) {
    constexpr int LPR = HD / 4, RPB = 256 / LPR / PAR;                           // lanes of a group, rows of a workgroup
    __shared__ float4 s_o[PAR][RPB][LPR];
    __shared__ float2 s_ml[PAR][RPB];
    const int rows = a.n_tokens * a.G, g = threadIdx.x / LPR % PAR, rb = threadIdx.x / LPR / PAR, ln = threadIdx.x % LPR;
    const int64_t n = (int64_t)rows * a.n_kv, i = (int64_t)blockIdx.x * RPB + rb, at = i < n ? i : n - 1;
    float m = -__builtin_huge_valf(), l = 0.f;
    const float kind = a.part_ml[at].y;                                          // -1: no text's row, -2: sees no key, otherwise a sum (or NaN)
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float2 ml, float4 x) {                                        // (a split that saw no key of the row has zeros and the maximum -inf)
        const float mn = fmaxf(m, ml.x), sub = mn == -__builtin_huge_valf() ? 0.f : mn;
        const float f = m == -__builtin_huge_valf() ? 0.f : __builtin_amdgcn_exp2f(m - sub), e = ml.x == -__builtin_huge_valf() && ml.y <= 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - sub);
        m = mn;
        l = l * f + e * ml.y;
        o.x = o.x * f + e * x.x; o.y = o.y * f + e * x.y; o.z = o.z * f + e * x.z; o.w = o.w * f + e * x.w;
    };
    constexpr int U = 8;                                                          // partials in flight
    for (int s0 = g; s0 < a.splits; s0 += U * PAR) {
        float2 ml[U];
        float4 x[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t s = min(s0 + u * PAR, a.splits - 1);
            ml[u] = a.part_ml[s * n + at];
            x[u] = *reinterpret_cast<const float4 *>(a.part_o + (s * n + at) * HD + ln * 4);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (s0 + u * PAR < a.splits) add(ml[u], x[u]);
    }
    if constexpr (PAR > 1) {
        s_o[g][rb][ln] = o;
        if (ln == 0) s_ml[g][rb] = make_float2(m, l);
        __syncthreads();
        if (g) return;
        for (int q = 1; q < PAR; ++q) add(s_ml[q][rb], s_o[q][rb][ln]);
    }
    if (i >= n) return;
    if (kind == -1.f && !a.zero_rest) return;
    const int d = ln * 4, kvh = (int)(i / rows), row = (int)(i % rows), token = row / a.G, head = kvh * a.G + row % a.G;
    const float inv = 1.0f / l;
    if (!(kind < 0.f)) prompt_store4<T, HD>(a, token, head, d, o.x * inv, o.y * inv, o.z * inv, o.w * inv);
    else prompt_store4<T, HD>(a, token, head, d, 0.f, 0.f, 0.f, 0.f);
}

// ---------------------------------------------------------------------------------------------------------------------
// Pages
// ---------------------------------------------------------------------------------------------------------------------
// What moves keys and values is bound by HBM where it moves much and by the launch (3 - 4 us) where it does not; a thread moves 16
// bytes, neighbours neighbouring ones on both sides.

// page numbers into an entry's table (they travel as kernel arguments: stream order is all that a later reader needs); 1.4 us
struct PcTableArgs {
    int32_t *dst;
    int n;
    int32_t val[960];
};
__global__ void __launch_bounds__(256) pc_table_kernel(PcTableArgs a) {
    for (int i = threadIdx.x; i < a.n; i += 256) a.dst[i] = a.val[i];
}

// keys and values of n tokens into the pages of an entry: a thread per (layer, token, key head, 8 dims) and K / V.  4000 tokens of 28
// layers (229 MB read and written): 36 us, 6.3 TB/s; 37 tokens: 3.2 us.
// k_inter: the source's dims are interleaved by rotary pair (2 f + h = pair f, half h); v_dim != 1: the source is V^T, elements
// v_dim apart.  Both only where the encoder stores a prompt, once.
struct PcWriteArgs {
    const bf16_t *k, *v;
    int64_t k_layer, k_token, k_head, v_layer, v_token, v_head, v_dim;
    bf16_t *pages;
    int64_t page_stride, layer_stride;
    const int32_t *table;
    int layer, n_layers, start, n, n_kv, hd, k_inter;
    // pages of the tokens' positions, from start / 64 on, where they travel with the launch: the last n_new of them are new, and the
    // first workgroup enters them in the table (n_pages = 0: the table holds them all)
    int n_pages, n_new;
    int32_t *new_at;
    int32_t pages_of[896];
};
__global__ void __launch_bounds__(256) pc_write_kernel(PcWriteArgs a) {
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < a.n_new; i += 256) a.new_at[i] = a.pages_of[a.n_pages - a.n_new + i];
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
    bf16_t *dst = a.pages + (a.n_pages ? a.pages_of[pos / PC_PAGE - a.start / PC_PAGE] : a.table[pos / PC_PAGE]) * a.page_stride + (a.layer + l) * a.layer_stride +
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

// the first `rows` rows of every (layer, key head, K / V) of page src[j] -> page dst[j].  grid (blocks, jobs): a thread takes four
// words, so that a launch of a few pages fills the chip too.  200 pages of 28 layers (734 MB read and written): 128 us, 5.7 TB/s, with
// the words of the tables where the pages move (a launch of their own took 4.6 us for 200 moves in 1600 words, latency); 200
// copies of 40 rows of one page: 35 us; four: 4.1.
struct PcCopyArgs {
    const bf16_t *from;
    bf16_t *to;
    int64_t page_stride;                  // elements
    int segs, hd, rows;                   // segments of a page: layers x key heads x 2
    // the tables of what is copied, written by the first workgroup of each job: `entry_table` [job] = dst (one entry's pages), or the
    // table of the job's own new entry, which begins with the first `shared` pages of parent_table (tables + kid * ld)
    int32_t *entry_table, *tables;
    const int32_t *parent_table;
    int64_t ld;
    int shared;
    // pages that move: remap_words words of all tables, in which src[j] -> dst[j] (src ascending; words behind an entry's length may
    // change too, nothing reads them).  Neither the copies nor the words wait for the other.
    int n;
    int64_t remap_words;
    int32_t src[320], dst[320], kid[320];
};
__global__ void __launch_bounds__(256) pc_copy_kernel(PcCopyArgs a) {
    if (blockIdx.x == 0) {
        if (a.entry_table && threadIdx.x == 0) a.entry_table[blockIdx.y] = a.dst[blockIdx.y];
        if (a.parent_table) {
            int32_t *t = a.tables + a.kid[blockIdx.y] * a.ld;
            for (int i = threadIdx.x; i <= a.shared; i += 256) t[i] = i < a.shared ? a.parent_table[i] : a.dst[blockIdx.y];
        }
    }
    const int64_t first = ((int64_t)blockIdx.y * gridDim.x + blockIdx.x) * 256;
    if (first < a.remap_words) {                              // (a word each thread, as far as they go, and a search in LDS)
        __shared__ int32_t src[320], dst[320];
        for (int i = threadIdx.x; i < a.n; i += 256) { src[i] = a.src[i]; dst[i] = a.dst[i]; }
        __syncthreads();
        for (int64_t i = first + threadIdx.x; i < a.remap_words; i += (int64_t)gridDim.y * gridDim.x * 256) {
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
    const int per = a.rows * a.hd / 8;                        // 16-byte words of a segment
    const int64_t total = (int64_t)a.segs * per;
    const bf16_t *s = a.from + a.src[blockIdx.y] * a.page_stride;
    bf16_t *d = a.to + a.dst[blockIdx.y] * a.page_stride;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
        const int64_t off = (i / per * PC_PAGE * a.hd) + i % per * 8;
        *reinterpret_cast<uint4 *>(d + off) = *reinterpret_cast<const uint4 *>(s + off);
    }
}

// words of new pages and tables: zeros
__global__ void __launch_bounds__(256) pc_zero_kernel(uint32_t *p, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

// the tables of new entries that begin as `parent` does, its pages all full
struct PcForkArgs {
    int32_t *tables;
    int64_t ld;
    int parent, shared, n;
    int32_t entry[480];
};
__global__ void __launch_bounds__(256) pc_fork_kernel(PcForkArgs a) {
    const int32_t *p = a.tables + a.parent * a.ld;
    int32_t *t = a.tables + a.entry[blockIdx.x] * a.ld;
    for (int i = threadIdx.x; i < a.shared; i += 256) t[i] = p[i];
}

}  // namespace mipc
