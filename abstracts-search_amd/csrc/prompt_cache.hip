// prompt_cache.hip -- the prompt cache of include/mi_encoder.h: bookkeeping of entries and pages on the host, kernels of
// prompt_kernels.h.
#include "prompt_cache.h"

#include <algorithm>
#include <cstring>
#include <memory>
#include <mutex>
#include <vector>

#include "prompt_kernels.h"

using namespace mi;
using namespace mipc;

namespace {

hipStream_t as_stream(void *s) { return reinterpret_cast<hipStream_t>(s); }
// stands for "whatever work used it is done": a page or an entry's place may be used on any stream
void *const ANY = reinterpret_cast<void *>(~uintptr_t(0));
// .. and for work of several streams: equal to none, so that whoever takes the page waits for the device
void *const SEVERAL = reinterpret_cast<void *>(~uintptr_t(1));

// work on a is in order with work on b (the per-thread handle is another stream in every thread)
bool same(void *a, void *b) { return a == b && a != reinterpret_cast<void *>(hipStreamPerThread); }

bool capturing(void *stream) {
    hipStreamCaptureStatus st = hipStreamCaptureStatusNone;
    MI_HIP(hipStreamIsCapturing(as_stream(stream), &st));
    return st != hipStreamCaptureStatusNone;
}

// a set of page numbers, read lowest first
struct PageSet {
    std::vector<uint64_t> bits;
    int count = 0;
    void reset(int n, int from) {                 // from .. n - 1
        bits.assign(((size_t)n + 63) / 64, 0);
        count = 0;
        for (int p = from; p < n; ++p) insert(p);
    }
    void insert(int p) { bits[p >> 6] |= 1ull << (p & 63); ++count; }
    void erase(int p) { bits[p >> 6] &= ~(1ull << (p & 63)); --count; }
    template <class F>
    void each(F &&f) const {                      // f(p) returns whether to go on
        for (size_t w = 0; w < bits.size(); ++w)
            for (uint64_t b = bits[w]; b; b &= b - 1)
                if (!f((int32_t)(w * 64 + __builtin_ctzll(b)))) return;
    }
};

struct Entry {
    bool live = false;
    int len = 0;
    std::vector<int32_t> pages;
    void *home = nullptr;      // the stream it was made on
    bool foreign = false;      // other streams or a captured graph read it: freeing it waits for the device
    int graph_from = INT32_MAX;   // captured writes (whose replays come when they come) reach its pages from this one on: never shared
    void *slot_tag = ANY;      // not live: the stream whose work may still read its table
};

}  // namespace

struct mi_prompt_cache {
    mi_prompt_cache_cfg cfg{};
    int device = 0;
    int64_t layer_stride = 0, page_stride = 0;   // elements
    int table_ld = 0;
    bf16_t *pages = nullptr;
    DevBuf own, tables;
    std::mutex mu;
    std::vector<int32_t> ref;            // entries that hold the page
    std::vector<void *> tag;             // the stream on which entries gave the page up: their work may still read it
    PageSet free_pages;
    std::vector<Entry> entries;

    Entry &at(int32_t e) {
        MI_REQUIRE(e >= 0 && e < (int32_t)entries.size() && entries[e].live, "prompt cache: no such entry");
        return entries[e];
    }
    int32_t *table(int32_t e) const { return tables.get<int32_t>() + (int64_t)e * table_ld; }

    void wait_all() {                    // everything issued so far is done: whatever is free is free for every stream
        wait_for_device();
        std::fill(tag.begin(), tag.end(), ANY);
        for (Entry &e : entries)
            if (!e.live) e.slot_tag = ANY;
    }
    // the n lowest free pages, fit for use on `stream` (still free: the caller takes them once its launches are out)
    std::vector<int32_t> pick_pages(int n, void *stream) {
        if (n > free_pages.count) throw Error("prompt cache: " + std::to_string(n) + " pages needed, " + std::to_string(free_pages.count) + " free");
        std::vector<int32_t> got;
        got.reserve(n);
        if (n) free_pages.each([&](int32_t p) { got.push_back(p); return (int)got.size() < n; });
        for (int32_t p : got)
            if (tag[p] != ANY && !same(tag[p], stream)) { wait_all(); break; }
        return got;
    }
    void take(int32_t p) { free_pages.erase(p); ref[p] = 1; tag[p] = ANY; }
    void drop(int32_t p, void *stream) {
        if (stream != ANY) tag[p] = tag[p] == ANY || same(tag[p], stream) ? stream : SEVERAL;
        if (--ref[p] == 0) free_pages.insert(p);
    }
    std::vector<int32_t> pick_entries(int n, void *stream) {
        std::vector<int32_t> got;
        for (int32_t e = 0; e < (int32_t)entries.size() && (int)got.size() < n; ++e)
            if (!entries[e].live) got.push_back(e);
        if ((int)got.size() != n) throw Error("prompt cache: more than max_entries (" + std::to_string(cfg.max_entries) + ") entries");
        for (int32_t e : got)
            if (entries[e].slot_tag != ANY && !same(entries[e].slot_tag, stream)) { wait_all(); break; }
        return got;
    }
    void open(int32_t e, int len, std::vector<int32_t> pg, void *stream) {
        Entry &x = entries[e];
        x.live = true; x.len = len; x.pages = std::move(pg); x.home = stream; x.foreign = false; x.graph_from = INT32_MAX; x.slot_tag = ANY;
    }
    void reads(Entry &e, void *stream, bool cap) {
        if (cap || !same(stream, e.home)) e.foreign = true;
    }
    // src[j] -> dst[j]; into: the new entry that the pages dst make up; kids, parent: the new entries that fork `parent`; move: the pages
    // leave src, whose numbers in all tables become dst's (ascending, and no page goes up: a word that one launch of the list has
    // rewritten is below all that later ones look for)
    void copy_pages(const bf16_t *from, bf16_t *to, const int32_t *src, const int32_t *dst, int n, int rows, hipStream_t st, int32_t into = -1,
                    const int32_t *kids = nullptr, int32_t parent = -1, int shared = 0, bool move = false);
    void check_room(const Entry &e, int32_t n) const {
        const int64_t most = cfg.max_tokens ? cfg.max_tokens : (int64_t)table_ld * PC_PAGE;
        if (n < 0 || (int64_t)e.len + n > most) throw Error("prompt cache: an entry holds at most " + std::to_string(most) + " tokens");
    }
    // the pages that n more tokens of an entry need, fit for use on `stream`
    std::vector<int32_t> pages_for(Entry &e, int32_t n, void *stream) {
        const int have = (int)e.pages.size(), need = (int)(((int64_t)e.len + n + PC_PAGE - 1) / PC_PAGE);
        if (need <= have) return {};
        std::vector<int32_t> got = pick_pages(need - have, stream);
        if (!same(stream, e.home)) {     // (its table may be in use on the home stream)
            wait_all();
            e.foreign = true;
        }
        return got;
    }
    void grow(Entry &e, int32_t n, const std::vector<int32_t> &got) {
        for (int32_t p : got) { take(p); e.pages.push_back(p); }
        e.len += n;
    }
    void set_table(int32_t e, int at_, const int32_t *val, int n, hipStream_t st);
};

void mi_prompt_cache::copy_pages(const bf16_t *from, bf16_t *to, const int32_t *src, const int32_t *dst, int n, int rows, hipStream_t st, int32_t into,
                                 const int32_t *kids, int32_t parent, int shared, bool move) {
    PcCopyArgs a{};
    a.from = from; a.to = to; a.page_stride = page_stride; a.segs = cfg.n_layers * cfg.n_kv_heads * 2; a.hd = cfg.head_dim; a.rows = rows;
    a.tables = tables.get<int32_t>(); a.ld = table_ld; a.shared = shared;
    if (kids) a.parent_table = table(parent);
    if (move) a.remap_words = (int64_t)cfg.max_entries * table_ld;
    constexpr int most = sizeof a.src / sizeof a.src[0];
    const int64_t words = (int64_t)a.segs * rows * cfg.head_dim / 8;
    for (int j0 = 0; j0 < n; j0 += most) {
        const int m = std::min(most, n - j0);
        a.n = m;
        std::copy(src + j0, src + j0 + m, a.src);
        std::copy(dst + j0, dst + j0 + m, a.dst);
        if (kids) std::copy(kids + j0, kids + j0 + m, a.kid);
        if (into >= 0) a.entry_table = table(into) + j0;
        hipLaunchKernelGGL(pc_copy_kernel, dim3((unsigned)((words + 1023) / 1024), (unsigned)m), dim3(256), 0, st, a);
        MI_HIP(hipGetLastError());
    }
}

void mi_prompt_cache::set_table(int32_t e, int at_, const int32_t *val, int n, hipStream_t st) {
    PcTableArgs a{};
    for (int i0 = 0; i0 < n; i0 += 960) {
        a.n = std::min(960, n - i0);
        a.dst = table(e) + at_ + i0;
        std::copy(val + i0, val + i0 + a.n, a.val);
        hipLaunchKernelGGL(pc_table_kernel, dim3(1), dim3(256), 0, st, a);
        MI_HIP(hipGetLastError());
    }
}

namespace {

// zeros by a kernel, which a capture in another thread does not mind
void zero(void *p, size_t bytes, hipStream_t st) {
    hipLaunchKernelGGL(pc_zero_kernel, dim3((unsigned)std::min<size_t>(4096, bytes / 4096 + 1)), dim3(256), 0, st, static_cast<uint32_t *>(p), (int64_t)(bytes / 4));
    MI_HIP(hipGetLastError());
}

// memory that a kernel on `device` may use
bool on_device(const void *p, int device) {
    hipPointerAttribute_t attr;
    if (hipPointerGetAttributes(&attr, p) != hipSuccess) {
        (void)hipGetLastError();
        return false;
    }
    return attr.type == hipMemoryTypeManaged || (attr.type == hipMemoryTypeDevice && attr.device == device);
}
bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

void check_strides(const mi_prompt_cache *c, int n, const void *k, const int64_t *ks, const void *v, const int64_t *vs) {
    MI_REQUIRE(aligned16(k) && aligned16(v), "prompt cache: keys and values must be 16-byte aligned");
    MI_REQUIRE(!n || (on_device(k, c->device) && on_device(v, c->device)), "prompt cache: memory of the cache's device only");
    for (int i = 0; i < 3; ++i) MI_REQUIRE(ks[i] % 8 == 0 && vs[i] % 8 == 0, "prompt cache: strides must be multiples of 8 elements");
}
void write_sources(PcWriteArgs &a, const void *k, const int64_t *ks, const void *v, const int64_t *vs) {
    a.k = static_cast<const bf16_t *>(k); a.k_layer = ks[0]; a.k_token = ks[1]; a.k_head = ks[2];
    a.v = static_cast<const bf16_t *>(v); a.v_layer = vs[0]; a.v_token = vs[1]; a.v_head = vs[2]; a.v_dim = 1;
}
void write_args(mi_prompt_cache *c, int32_t entry, int32_t layer, int32_t n_layers, int32_t start, int32_t n, PcWriteArgs &a, void *stream) {
    Entry &e = c->at(entry);
    MI_REQUIRE(layer >= 0 && n_layers >= 1 && n_layers <= c->cfg.n_layers - layer, "prompt cache: layer out of range");
    MI_REQUIRE(start >= 0 && n >= 0 && n <= e.len - start, "prompt cache: tokens out of the entry's range");
    const bool cap = capturing(stream);
    bool wait = false;                   // an entry that shared a page gave it up on another stream, where its reading may be under way
    for (int p = start / PC_PAGE; p < (start + n + PC_PAGE - 1) / PC_PAGE; ++p) {
        MI_REQUIRE(c->ref[e.pages[p]] == 1, "prompt cache: tokens in a page that other entries share cannot be written");
        void *const t = c->tag[e.pages[p]];
        wait = wait || (t != ANY && (!same(t, stream) || cap));         // (a replay may run on any stream)
    }
    if (wait) c->wait_all();
    if (cap && n) e.graph_from = std::min(e.graph_from, start / PC_PAGE);
    c->reads(e, stream, cap);
    a.pages = c->pages; a.page_stride = c->page_stride; a.layer_stride = c->layer_stride; a.table = c->table(entry);
    a.layer = layer; a.n_layers = n_layers; a.start = start; a.n = n; a.n_kv = c->cfg.n_kv_heads; a.hd = c->cfg.head_dim;
}
void write_launch(const PcWriteArgs &a, void *stream) {
    const int64_t total = (int64_t)a.n_layers * a.n * a.n_kv * (a.hd / 8) * 2, blocks = (total + 255) / 256;
    if (!blocks) return;
    MI_REQUIRE(blocks <= 0x7fffffff, "prompt cache: write of more than 2^31 blocks");
    hipLaunchKernelGGL(pc_write_kernel, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), a);
    MI_HIP(hipGetLastError());
}

// checks what the kernels take for granted, and fills in their arguments
PromptArgs attention_args(mi_prompt_cache *c, const mi_prompt_attn &x, const PromptForms &f) {
    const mi_prompt_cache_cfg &g = c->cfg;
    Entry &e = c->at(x.entry);
    MI_REQUIRE(x.layer >= 0 && x.layer < g.n_layers, "prompt attention: layer out of range");
    MI_REQUIRE(x.n_heads > 0 && x.n_heads % g.n_kv_heads == 0, "prompt attention: n_heads must be a multiple of the cache's n_kv_heads");
    MI_REQUIRE(x.n_tokens >= 0 && x.n_keys >= 0 && x.n_texts >= 1, "prompt attention: negative count, or no text");
    MI_REQUIRE(x.n_tokens <= 0x7fffff00 / x.n_heads, "prompt attention: more than 2^31 rows");
    MI_REQUIRE(x.n_keys <= 0x7fffff00, "prompt attention: more than 2^31 keys");   // (a chunk's end stays an int)
    MI_REQUIRE(!x.n_tokens || (x.q && x.out), "null argument");
    MI_REQUIRE(!x.n_keys || (x.k && x.v), "null argument");
    MI_REQUIRE((x.cu_q != nullptr) == (x.cu_k != nullptr), "prompt attention: cu_q and cu_k come together");
    MI_REQUIRE(x.cu_q || x.n_texts == 1, "prompt attention: several texts need cu_q and cu_k");
    MI_REQUIRE(x.scale >= 0.f && x.scale < __builtin_huge_valf(), "prompt attention: scale must be finite and not negative");
    for (const void *p : {x.q, x.k, x.v, static_cast<const void *>(x.out)}) MI_REQUIRE(aligned16(p), "prompt attention: tensors must be 16-byte aligned");
    for (int64_t s : {x.q_token, x.q_head, x.k_token, x.k_head, x.v_token, x.v_head, x.o_token, x.o_head})
        MI_REQUIRE(s % 8 == 0, "prompt attention: strides must be multiples of 8 elements");
    MI_REQUIRE((x.n_tokens <= 1 || x.o_token) && (x.n_heads == 1 || x.o_head), "prompt attention: rows of out are the same memory");
    MI_REQUIRE(std::max(std::abs(x.k_token), std::abs(x.v_token)) < 1 << 23 && x.k_token >= 0 && x.v_token >= 0,
               "prompt attention: tokens of k and v must be less than 2^23 elements apart");
    PromptArgs a{};
    a.q = static_cast<const bf16_t *>(x.q); a.k = static_cast<const bf16_t *>(x.k); a.v = static_cast<const bf16_t *>(x.v);
    a.out = static_cast<bf16_t *>(x.out);
    a.q_token = x.q_token; a.q_head = x.q_head; a.k_token = x.k_token; a.k_head = x.k_head; a.v_token = x.v_token; a.v_head = x.v_head;
    a.o_token = x.o_token; a.o_head = x.o_head;
    a.pages = c->pages + x.layer * c->layer_stride; a.page_stride = c->page_stride; a.table = c->table(x.entry); a.P = f.prompt_tokens < 0 ? e.len : std::min(f.prompt_tokens, e.len);
    a.n_tokens = x.n_tokens; a.n_keys = x.n_keys; a.n_texts = x.n_texts; a.cu_q = x.cu_q; a.cu_k = x.cu_k;
    a.n_heads = x.n_heads; a.n_kv = g.n_kv_heads; a.G = x.n_heads / g.n_kv_heads; a.causal = x.causal; a.zero_rest = x.zero_rest;
    a.scale2 = std::max(x.scale * 1.4426950408889634f, 1e-30f);   // (0 means equal weights; a masked score is -inf, and 0 x inf is no number)
    a.vt = f.vt; a.inter = f.inter; a.frag = static_cast<bf16_t *>(f.frag); a.frag_mt = f.frag_mt;
    return a;
}

// How a call is cut up: tiles of 128 rows of a key head, and where these do not fill the chip the keys `splits` ways, so that there
// is a workgroup for each of the 256 CUs -- two, if each still has eight chunks of 64 keys or more: the 1024 chunks of four tokens
// behind 65 500 take a third longer with 32 splits than with 64; but the 82 chunks of 64 single tokens behind 2048 a fifth longer with 32
// than with 16, because every split's partials are written and read again.  Up to 256 rows a split may be one chunk, beyond it is two at
// least (ten tokens of 12 heads behind 400: 8 % less with 8 splits of one than with 4 of two; but 30 single tokens of 28 heads behind 400
// 22 % more with 12 splits than with 7); up to four chunks go unsplit, where the join costs as much as they do (behind 150: 11 % more in two).
struct Plan {
    int splits, tiles;
    int64_t rows;                        // of all key heads
    int64_t o_bytes, bytes;              // partials, workspace
};

Plan plan_of(const PromptArgs &a, int hd) {
    constexpr int R = 32 * PA_WAVES;
    Plan p{};
    const int64_t per_head = (int64_t)a.n_tokens * a.G;
    p.rows = per_head * a.n_kv;
    p.tiles = (int)((per_head + R - 1) / R);
    // chunks that a tile goes through: the prompt's, and its texts' share of the own keys
    const int64_t wgs = (int64_t)p.tiles * a.n_kv, own = a.n_keys * std::min<int64_t>(per_head, R) / per_head;
    const int64_t chunks = (a.P + PC_PAGE - 1) / PC_PAGE + (own + PC_PAGE - 1) / PC_PAGE, target = chunks * wgs >= 8 * 512 ? 512 : 256;
    p.splits = (int)std::max<int64_t>(1, std::min<int64_t>(target / wgs, chunks < 5 ? 1 : p.rows <= 256 ? chunks : chunks / 2));
    p.o_bytes = p.splits > 1 ? p.splits * p.rows * hd * 4 : 0;
    p.bytes = p.splits > 1 ? p.o_bytes + p.splits * p.rows * 8 : 0;
    return p;
}

template <class T, int HD, bool VT>
void attention_launch(const PromptArgs &a, const Plan &p, hipStream_t st) {
    const dim3 grid((unsigned)(((int64_t)p.tiles * p.splits * a.n_kv + 7) / 8 * 8));
    // few rows of a key head: the probabilities in two parts (see the kernel)
    const dim3 block(64 * PA_WAVES);
    if (p.tiles <= 2) hipLaunchKernelGGL((prompt_tile_kernel<T, HD, VT, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((prompt_tile_kernel<T, HD, VT, false>), grid, block, 0, st, a);
    MI_HIP(hipGetLastError());
    if (p.splits > 1) {
        constexpr int per_wg = 256 / (HD / 4);                                    // groups of lanes
        if (p.splits > 8) hipLaunchKernelGGL((prompt_join_kernel<T, HD, 4>), dim3((unsigned)((p.rows + per_wg / 4 - 1) / (per_wg / 4))), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((prompt_join_kernel<T, HD, 1>), dim3((unsigned)((p.rows + per_wg - 1) / per_wg)), dim3(256), 0, st, a);
        MI_HIP(hipGetLastError());
    }
}

}  // namespace

namespace mi {

int64_t prompt_attention_workspace(mi_prompt_cache *c, const mi_prompt_attn &x) {
    std::lock_guard<std::mutex> lk(c->mu);
    const PromptArgs a = attention_args(c, x, PromptForms{});
    return x.n_tokens ? plan_of(a, c->cfg.head_dim).bytes : 0;
}

void prompt_attention(mi_prompt_cache *c, const mi_prompt_attn &x, const PromptForms &f, void *stream) {
    // (held over the launch: a page that this call reads is not moved or given away in between)
    std::lock_guard<std::mutex> lk(c->mu);
    PromptArgs a = attention_args(c, x, f);
    if (!x.n_tokens) return;
    const bool f16 = c->cfg.dtype == MI_DTYPE_F16, wide = c->cfg.head_dim == 128;
    const Plan p = plan_of(a, c->cfg.head_dim);
    MI_REQUIRE(!p.bytes || (x.workspace && aligned16(x.workspace) && x.workspace_bytes >= p.bytes),
               "prompt attention: a workspace of " + std::to_string(p.bytes) + " bytes is needed (mi_prompt_attention_workspace)");
    MI_REQUIRE(!f.vt || !f16, "prompt attention: V^T operands are bf16");
    a.splits = p.splits; a.tiles = p.tiles;
    a.r_tiles = 1.0f / (float)p.tiles; a.r_splits = 1.0f / (float)p.splits; a.r_G = 1.0f / (float)a.G;
    a.part_o = static_cast<float *>(x.workspace);
    a.part_ml = reinterpret_cast<float2 *>(static_cast<char *>(x.workspace) + p.o_bytes);
    c->reads(c->at(x.entry), stream, capturing(stream));
    hipStream_t st = as_stream(stream);
    if (f16) wide ? attention_launch<TF16, 128, false>(a, p, st) : attention_launch<TF16, 64, false>(a, p, st);
    else if (f.vt) wide ? attention_launch<TBf16, 128, true>(a, p, st) : attention_launch<TBf16, 64, true>(a, p, st);
    else wide ? attention_launch<TBf16, 128, false>(a, p, st) : attention_launch<TBf16, 64, false>(a, p, st);
}

void prompt_cache_write_vt(mi_prompt_cache *c, int32_t entry, int32_t layer, int32_t start, int32_t n, const void *k, int64_t k_token, bool k_inter,
                           const void *vt, int64_t ldvt, void *stream) {
    std::lock_guard<std::mutex> lk(c->mu);
    PcWriteArgs a{};
    write_args(c, entry, layer, 1, start, n, a, stream);
    a.k = static_cast<const bf16_t *>(k); a.k_token = k_token; a.k_head = c->cfg.head_dim; a.k_inter = k_inter;
    a.v = static_cast<const bf16_t *>(vt); a.v_token = 1; a.v_head = (int64_t)c->cfg.head_dim * ldvt; a.v_dim = ldvt;
    write_launch(a, stream);
}

}  // namespace mi

extern "C" {

int mi_prompt_cache_create(const mi_prompt_cache_cfg *cfg, int device, void *pages, mi_prompt_cache **out) {
    return guard([&] {
        MI_REQUIRE(cfg && out, "null argument");
        const mi_prompt_cache_cfg &g = *cfg;
        MI_REQUIRE(g.head_dim == 64 || g.head_dim == 128, "prompt cache: head_dim must be 64 or 128");
        MI_REQUIRE(g.dtype == MI_DTYPE_BF16 || g.dtype == MI_DTYPE_F16, "prompt cache: dtype must be bf16 or f16");
        MI_REQUIRE(g.n_layers > 0 && g.n_kv_heads > 0 && g.n_pages > 0 && g.max_entries > 0 && g.max_tokens >= 0, "prompt cache: bad config");
        MI_REQUIRE(g.n_pages <= 0x7fffffff / PC_PAGE, "prompt cache: more than 2^31 tokens");
        MI_REQUIRE((int64_t)g.n_layers * g.n_kv_heads <= 1 << 20, "prompt cache: bad config");
        int ndev = 0;
        if (hipGetDeviceCount(&ndev) != hipSuccess || ndev == 0) {
            (void)hipGetLastError();
            throw Error("no HIP device available: the MI355X prompt cache has no CPU fallback");
        }
        MI_REQUIRE(device >= 0 && device < ndev, "invalid device ordinal");
        MI_REQUIRE(!pages || (aligned16(pages) && on_device(pages, device)), "prompt cache: pages must be 16-byte aligned memory of the device");
        DeviceGuard dg(device);
        auto c = std::make_unique<mi_prompt_cache>();
        c->cfg = g;
        c->device = device;
        c->layer_stride = (int64_t)g.n_kv_heads * 2 * PC_PAGE * g.head_dim;
        c->page_stride = c->layer_stride * g.n_layers;
        c->table_ld = g.max_tokens ? (int)(((int64_t)g.max_tokens + PC_PAGE - 1) / PC_PAGE) : g.n_pages;
        const size_t bytes = (size_t)c->page_stride * 2 * g.n_pages, tbytes = (size_t)g.max_entries * c->table_ld * 4;
        BesideCaptures beside;
        if (!pages) {                    // zeros: what a reserved token holds before it is written is at least finite
            pages = c->own.reserve(bytes);
            zero(pages, bytes, hipStreamPerThread);
        }
        c->pages = static_cast<bf16_t *>(pages);
        zero(c->tables.reserve(tbytes), tbytes, hipStreamPerThread);   // (every word of a table is a page number, whatever is read)
        wait_for_device();
        c->ref.assign(g.n_pages, 0);
        c->tag.assign(g.n_pages, ANY);
        c->free_pages.reset(g.n_pages, 0);
        c->entries.resize(g.max_entries);
        *out = c.release();
    });
}

int mi_prompt_cache_destroy(mi_prompt_cache *c) {
    return guard([&] {
        if (!c) return;
        DeviceGuard dg(c->device);
        BesideCaptures beside;
        wait_for_device();
        delete c;
    });
}

int mi_prompt_cache_new(mi_prompt_cache *c, void *stream, int32_t *entry) {
    return guard([&] {
        MI_REQUIRE(c && entry, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot be made while the stream is captured");
        const int32_t e = c->pick_entries(1, stream)[0];
        c->open(e, 0, {}, stream);
        *entry = e;
    });
}

int mi_prompt_cache_reserve(mi_prompt_cache *c, int32_t entry, int32_t n, void *stream) {
    return guard([&] {
        MI_REQUIRE(c, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot grow while the stream is captured");
        Entry &e = c->at(entry);
        c->check_room(e, n);
        const std::vector<int32_t> got = c->pages_for(e, n, stream);
        if (!got.empty()) c->set_table(entry, (int)e.pages.size(), got.data(), (int)got.size(), as_stream(stream));
        c->grow(e, n, got);
    });
}

int mi_prompt_cache_extend(mi_prompt_cache *c, int32_t entry, int32_t n, const void *k, const int64_t ks[3], const void *v, const int64_t vs[3],
                           void *stream) {
    return guard([&] {
        MI_REQUIRE(c && ks && vs && (!n || (k && v)), "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot grow while the stream is captured");
        Entry &e = c->at(entry);
        c->check_room(e, n);
        check_strides(c, n, k, ks, v, vs);
        const int start = e.len, have = (int)e.pages.size();
        const std::vector<int32_t> got = c->pages_for(e, n, stream);
        PcWriteArgs a{};
        const int first = start / PC_PAGE, touched = have + (int)got.size() - first;
        if (touched <= (int)(sizeof a.pages_of / sizeof a.pages_of[0])) {   // one launch: the pages' numbers go with it
            std::copy(e.pages.begin() + first, e.pages.end(), a.pages_of);
            std::copy(got.begin(), got.end(), a.pages_of + have - first);
            a.n_pages = touched; a.n_new = (int)got.size(); a.new_at = c->table(entry) + have;
        } else {
            c->set_table(entry, have, got.data(), (int)got.size(), as_stream(stream));
        }
        c->grow(e, n, got);
        write_args(c, entry, 0, c->cfg.n_layers, start, n, a, stream);
        write_sources(a, k, ks, v, vs);
        write_launch(a, stream);
    });
}

int mi_prompt_cache_write(mi_prompt_cache *c, int32_t entry, int32_t layer, int32_t n_layers, int32_t start, int32_t n, const void *k,
                          const int64_t ks[3], const void *v, const int64_t vs[3], void *stream) {
    return guard([&] {
        MI_REQUIRE(c && ks && vs && (!n || (k && v)), "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        check_strides(c, n, k, ks, v, vs);
        PcWriteArgs a{};
        write_args(c, entry, layer, n_layers, start, n, a, stream);
        write_sources(a, k, ks, v, vs);
        write_launch(a, stream);
    });
}

int mi_prompt_cache_fork(mi_prompt_cache *c, int32_t entry, int32_t count, int32_t *out, int32_t *page, void *stream) {
    return guard([&] {
        MI_REQUIRE(c && (out || !count), "null argument");
        MI_REQUIRE(count >= 0, "prompt cache: negative count");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot be forked while the stream is captured");
        Entry &e = c->at(entry);
        if (!count) return;
        const std::vector<int32_t> kids = c->pick_entries(count, stream);
        // full pages are shared, but for those that a graph may write later; of the others one is copied as far as it is used, or several whole
        const int pages = (int)e.pages.size(), shared = std::min(e.len / PC_PAGE, e.graph_from), each = pages - shared;
        const int rows = each == 1 && e.len % PC_PAGE ? e.len % PC_PAGE : 0;
        if ((int64_t)each * count > c->cfg.n_pages) throw Error("prompt cache: " + std::to_string((int64_t)each * count) + " pages needed, " + std::to_string(c->free_pages.count) + " free");
        const std::vector<int32_t> own = c->pick_pages(each * count, stream);
        const std::vector<int32_t> base(e.pages.begin(), e.pages.begin() + shared);
        auto pages_of = [&](int j) {
            std::vector<int32_t> pg;
            pg.reserve(pages);
            pg = base;
            pg.insert(pg.end(), own.begin() + (int64_t)j * each, own.begin() + (int64_t)(j + 1) * each);
            return pg;
        };
        hipStream_t st = as_stream(stream);
        if (rows) {
            const std::vector<int32_t> src(count, e.pages[shared]);
            c->copy_pages(c->pages, c->pages, src.data(), own.data(), count, rows, st, -1, kids.data(), entry, shared);
        } else if (each) {
            for (int j = 0; j < count; ++j) {
                c->set_table(kids[j], 0, pages_of(j).data(), pages, st);
                c->copy_pages(c->pages, c->pages, e.pages.data() + shared, own.data() + (int64_t)j * each, each, PC_PAGE, st);
            }
        } else if (shared) {
            PcForkArgs a{};
            a.tables = c->tables.get<int32_t>(); a.ld = c->table_ld; a.parent = entry; a.shared = shared;
            for (int j0 = 0; j0 < count; j0 += 480) {
                a.n = std::min(480, count - j0);
                std::copy(kids.begin() + j0, kids.begin() + j0 + a.n, a.entry);
                hipLaunchKernelGGL(pc_fork_kernel, dim3((unsigned)a.n), dim3(256), 0, st, a);
                MI_HIP(hipGetLastError());
            }
        }
        c->reads(e, stream, false);
        const int len = e.len;
        for (int32_t p : base) c->ref[p] += count;
        for (int32_t p : own) c->take(p);
        for (int j = 0; j < count; ++j) {
            if (page) page[j] = rows ? own[j] : each ? -2 : -1;
            c->open(kids[j], len, pages_of(j), stream);
            out[j] = kids[j];
        }
    });
}

int mi_prompt_cache_copy(mi_prompt_cache *c, int32_t entry, int32_t *copy, void *stream) {
    return guard([&] {
        MI_REQUIRE(c && copy, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot be copied while the stream is captured");
        Entry &e = c->at(entry);
        const int n = (int)e.pages.size();
        const int32_t to = c->pick_entries(1, stream)[0];
        std::vector<int32_t> own = c->pick_pages(n, stream);
        c->copy_pages(c->pages, c->pages, e.pages.data(), own.data(), n, PC_PAGE, as_stream(stream), to);
        c->reads(e, stream, false);
        for (int32_t p : own) c->take(p);
        c->open(to, e.len, std::move(own), stream);
        *copy = to;
    });
}

int mi_prompt_cache_free(mi_prompt_cache *c, int32_t n, const int32_t *list, void *stream) {
    return guard([&] {
        MI_REQUIRE(c && (list || !n) && n >= 0, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: entries cannot be freed while the stream is captured");
        bool wait = false;
        std::vector<bool> seen(c->entries.size());
        for (int32_t i = 0; i < n; ++i) {
            const Entry &e = c->at(list[i]);
            if (seen[list[i]]) throw Error("prompt cache: an entry is freed twice");
            seen[list[i]] = true;
            wait = wait || e.foreign || !same(e.home, stream);
        }
        if (wait) c->wait_all();
        void *const tag = wait ? ANY : stream;
        for (int32_t i = 0; i < n; ++i) {
            Entry &e = c->entries[list[i]];
            for (int32_t p : e.pages) c->drop(p, tag);
            e.live = false;
            e.len = 0;
            e.pages.clear();
            e.slot_tag = tag;
        }
    });
}

int mi_prompt_cache_compact(mi_prompt_cache *c, void *stream, int32_t *moved) {
    return guard([&] {
        MI_REQUIRE(c, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: pages cannot be moved while the stream is captured");
        const int32_t n = c->cfg.n_pages, used = n - c->free_pages.count;
        std::vector<int32_t> dst, src;
        c->free_pages.each([&](int32_t p) {
            if (p < used) dst.push_back(p);
            return p < used;
        });
        for (int32_t p = used; p < n && src.size() < dst.size(); ++p)
            if (c->ref[p]) src.push_back(p);
        if (moved) *moved = (int32_t)src.size();
        if (src.empty()) return;
        bool cross = false;
        for (const Entry &e : c->entries) cross = cross || (e.live && (e.foreign || !same(e.home, stream)));
        for (const std::vector<int32_t> *pages : {&dst, &src})
            for (int32_t p : *pages) cross = cross || (c->tag[p] != ANY && !same(c->tag[p], stream));
        if (cross) c->wait_all();
        c->copy_pages(c->pages, c->pages, src.data(), dst.data(), (int)src.size(), PC_PAGE, as_stream(stream), -1, nullptr, -1, 0, true);
        std::vector<int32_t> to(n);
        for (int32_t p = 0; p < n; ++p) to[p] = p;
        for (size_t j = 0; j < src.size(); ++j) {
            to[src[j]] = dst[j];
            c->ref[dst[j]] = c->ref[src[j]];
            c->ref[src[j]] = 0;
            c->free_pages.erase(dst[j]);
            c->free_pages.insert(src[j]);
            c->tag[dst[j]] = ANY;
            c->tag[src[j]] = stream;
        }
        for (Entry &e : c->entries)
            for (int32_t &p : e.pages) p = to[p];
        if (cross) c->wait_all();        // other streams' next reads find the pages where the tables now say
    });
}

int mi_prompt_cache_resize(mi_prompt_cache *c, void *pages, int32_t n_pages, void *stream) {
    return guard([&] {
        MI_REQUIRE(c, "null argument");
        DeviceGuard dg(c->device);
        std::lock_guard<std::mutex> lk(c->mu);
        MI_REQUIRE(!capturing(stream), "prompt cache: the pool cannot be replaced while the stream is captured");
        std::vector<int32_t> src, dst;
        for (int32_t p = 0; p < c->cfg.n_pages; ++p)
            if (c->ref[p]) { dst.push_back((int32_t)src.size()); src.push_back(p); }
        MI_REQUIRE(n_pages > 0 && n_pages >= (int32_t)src.size(), "prompt cache: " + std::to_string(src.size()) + " pages are in use");
        MI_REQUIRE(n_pages <= 0x7fffffff / PC_PAGE, "prompt cache: more than 2^31 tokens");
        MI_REQUIRE(!pages || (aligned16(pages) && on_device(pages, c->device)), "prompt cache: pages must be 16-byte aligned memory of the device");
        const size_t bytes = (size_t)c->page_stride * 2 * n_pages;
        BesideCaptures beside;
        DevBuf own;
        if (!pages) {
            pages = own.reserve(bytes);
            zero(pages, bytes, as_stream(stream));
        }
        c->wait_all();
        c->copy_pages(c->pages, static_cast<bf16_t *>(pages), src.data(), dst.data(), (int)src.size(), PC_PAGE, as_stream(stream), -1, nullptr, -1, 0, true);
        c->wait_all();
        std::vector<int32_t> to(c->cfg.n_pages, 0), ref(n_pages, 0);
        for (size_t j = 0; j < src.size(); ++j) { to[src[j]] = dst[j]; ref[dst[j]] = c->ref[src[j]]; }
        for (Entry &e : c->entries)
            for (int32_t &p : e.pages) p = to[p];
        c->ref = std::move(ref);
        c->tag.assign(n_pages, ANY);
        c->free_pages.reset(n_pages, (int)src.size());
        c->pages = static_cast<bf16_t *>(pages);
        c->cfg.n_pages = n_pages;
        std::swap(c->own.p, own.p);
        std::swap(c->own.cap, own.cap);
    });
}

int mi_prompt_cache_entry(mi_prompt_cache *c, int32_t entry, int32_t *length, int32_t *table, int32_t cap) {
    return guard([&] {
        MI_REQUIRE(c, "null argument");
        std::lock_guard<std::mutex> lk(c->mu);
        const Entry &e = c->at(entry);
        if (length) *length = e.len;
        if (table)
            for (int32_t i = 0; i < cap && i < (int32_t)e.pages.size(); ++i) table[i] = e.pages[i];
    });
}

int mi_prompt_cache_used(mi_prompt_cache *c, int32_t *used_pages, int32_t *entries) {
    return guard([&] {
        MI_REQUIRE(c, "null argument");
        std::lock_guard<std::mutex> lk(c->mu);
        if (used_pages) *used_pages = c->cfg.n_pages - c->free_pages.count;
        if (entries) *entries = (int32_t)std::count_if(c->entries.begin(), c->entries.end(), [](const Entry &e) { return e.live; });
    });
}

int mi_prompt_attention_workspace(mi_prompt_cache *c, const mi_prompt_attn *a, int64_t *bytes) {
    return guard([&] {
        MI_REQUIRE(c && a && bytes, "null argument");
        *bytes = prompt_attention_workspace(c, *a);
    });
}

int mi_prompt_attention(mi_prompt_cache *c, const mi_prompt_attn *a, void *stream) {
    return guard([&] {
        MI_REQUIRE(c && a, "null argument");
        DeviceGuard dg(c->device);
        for (const void *p : {a->q, a->k, a->v, static_cast<const void *>(a->out), static_cast<const void *>(a->cu_q), static_cast<const void *>(a->cu_k),
                              static_cast<const void *>(a->workspace)})
            MI_REQUIRE(!p || on_device(p, c->device), "prompt attention: memory of the cache's device only");
        prompt_attention(c, *a, PromptForms{}, stream);
    });
}

}  // extern "C"
