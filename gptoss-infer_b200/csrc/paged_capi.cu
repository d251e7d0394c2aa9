// C ABI of the paged key/value cache and its operators (include/gptoss.h): argument checks, the pool handle with its
// workspaces, and the per-thread workspace of the beam selection.
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include "capi_guard.h"
#include "common.cuh"
#include "gptoss.h"
#include "paged.h"
#include "tma.h"

using gpt::abi_guard;
using gpt::require;

struct gptoss_kv_pool {
    gpt::KvPages pages{};
    gpt::KvMaps maps{};
    int box_log = 0;
    gpt::FastDiv div{};
    int type = 0, dim = 0, device = 0;
    int* err = nullptr;
    void* attn_ws = nullptr;
    void* page_mem = nullptr;                 // of page_ws
    gpt::PageWs page_ws{};

    gpt::KvView view(int layer) const {
        gpt::KvView v{};
        v.k = pages.k + layer * pages.layer_stride;
        v.v = pages.v + layer * pages.layer_stride;
        v.page_stride = pages.page_stride;
        v.token_stride = pages.token_stride;
        v.head_stride = pages.head_stride;
        v.num_pages = pages.num_pages;
        v.kv_heads = pages.kv_heads;
        v.dim = dim;
        v.page = div;
        v.err = err;
        v.layer = layer;
        v.box_log = box_log;
        return v;
    }
    ~gptoss_kv_pool() {
        cudaFree(err);
        cudaFree(attn_ws);
        cudaFree(page_mem);
    }
};

namespace {

bool aligned(const void* p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }
bool known_type(int t) { return t >= gpt::kF32 && t <= gpt::kBF16; }
int type_bytes(int t) { return t == gpt::kF32 ? 4 : 2; }

void check_pool(const gptoss_kv_pool* p, const char* who) {
    if (!p) throw std::runtime_error(std::string(who) + ": null pool");
}

// The pool's buffers live on the device that was current at its creation.
void check_device(const gptoss_kv_pool* p, const char* who) {
    int dev = -1;
    GPT_CHECK(cudaGetDevice(&dev));
    if (dev != p->device) throw std::runtime_error(std::string(who) + ": the pool was created on another device");
}

gpt::KvBatch check_batch(const gptoss_kv_pool* p, int layer, const gptoss_kv_batch* b, const char* who) {
    const std::string w(who);
    check_pool(p, who);
    if (layer < 0 || layer >= p->pages.layers) throw std::runtime_error(w + ": layer outside the pool");
    if (!b) throw std::runtime_error(w + ": null batch");
    if (b->seqs < 0 || b->tokens < 0 || b->max_new < 0 || b->table_stride < 0)
        throw std::runtime_error(w + ": negative size in the batch");
    if (b->seqs > 0 && b->tokens > 0 && (!b->cu_tokens || !b->kv_lens || (!b->tables && b->table_stride > 0)))
        throw std::runtime_error(w + ": null pointer in the batch");
    gpt::KvBatch r{};
    r.cu = b->cu_tokens;
    r.lens = b->kv_lens;
    r.tables = b->tables;
    r.seqs = b->seqs;
    r.tokens = b->tokens;
    r.table_stride = b->table_stride;
    r.max_new = b->max_new;
    r.most = gpt::most_positions(b->table_stride, p->pages.page_size);
    return r;
}

// Grow-only workspace owned by the calling thread, one per device, zeroed when made. A stream capture keeps the address
// that its call had, so what growth leaves behind stays until the thread ends (each is at least twice the one before it,
// or 64 MB larger).
struct ThreadWs {
    struct Held {
        std::vector<void*> all;               // the last is the present one
        size_t n = 0;
    };
    Held held[64];
    ~ThreadWs() {
        for (const Held& h : held)
            for (void* p : h.all) cudaFree(p);
    }
    void* get(size_t bytes) {
        int dev = 0;
        GPT_CHECK(cudaGetDevice(&dev));
        if (dev < 0 || dev >= 64) throw std::runtime_error("device index out of range");
        Held& h = held[dev];
        if (h.n < bytes) {
            const size_t n = std::max(bytes, h.n + std::min(h.n, size_t(64) << 20));
            h.all.reserve(h.all.size() + 1);
            void* p = nullptr;
            GPT_CHECK(cudaMalloc(&p, n));
            h.all.push_back(p);
            h.n = 0;                          // until it is zeroed
            GPT_CHECK(cudaMemset(p, 0, n));
            GPT_CHECK(cudaDeviceSynchronize());   // the caller's stream may not be ordered with the memset's
            h.n = n;
        }
        return h.all.back();
    }
};
thread_local ThreadWs g_beam_ws;

}  // namespace

extern "C" {

gptoss_kv_pool* gptoss_kv_pool_create(void* k, void* v, int type, int layers, int num_pages, int page_size,
                                      int kv_heads, int head_dim, const long long* strides) {
    gptoss_kv_pool* made = nullptr;
    const int rc = abi_guard([&] {
        require(type == gpt::kF16 || type == gpt::kBF16, "kv_pool_create: the cache type is 1 (fp16) or 2 (bf16)");
        require(head_dim == 64 || head_dim == 128, "kv_pool_create: head_dim is 64 or 128");
        require(layers >= 1 && num_pages >= 1 && page_size >= 1 && kv_heads >= 1,
                "kv_pool_create: layers, num_pages, page_size and kv_heads are at least 1");
        require(kv_heads <= 1024 && page_size <= (1 << 20) && layers <= 4096,
                "kv_pool_create: kv_heads <= 1024, page_size <= 2^20, layers <= 4096");
        require(k && v && strides, "kv_pool_create: null pointer");
        require(aligned(k, 16) && aligned(v, 16), "kv_pool_create: k and v must be 16-byte aligned");
        for (int i = 0; i < 4; ++i)
            require(strides[i] >= 0 && strides[i] % 8 == 0, "kv_pool_create: strides are multiples of 8 elements");
        auto p = std::unique_ptr<gptoss_kv_pool>(new gptoss_kv_pool);
        p->pages.k = static_cast<char*>(k);
        p->pages.v = static_cast<char*>(v);
        p->pages.layer_stride = strides[0] * 2;
        p->pages.page_stride = strides[1] * 2;
        p->pages.token_stride = strides[2] * 2;
        p->pages.head_stride = strides[3] * 2;
        p->pages.layers = layers;
        p->pages.num_pages = num_pages;
        p->pages.page_size = page_size;
        p->pages.kv_heads = kv_heads;
        p->pages.row_bytes = head_dim * 2;
        p->type = type;
        p->dim = head_dim;
        p->div = gpt::FastDiv::of(uint32_t(page_size));
        p->box_log = gpt::make_kv_maps(p->pages, head_dim, type == gpt::kBF16, &p->maps);
        GPT_CHECK(cudaGetDevice(&p->device));
        GPT_CHECK(cudaMalloc(&p->err, sizeof(int)));
        GPT_CHECK(cudaMemset(p->err, 0, sizeof(int)));
        p->pages.err = p->err;
        const size_t n = gpt::paged_attention_ws_bytes(head_dim);
        GPT_CHECK(cudaMalloc(&p->attn_ws, n));
        GPT_CHECK(cudaMemset(p->attn_ws, 0, n));
        const size_t pages_n = gpt::kv_pages_ws_bytes(num_pages);
        GPT_CHECK(cudaMalloc(&p->page_mem, pages_n));
        GPT_CHECK(cudaMemset(p->page_mem, 0, pages_n));
        p->page_ws = gpt::make_kv_pages_ws(p->page_mem, num_pages);
        GPT_CHECK(cudaDeviceSynchronize());
        made = p.release();
    });
    return rc == 0 ? made : nullptr;
}

void gptoss_kv_pool_destroy(gptoss_kv_pool* p) { delete p; }

int gptoss_kv_pool_status(gptoss_kv_pool* p, int* code) {
    return abi_guard([&] {
        check_pool(p, "kv_pool_status");
        require(code != nullptr, "kv_pool_status: null output");
        check_device(p, "kv_pool_status");
        GPT_CHECK(cudaDeviceSynchronize());
        GPT_CHECK(cudaMemcpy(code, p->err, sizeof(int), cudaMemcpyDeviceToHost));
        if (*code) {
            GPT_CHECK(cudaMemset(p->err, 0, sizeof(int)));
            GPT_CHECK(cudaDeviceSynchronize());   // or it could clear what a later call on another stream reports
        }
    });
}

int gptoss_kv_append(gptoss_kv_pool* p, int layer, const gptoss_kv_batch* batch, const void* q, const void* k,
                     const void* v, int type, long long q_stride, long long kv_stride, int q_heads,
                     const float* cos_t, const float* sin_t, int positions, int rot_dim, int interleaved, void* q_out,
                     int q_out_type, void* stream) {
    return abi_guard([&] {
        const gpt::KvBatch b = check_batch(p, layer, batch, "kv_append");
        require(known_type(type) && known_type(q_out_type), "kv_append: unknown type");
        require(q_heads >= 0 && q_heads <= 4096, "kv_append: q_heads must be 0 .. 4096");
        require(rot_dim >= 0 && rot_dim <= p->dim && rot_dim % 2 == 0, "kv_append: rot_dim is even and at most head_dim");
        require(positions >= 0, "kv_append: negative positions");
        if (b.seqs == 0 || b.tokens == 0) return;
        require(k && v && (q_heads == 0 || (q && q_out)), "kv_append: null pointer");
        require(rot_dim == 0 || (cos_t && sin_t && positions > 0), "kv_append: null cos/sin table");
        require(q_stride >= (long long)q_heads * p->dim || b.tokens == 1, "kv_append: q_stride is shorter than a row");
        require(kv_stride >= (long long)p->pages.kv_heads * p->dim || b.tokens == 1,
                "kv_append: kv_stride is shorter than a row");
        const int e = type_bytes(type);
        require(aligned(k, e) && aligned(v, e) && aligned(q, e) && aligned(q_out, type_bytes(q_out_type)),
                "kv_append: a pointer is not aligned to its type");
        check_device(p, "kv_append");
        gpt::AppendArgs a{q, k, v, q_stride, kv_stride, cos_t, sin_t, q_out, type, q_out_type, p->type, q_heads,
                          positions, rot_dim, interleaved != 0};
        gpt::launch_kv_append(p->view(layer), b, a, static_cast<cudaStream_t>(stream));
    });
}

int gptoss_paged_attention(gptoss_kv_pool* p, int layer, const gptoss_kv_batch* batch, const void* q, int type,
                           long long q_stride, int q_heads, const float* sinks, float scale, int window, void* out,
                           long long out_stride, void* stream) {
    return abi_guard([&] {
        const gpt::KvBatch b = check_batch(p, layer, batch, "paged_attention");
        require((type == gpt::kF32 && p->type == gpt::kF16) || type == p->type,
                "paged_attention: q and out have the cache's type, or are fp32 beside an fp16 cache");
        const int kvh = p->pages.kv_heads;
        require(q_heads >= kvh && q_heads % kvh == 0 && q_heads <= 4096,
                "paged_attention: q_heads is a multiple of kv_heads, at most 4096");
        require(window >= 0, "paged_attention: negative window");
        require(std::isfinite(scale) && scale != 0.f, "paged_attention: the scale must be finite and not 0");
        if (b.seqs == 0 || b.tokens == 0) return;
        require(q && out, "paged_attention: null pointer");
        const long long row = (long long)q_heads * p->dim;
        require((q_stride >= row && out_stride >= row) || b.tokens == 1, "paged_attention: a stride is shorter than a row");
        const int n = 16 / type_bytes(type);
        require(aligned(q, 16) && aligned(out, 16) && q_stride % n == 0 && out_stride % n == 0,
                "paged_attention: q and out rows must be 16-byte aligned");
        require((long long)b.tokens * q_heads < (1ll << 31) && b.tokens < (1 << 24),
                "paged_attention: too many tokens in one call");
        check_device(p, "paged_attention");
        gpt::PagedAttnArgs a{q, out, sinks, q_stride, out_stride, type, p->type, q_heads, window, scale, 0, 0x7fffffff};
        gpt::launch_paged_attention(p->maps, p->view(layer), b, a, p->attn_ws, static_cast<cudaStream_t>(stream));
    });
}

int gptoss_beam_select(const void* logits, int type, long long row_stride, const float* scores, const uint8_t* done,
                       int done_token, int batch, int beams, int vocab, int picks, float* out_scores, int32_t* rows,
                       int32_t* tokens, void* stream) {
    return abi_guard([&] {
        require(known_type(type), "beam_select: unknown type");
        require(batch >= 0 && beams >= 1 && beams <= 64 && picks >= 1 && picks <= 64,
                "beam_select: batch >= 0, beams and picks in 1 .. 64");
        require(vocab >= 1 && (long long)beams * vocab < (1ll << 31), "beam_select: beams * vocab must be 1 .. 2^31 - 1");
        require(batch <= (1 << 16), "beam_select: at most 65536 requests in one call");
        require(row_stride >= vocab || (long long)batch * beams <= 1, "beam_select: row_stride is shorter than a row");
        require(!done || (done_token >= 0 && done_token < vocab), "beam_select: done_token outside the vocabulary");
        if (batch == 0) return;
        require(logits && scores && out_scores && rows && tokens, "beam_select: null pointer");
        require(aligned(logits, type_bytes(type)), "beam_select: logits are not aligned to their type");
        gpt::BeamArgs a{logits, row_stride, scores, done, out_scores, rows, tokens, type, done_token, batch, beams,
                        vocab, picks};
        gpt::launch_beam_select(a, g_beam_ws.get(gpt::beam_ws_bytes(a)), static_cast<cudaStream_t>(stream));
    });
}

int gptoss_kv_fork(gptoss_kv_pool* p, const int32_t* refs, const int32_t* tables, const int32_t* lens, int seqs,
                   const int32_t* parents, const int32_t* extra, int children, int table_stride, int32_t* refs_out,
                   int32_t* tables_out, int32_t* lens_out, void* stream) {
    return abi_guard([&] {
        check_pool(p, "kv_fork");
        require(seqs >= 0 && children >= 0 && table_stride >= 0, "kv_fork: negative size");
        require(seqs <= (1 << 20) && children <= (1 << 20), "kv_fork: at most 2^20 sequences and children");
        require(refs && refs_out, "kv_fork: null reference counts");
        require(seqs == 0 || (lens && (tables || table_stride == 0)), "kv_fork: null tables or lengths");
        require(children == 0 || (parents && lens_out && (tables_out || table_stride == 0)), "kv_fork: null children");
        require(seqs == 0 || children == 0 || ((tables_out != tables || table_stride == 0) && lens_out != lens),
                "kv_fork: the children's tables and lengths need arrays of their own");
        check_device(p, "kv_fork");
        gpt::ForkArgs a{refs, tables, lens, parents, extra, refs_out, tables_out, lens_out, seqs, children,
            table_stride, gpt::most_positions(table_stride, p->pages.page_size)};
        gpt::launch_kv_fork(p->pages, a, p->page_ws, static_cast<cudaStream_t>(stream));
    });
}

int gptoss_kv_compact(gptoss_kv_pool* p, const int32_t* refs, const int32_t* tables, const int32_t* lens, int seqs,
                      int table_stride, int32_t* refs_out, int32_t* tables_out, int32_t* remap, int32_t* live,
                      void* stream) {
    return abi_guard([&] {
        check_pool(p, "kv_compact");
        require(seqs >= 0 && table_stride >= 0 && seqs <= (1 << 20), "kv_compact: seqs and table_stride out of range");
        require(refs && refs_out && remap && live, "kv_compact: null pointer");
        require(seqs == 0 || table_stride == 0 || (tables && lens && tables_out), "kv_compact: null tables or lengths");
        check_device(p, "kv_compact");
        gpt::CompactArgs a{refs, tables, lens, refs_out, tables_out, remap, live, seqs, table_stride,
            gpt::most_positions(table_stride, p->pages.page_size)};
        gpt::launch_kv_compact(p->pages, a, p->page_ws, static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
