// The paged key/value cache and its operators: what the kernels see of a pool and of a batch of sequences, and the
// host launchers. Every launcher throws std::runtime_error on a launch failure; the C ABI (paged_capi.cu) checks the
// arguments first and turns exceptions into -1.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>

namespace gpt {

enum KvType : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

// Codes of a pool's device-side error word (gptoss_kv_pool_status).
enum KvError : int {
    kKvBadPage = 300,        // a table names a page outside the pool
    kKvBadLength = 301,      // a cache length is negative, longer than its table or near 2^31
    kKvBadBatch = 302,       // cu_tokens runs backwards or past the batch's tokens
    kKvBadPosition = 303,    // a new token's position is negative or past the cos/sin table
    kKvOutOfPages = 304,     // gptoss_kv_fork found fewer free pages than it needs
    kKvBadParent = 305,      // a parent outside the given sequences
    kKvTooMuch = 306,        // new tokens times cached positions past what one call of the attention counts
    kKvWait = 310            // a bounded wait inside a kernel gave up (310 .. 319)
};

// n / d for 0 <= n < 2^31 by a multiplication: m = floor(2^(31+s) / d) + 1 with 2^(s-1) < d <= 2^s, so the error
// e = m d - 2^(31+s) is at most d <= 2^s and n e < 2^(31+s) keeps the quotient exact.
struct FastDiv {
    uint32_t m, s, d;
    static FastDiv of(uint32_t d) {
        uint32_t s = 0;
        while ((1ull << s) < d) ++s;
        return {static_cast<uint32_t>((1ull << (31 + s)) / d + 1), 31 + s, d};
    }
    __host__ __device__ __forceinline__ uint32_t div(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<unsigned long long>(n) * m) >> s);
    }
};

// One layer of a pool. Strides in bytes; a row (one token's head) is contiguous.
struct KvView {
    char *k, *v;
    long long page_stride, token_stride, head_stride;
    int num_pages, kv_heads, dim;
    FastDiv page;            // division by the page size
    int* err;
    int layer, box_log;      // coordinates of KvMaps: the layer, 2^box_log slots per box (below 3: no maps)
};

// Tensor maps of a pool, [layer][page][slot][head][dim] in boxes of 2^box_log slots x 64 dims with the 128-byte
// swizzle.
struct KvMaps {
    CUtensorMap k, v;
};

// The longest cache length of a table: its pages, and no more than positions a few tiles further on can be counted to in
// 32 bits.
inline int most_positions(int table_stride, int page_size) {
    const long long n = static_cast<long long>(table_stride) * page_size;
    return n < 0x7fffffff - 4095 ? static_cast<int>(n) : 0x7fffffff - 4095;
}

// Sequence b's new tokens are rows cu[b] .. cu[b + 1) of the batch; its cache holds lens[b] positions with them.
struct KvBatch {
    const int* cu;
    const int* lens;
    const int* tables;
    int seqs, tokens, table_stride, max_new;
    int most;                    // longest length of a table (most_positions)
};

struct AppendArgs {
    const void *q, *k, *v;
    long long q_stride, kv_stride;           // elements between tokens
    const float *cos_t, *sin_t;              // [positions][rot / 2]
    void* q_out;                             // [tokens][q_heads][dim]
    int in_type, q_type, kv_type, q_heads, positions, rot, interleaved;
};
void launch_kv_append(const KvView& c, const KvBatch& b, const AppendArgs& a, cudaStream_t s);

struct PagedAttnArgs {
    const void* q;
    void* out;
    const float* sinks;                      // per query head, or null
    long long q_stride, out_stride;          // elements between tokens
    int type, kv_type, q_heads, window;
    float scale;
    int rows_from, rows_to;                  // sequences with so many query rows per key/value head; others are left out
    bool check;                              // set by the launchers (many_groups in paged_schedule.cuh)
};
// Workspace of launch_paged_attention: counters and partial results; zeroed once, the kernels leave the counters at 0.
// The two kernels share it (their counters are the same words).
constexpr size_t kCounterBytes = 2048;            // of both kernels, before the partial results
size_t paged_attention_ws_bytes(int dim);
size_t paged_tiles_ws_bytes(int dim);
void launch_paged_tiles(const KvMaps& m, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws,
    cudaStream_t s);
void launch_paged_attention(const KvMaps& m, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws,
    cudaStream_t s);

struct BeamArgs {
    const void* logits;
    long long row_stride;
    const float* scores;
    const uint8_t* done;                     // or null
    float* out_scores;
    int *rows, *tokens;
    int type, done_token, batch, beams, vocab, picks;
};
// Workspace: a counter per request in the first kBeamCounters bytes (zeroed once, left at 0), then the parts' results.
constexpr size_t kBeamCounters = 1 << 18;
size_t beam_ws_bytes(const BeamArgs& a);
void launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t s);

struct ForkArgs {
    const int *refs, *tables, *lens, *parents, *extra;
    int *refs_out, *tables_out, *lens_out;
    int seqs, children, stride;
    int most;                                // longest length of a table (most_positions)
};
struct CompactArgs {
    const int *refs, *tables, *lens;
    int *refs_out, *tables_out, *remap, *live;
    int seqs, stride;
    int most;
};
// All layers of a pool, for copies of whole pages. Strides in bytes.
struct KvPages {
    char *k, *v;
    long long layer_stride, page_stride, token_stride, head_stride;
    int layers, num_pages, page_size, kv_heads, row_bytes;
    int* err;
};
// Workspace of both: zeroed memory, laid out and prepared once by make_kv_pages_ws (on the legacy default stream). The
// kernels leave it as they found it. Every move has a destination page of its own, so the pages bound the moves.
struct PageWs {
    int* barrier;                  // arrivals, left at 0, and the number of the last barrier passed
    int* count;                    // [0] moves
    int* delta;                    // [num_pages] change of the counts; left at 0
    int* free_page;                // [num_pages]
    int* first;                    // [num_pages] first child whose part-filled last page it is; left at the largest int
    int2* moves;                   // [num_pages] (source, destination)
};
size_t kv_pages_ws_bytes(int num_pages);
PageWs make_kv_pages_ws(void* ws, int num_pages);
void launch_kv_fork(const KvPages& p, const ForkArgs& a, const PageWs& w, cudaStream_t s);
void launch_kv_compact(const KvPages& p, const CompactArgs& a, const PageWs& w, cudaStream_t s);

}  // namespace gpt
