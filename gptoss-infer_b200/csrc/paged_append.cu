// Rotary positions and the append to the paged cache in one pass.
//
// Token t of sequence b stands at p = len_b - new_b + (t - cu_b). Queries and keys are rotated in pairs (a, b) ->
// (a cos - b sin, b cos + a sin) with the table's row p; pairs are (j, j + rot/2) or, interleaved, (2j, 2j + 1); the
// dims from rot on pass through. All arithmetic is fp32; a value is rounded once, to the type it is stored in.
//
// Bound: bytes (each value read once and written once; nothing is reused but the token's cos/sin row, which stays in
// registers). A work item is 16 values of one head: 8 pairs, so both halves of a pair are in one thread.
#include <type_traits>

#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kThreads = 256;
constexpr int kTokens = 8;       // tokens per CTA, at most: one warp looks up each

struct Place {
    char *k, *v;                 // the token's cache rows (head 0), or null: not stored
    int pos;                     // row of the cos/sin table, or -1: token not in a sequence or out of range
};

// VEC: every run of eight values is 16-byte aligned in memory and pairs do not straddle a run.
template <class T, bool VEC>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvView c, KvBatch b, AppendArgs a, int per_cta) {
    __shared__ Place place[kTokens];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int t0 = blockIdx.x * per_cta, nt = min(per_cta, b.tokens - t0);
    if (warp < nt) {
        const int t = t0 + warp, i = find_sequence(b.cu, b.seqs, t, lane);
        if (lane == 0) {
            Place w{nullptr, nullptr, -1};
            const Seq q = load_seq(b, c.page, i, c.err);
            if (t >= q.row0 && t < q.row0 + q.n) {
                const int pos = q.len - q.n + (t - q.row0);
                if (pos < 0 || (a.rot > 0 && pos >= a.positions)) {
                    report(c.err, kKvBadPosition);
                } else {
                    w.pos = pos;
                    const uint32_t pg = c.page.div(pos);
                    const int id = b.tables[(long long)i * b.table_stride + pg];
                    if (unsigned(id) < unsigned(c.num_pages)) {
                        const long long off = id * c.page_stride + (pos - int(pg * c.page.d)) * c.token_stride;
                        w.k = c.k + off;
                        w.v = c.v + off;
                    } else {
                        report(c.err, kKvBadPage);
                    }
                }
            }
            place[warp] = w;
        }
    }
    __syncthreads();
    const int per_head = VEC ? c.dim / 16 : c.dim / 2, heads = a.q_heads + 2 * c.kv_heads;
    const int half = a.rot / 2, q_bytes = a.q_type == kF32 ? 4 : 2;
    const int items = heads * per_head;
    // blockDim is a multiple of per_head: a thread keeps its dims over the heads, and its cos/sin values per token
    const int j = threadIdx.x % per_head;
    for (int u = 0; u < nt; ++u) {
        const Place w = place[u];
        if (w.pos < 0) continue;
        const long long t = t0 + u;
        const T* q = static_cast<const T*>(a.q) + t * a.q_stride;
        const T* k = static_cast<const T*>(a.k) + t * a.kv_stride;
        const T* v = static_cast<const T*>(a.v) + t * a.kv_stride;
        char* qo = static_cast<char*>(a.q_out) + t * a.q_heads * c.dim * q_bytes;
        const long long tab = (long long)w.pos * half;
        if constexpr (VEC) {
            const bool turned = j * 16 < a.rot;
            float cs[8], sn[8];
            if (turned) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    cs[i] = __ldg(a.cos_t + tab + j * 8 + i);
                    sn[i] = __ldg(a.sin_t + tab + j * 8 + i);
                }
            }
            for (int it = threadIdx.x; it < items; it += kThreads) {
                const int h = it / per_head;
                const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
                const int hk = is_q ? 0 : is_v ? h - a.q_heads - c.kv_heads : h - a.q_heads;
                const T* src = is_q ? q + h * c.dim : (is_v ? v : k) + hk * c.dim;
                const bool rot = turned && !is_v;
                // first and second run of eight
                const int d0 = rot && !a.interleaved ? j * 8 : j * 16;
                const int d1 = rot && !a.interleaved ? half + j * 8 : j * 16 + 8;
                float x[8], y[8];
                load8(src + d0, x);
                load8(src + d1, y);
                if (rot) {
                    if (a.interleaved) {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const float p = x[2 * i], r = x[2 * i + 1], s = y[2 * i], z = y[2 * i + 1];
                            x[2 * i] = p * cs[i] - r * sn[i];
                            x[2 * i + 1] = r * cs[i] + p * sn[i];
                            y[2 * i] = s * cs[4 + i] - z * sn[4 + i];
                            y[2 * i + 1] = z * cs[4 + i] + s * sn[4 + i];
                        }
                    } else {
#pragma unroll
                        for (int i = 0; i < 8; ++i) {
                            const float p = x[i], r = y[i];
                            x[i] = p * cs[i] - r * sn[i];
                            y[i] = r * cs[i] + p * sn[i];
                        }
                    }
                }
                if (is_q) {
                    store8(qo + (long long)(h * c.dim + d0) * q_bytes, x, a.q_type);
                    store8(qo + (long long)(h * c.dim + d1) * q_bytes, y, a.q_type);
                } else if (w.k) {
                    char* dst = (is_v ? w.v : w.k) + hk * c.head_stride;
                    store8(dst + d0 * 2, x, a.kv_type);
                    store8(dst + d1 * 2, y, a.kv_type);
                }
            }
        } else {
            const bool turned = j < half;
            const float cs = turned ? __ldg(a.cos_t + tab + j) : 1.f, sn = turned ? __ldg(a.sin_t + tab + j) : 0.f;
            for (int it = threadIdx.x; it < items; it += kThreads) {
                const int h = it / per_head;
                const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
                const int hk = is_q ? 0 : is_v ? h - a.q_heads - c.kv_heads : h - a.q_heads;
                const T* src = is_q ? q + h * c.dim : (is_v ? v : k) + hk * c.dim;
                const bool rot = turned && !is_v, apart = rot && !a.interleaved;
                const int d0 = apart ? j : 2 * j, d1 = apart ? half + j : 2 * j + 1;
                float x = to_f32(src[d0]), y = to_f32(src[d1]);
                if (rot) {
                    const float p = x, r = y;
                    x = p * cs - r * sn;
                    y = r * cs + p * sn;
                }
                if (is_q) {
                    store_as(qo, h * c.dim + d0, x, a.q_type);
                    store_as(qo, h * c.dim + d1, y, a.q_type);
                } else if (w.k) {
                    char* dst = (is_v ? w.v : w.k) + hk * c.head_stride;
                    store_as(dst, d0, x, a.kv_type);
                    store_as(dst, d1, y, a.kv_type);
                }
            }
        }
    }
}

template <class T>
void launch(const KvView& c, const KvBatch& b, const AppendArgs& a, cudaStream_t s) {
    const auto al = [](const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; };
    const int run = 16 / int(sizeof(T));
    const bool vec = al(a.q) && al(a.k) && al(a.v) && al(a.q_out) && a.q_stride % run == 0 && a.kv_stride % run == 0 &&
                     a.rot % 16 == 0;
    const int per = b.tokens >= 148 * 8 * kTokens ? kTokens : 1;
    const int grid = (b.tokens + per - 1) / per;
    if (vec) kv_append_kernel<T, true><<<grid, kThreads, 0, s>>>(c, b, a, per);
    else kv_append_kernel<T, false><<<grid, kThreads, 0, s>>>(c, b, a, per);
    check_launch("kv_append");
}

}  // namespace

void launch_kv_append(const KvView& c, const KvBatch& b, const AppendArgs& a, cudaStream_t s) {
    if (a.in_type == kF32) launch<float>(c, b, a, s);
    else if (a.in_type == kF16) launch<__half>(c, b, a, s);
    else launch<__nv_bfloat16>(c, b, a, s);
}

}  // namespace gpt
