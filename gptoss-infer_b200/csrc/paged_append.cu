// Rotary positions and the append to the paged cache in one pass.
//
// Token t of sequence b stands at p = len_b - new_b + (t - cu_b). Queries and keys are rotated in pairs (a, b) ->
// (a cos - b sin, b cos + a sin) with the table's row p; pairs are (j, j + rot/2) or, interleaved, (2j, 2j + 1); the
// dims from rot on pass through. All arithmetic is fp32; a value is rounded once, to the type it is stored in.
//
// Bound: bytes (each value read once and written once; nothing is reused but the token's cos/sin row, which the heads
// find in L1). A work item is two runs of eight values of one head with whole pairs in them.
#include <type_traits>

#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kThreads = 256;
constexpr int kTokens = 8;       // tokens per CTA, at most: one warp looks up each
// Items of a thread in flight: more of them cost more in resident threads than they bring (16383 bf16 tokens of 48
// heads of 128: 1 item 70 us, 2 75 us, 4 91 us).
constexpr int kBatch = 1;

struct Place {
    char *k, *v;                 // the token's cache rows (head 0), or null: not stored
    int pos;                     // row of the cos/sin table, or -1: token not in a sequence or out of range
};

__device__ __forceinline__ void turn(float& a, float& b, float cs, float sn) {
    const float p = a, r = b;
    a = p * cs - r * sn;
    b = r * cs + p * sn;
}
template <int RUN>
__device__ __forceinline__ void turn_pairs(float (&x)[RUN], const float* cs, const float* sn) {
    if constexpr (RUN == 8) {
        const float4 c4 = __ldg(reinterpret_cast<const float4*>(cs)), s4 = __ldg(reinterpret_cast<const float4*>(sn));
        turn(x[0], x[1], c4.x, s4.x);
        turn(x[2], x[3], c4.y, s4.y);
        turn(x[4], x[5], c4.z, s4.z);
        turn(x[6], x[7], c4.w, s4.w);
    }
}

// RUN values of a run as loaded, unpacked and stored: 8 (16 bytes of 16-bit values) or 4.
template <class T, int RUN, int Q>
__device__ __forceinline__ void load_run(const T* p, uint4 (&raw)[Q]) {
    if constexpr (RUN * sizeof(T) == 8) {
        const uint2 x = __ldg(reinterpret_cast<const uint2*>(p));
        raw[0].x = x.x;
        raw[0].y = x.y;
    } else {
#pragma unroll
        for (int e = 0; e < Q; ++e) raw[e] = __ldg(reinterpret_cast<const uint4*>(p) + e);
    }
}
template <class T, int RUN, int Q>
__device__ __forceinline__ void unpack_run(const uint4 (&raw)[Q], float (&x)[RUN]) {
    if constexpr (RUN == 8) {
        unpack8<T>(raw, x);
    } else {
        const uint4 both[2] = {raw[0], raw[0]};
        float y[8];
        if constexpr (sizeof(T) == 4) unpack8<T>(both, y);
        else unpack8<T>(raw, y);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = y[i];
    }
}
template <int RUN>
__device__ __forceinline__ void store_run(char* p, const float (&x)[RUN], int type) {
    if constexpr (RUN == 8) store8(p, x, type);
    else if (type == kF32) *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack2(x[0], x[1], type == kF16), pack2(x[2], x[3], type == kF16));
}

// RUN 8 or 4: runs of so many values are aligned to their loads and pairs lie in one run or in the two of an item (4: a
// rotated half that is a multiple of 4 only); RUN 1: one pair at a time.
template <class T, int RUN>
__global__ void __launch_bounds__(kThreads) kv_append_kernel(KvView c, KvBatch b, AppendArgs a, int per_cta,
    FastDiv per_token) {
    __shared__ Place place[kTokens];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int t0 = blockIdx.x * per_cta, nt = min(per_cta, b.tokens - t0);
    if (warp < nt) {
        const int t = t0 + warp, i = find_sequence(b.cu, b.seqs, t, lane);
        if (lane == 0) {
            Place w{nullptr, nullptr, -1};
            const Seq q = load_seq(b, i, c.err);
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
    const int per_head = RUN > 1 ? c.dim / (2 * RUN) : c.dim / 2, heads = a.q_heads + 2 * c.kv_heads;
    const int half = a.rot / 2, q_bytes = a.q_type == kF32 ? 4 : 2;
    const int items = heads * per_head;
    if constexpr (RUN > 1) {
        constexpr int Q = RUN * sizeof(T) > 16 ? 2 : 1;   // loads of a run
        // First dims of an item's two runs: the halves of the rotated dims in the half layout, and of what passes
        // behind them; the halves of the head otherwise. Neighbouring threads take neighbouring runs.
        const auto runs_of = [&](int j, bool is_v, int& d0, int& d1) {
            if (is_v || a.interleaved) {
                d0 = j * RUN;
                d1 = c.dim / 2 + j * RUN;
            } else if (j * 2 * RUN < a.rot) {
                d0 = j * RUN;
                d1 = half + j * RUN;
            } else {
                d0 = a.rot + (j - a.rot / (2 * RUN)) * RUN;
                d1 = d0 + (c.dim - a.rot) / 2;
            }
        };
        // kBatch items of a thread have their loads in flight before the first is worked on
        for (int i0 = threadIdx.x; i0 < nt * items; i0 += kBatch * kThreads) {
            uint4 raw[kBatch][2][Q];
            int what[kBatch];                         // token << 16 | head, or -1
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                const int i = i0 + n * kThreads;
                what[n] = -1;
                if (i >= nt * items) continue;
                const int u = int(per_token.div(i)), it = i - u * items, h = it / per_head, j = it % per_head;
                if (place[u].pos < 0) continue;
                const long long t = t0 + u;
                const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
                const T* src = is_q ? static_cast<const T*>(a.q) + t * a.q_stride + h * c.dim
                                    : static_cast<const T*>(is_v ? a.v : a.k) + t * a.kv_stride +
                                          (h - a.q_heads - (is_v ? c.kv_heads : 0)) * c.dim;
                int d0, d1;
                runs_of(j, is_v, d0, d1);
                load_run<T, RUN>(src + d0, raw[n][0]);
                load_run<T, RUN>(src + d1, raw[n][1]);
                what[n] = u << 16 | h;
            }
#pragma unroll
            for (int n = 0; n < kBatch; ++n) {
                if (what[n] < 0) continue;
                const int u = what[n] >> 16, h = what[n] & 0xffff, j = (i0 + n * kThreads) % per_head;
                const Place w = place[u];
                const bool is_q = h < a.q_heads, is_v = h >= a.q_heads + c.kv_heads;
                int d0, d1;
                runs_of(j, is_v, d0, d1);
                float x[RUN], y[RUN];
                unpack_run<T, RUN>(raw[n][0], x);
                unpack_run<T, RUN>(raw[n][1], y);
                const long long tab = (long long)w.pos * half;
                if (RUN == 8 && !is_v && a.interleaved) {   // each run: four pairs of its own
                    if (d0 < a.rot) turn_pairs<RUN>(x, a.cos_t + tab + d0 / 2, a.sin_t + tab + d0 / 2);
                    if (d1 < a.rot) turn_pairs<RUN>(y, a.cos_t + tab + d1 / 2, a.sin_t + tab + d1 / 2);
                } else if (!is_v && j * 2 * RUN < a.rot) {  // RUN pairs across the runs
                    const float4* ct = reinterpret_cast<const float4*>(a.cos_t + tab + d0);
                    const float4* st = reinterpret_cast<const float4*>(a.sin_t + tab + d0);
#pragma unroll
                    for (int e = 0; e < RUN / 4; ++e) {
                        const float4 c4 = __ldg(ct + e), s4 = __ldg(st + e);
                        turn(x[4 * e], y[4 * e], c4.x, s4.x);
                        turn(x[4 * e + 1], y[4 * e + 1], c4.y, s4.y);
                        turn(x[4 * e + 2], y[4 * e + 2], c4.z, s4.z);
                        turn(x[4 * e + 3], y[4 * e + 3], c4.w, s4.w);
                    }
                }
                if (is_q) {
                    char* qo = static_cast<char*>(a.q_out) + ((t0 + u) * (long long)a.q_heads + h) * c.dim * q_bytes;
                    store_run<RUN>(qo + d0 * q_bytes, x, a.q_type);
                    store_run<RUN>(qo + d1 * q_bytes, y, a.q_type);
                } else if (w.k) {
                    char* dst = (is_v ? w.v : w.k) + (h - a.q_heads - (is_v ? c.kv_heads : 0)) * c.head_stride;
                    store_run<RUN>(dst + d0 * 2, x, a.kv_type);
                    store_run<RUN>(dst + d1 * 2, y, a.kv_type);
                }
            }
        }
    } else {
        // blockDim is a multiple of per_head: a thread keeps its pair's number over the heads
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
    const bool even = al(a.q) && al(a.k) && al(a.v) && al(a.q_out) && al(a.cos_t) && al(a.sin_t) && a.rot % 8 == 0 &&
        a.q_stride % run == 0 && a.kv_stride % run == 0;
    const int per = b.tokens >= 148 * 8 * kTokens ? kTokens : 1;
    const int grid = (b.tokens + per - 1) / per, heads = a.q_heads + 2 * c.kv_heads;
    const auto div = [&](int n) { return FastDiv::of(uint32_t(heads * (c.dim / n))); };
    if (even && (a.interleaved || a.rot % 16 == 0))
        kv_append_kernel<T, 8><<<grid, kThreads, 0, s>>>(c, b, a, per, div(16));
    else if (even)
        kv_append_kernel<T, 4><<<grid, kThreads, 0, s>>>(c, b, a, per, div(8));
    else
        kv_append_kernel<T, 1><<<grid, kThreads, 0, s>>>(c, b, a, per, div(2));
    check_launch("kv_append");
}

}  // namespace

void launch_kv_append(const KvView& c, const KvBatch& b, const AppendArgs& a, cudaStream_t s) {
    if (a.in_type == kF32) launch<float>(c, b, a, s);
    else if (a.in_type == kF16) launch<__half>(c, b, a, s);
    else launch<__nv_bfloat16>(c, b, a, s);
}

}  // namespace gpt
