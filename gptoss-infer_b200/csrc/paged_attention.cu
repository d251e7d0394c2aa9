// Attention of new tokens over the paged cache, one warp per (token, query head).
//
// out = sum_j w_j v_j / (sum_j w_j [+ exp(sink)]), w_j = exp(scale q.k_j), j over the positions max(0, p - window + 1)
// .. p of the token at p; one pass with the running maximum and sum in fp32.
#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

template <class T, class C, int D>
__global__ void __launch_bounds__(128) paged_attention_simple_kernel(KvView c, KvBatch b, PagedAttnArgs a) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x % 32;
    const long long item = (long long)blockIdx.x * 4 + threadIdx.x / 32;
    if (item >= (long long)b.tokens * a.q_heads) return;
    const int t = int(item / a.q_heads), h = int(item % a.q_heads), kh = h / (a.q_heads / c.kv_heads);
    const int i = find_sequence(b.cu, b.seqs, t, lane);
    const Seq s = load_seq(b, c.page, i, c.err);
    if (t < s.row0 || t >= s.row0 + s.n) return;
    const int p = s.len - s.n + (t - s.row0);
    const int lo = a.window ? max(0, p - a.window + 1) : 0;
    float q[E], o[E] = {};
    for (int e = 0; e < E; ++e)
        q[e] = to_f32(static_cast<const T*>(a.q)[t * a.q_stride + h * D + lane * E + e]) * a.scale;
    float m = -INFINITY, z = 0.f;
    if (a.sinks) {
        m = a.sinks[h];
        z = m > -INFINITY ? 1.f : 0.f;
    }
    for (int j = lo; j <= p; ++j) {
        const int pg = c.page.div(j);
        const int id = safe_page(b.tables[(long long)i * b.table_stride + pg], c);
        const long long off = id * c.page_stride + (j - pg * int(c.page.d)) * c.token_stride + kh * c.head_stride;
        const C* k = reinterpret_cast<const C*>(c.k + off) + lane * E;
        const C* v = reinterpret_cast<const C*>(c.v + off) + lane * E;
        float x = 0.f;
        for (int e = 0; e < E; ++e) x += q[e] * to_f32(k[e]);
        x = warp_sum(x);
        const float mm = fmaxf(m, x), f = mm == -INFINITY ? 1.f : __expf(m - mm), w = x == -INFINITY ? 0.f : expf(x - mm);
        z = z * f + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * to_f32(v[e]);
        m = mm;
    }
    for (int e = 0; e < E; ++e)
        store_as(a.out, t * a.out_stride + h * D + lane * E + e, z > 0.f ? o[e] / z : 0.f, a.type);
}

template <class T, class C>
void launch(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, cudaStream_t s) {
    const int grid = int(((long long)b.tokens * a.q_heads + 3) / 4);
    if (c.dim == 64) paged_attention_simple_kernel<T, C, 64><<<grid, 128, 0, s>>>(c, b, a);
    else paged_attention_simple_kernel<T, C, 128><<<grid, 128, 0, s>>>(c, b, a);
    check_launch("paged_attention");
}

}  // namespace

size_t paged_attention_ws_bytes() { return 16; }

void launch_paged_attention(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void*, cudaStream_t s) {
    if (a.type == kF32) launch<float, __half>(c, b, a, s);
    else if (a.type == kF16) launch<__half, __half>(c, b, a, s);
    else launch<__nv_bfloat16, __nv_bfloat16>(c, b, a, s);
}

}  // namespace gpt
