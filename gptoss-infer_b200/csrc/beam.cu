// Beam selection: the best `picks` of beams x vocab candidates of each request.
//
// score(r, v) = s_r + x_rv - lse_r with lse_r = log sum_v exp(x_rv), ranked by (score in fp64, lower flattened index
// r * vocab + v first); a NaN logit counts as -inf, and candidates of score -inf or NaN are never picked. A finished
// row's only candidate is done_token at the row's own score.
#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kThreads = 512;

struct Best {
    double score;
    int at;
};
__device__ __forceinline__ bool better(double s, int i, double t, int j) { return s > t || (s == t && i < j); }

template <class T>
__global__ void __launch_bounds__(kThreads) beam_select_kernel(BeamArgs a) {
    __shared__ double lse[64];
    __shared__ Best part[kThreads / 32];
    __shared__ Best last;
    const int req = blockIdx.x, warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const T* base = static_cast<const T*>(a.logits) + (long long)req * a.beams * a.row_stride;
    for (int r = warp; r < a.beams; r += kThreads / 32) {
        float m = -INFINITY, z = 0.f;
        for (int v = lane; v < a.vocab; v += 32) {
            float x = to_f32(base[r * a.row_stride + v]);
            if (!(x == x)) x = -INFINITY;
            if (x > m) {
                z = z * expf(m - x) + 1.f;
                m = x;
            } else if (x > -INFINITY) {
                z += expf(x - m);
            }
        }
        float mm = m;
        for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(kFull, mm, o));
        const double zz = warp_sum(m > -INFINITY ? double(z) * exp(double(m) - mm) : 0.0);
        if (lane == 0) lse[r] = double(mm) + log(zz);
    }
    if (threadIdx.x == 0) last = {INFINITY, -1};
    __syncthreads();
    const int total = a.beams * a.vocab;
    for (int pick = 0; pick < a.picks; ++pick) {
        Best b{-INFINITY, 0x7fffffff};
        const Best prev = last;
        for (int i = threadIdx.x; i < total; i += kThreads) {
            const int r = i / a.vocab, v = i - r * a.vocab;
            double sc = a.scores[req * a.beams + r];
            if (a.done && a.done[req * a.beams + r]) {
                if (v != a.done_token) continue;
            } else {
                const float x = to_f32(base[r * a.row_stride + v]);
                sc = sc + (double(x) - lse[r]);
            }
            if (!(sc > -INFINITY)) continue;
            if (better(prev.score, prev.at, sc, i) && better(sc, i, b.score, b.at)) b = {sc, i};
        }
        for (int o = 16; o; o >>= 1) {
            const double s = __shfl_xor_sync(kFull, b.score, o);
            const int j = __shfl_xor_sync(kFull, b.at, o);
            if (better(s, j, b.score, b.at)) b = {s, j};
        }
        if (lane == 0) part[warp] = b;
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int w = 1; w < kThreads / 32; ++w)
                if (better(part[w].score, part[w].at, b.score, b.at)) b = part[w];
            const bool none = b.at == 0x7fffffff;
            const int o = req * a.picks + pick;
            a.out_scores[o] = none ? -INFINITY : float(b.score);
            a.rows[o] = none ? -1 : req * a.beams + b.at / a.vocab;
            a.tokens[o] = none ? -1 : b.at % a.vocab;
            last = b;
        }
        __syncthreads();
    }
}

}  // namespace

size_t beam_ws_bytes(const BeamArgs&) { return 16; }

void launch_beam_select(const BeamArgs& a, void*, cudaStream_t s) {
    if (a.type == kF32) beam_select_kernel<float><<<a.batch, kThreads, 0, s>>>(a);
    else if (a.type == kF16) beam_select_kernel<__half><<<a.batch, kThreads, 0, s>>>(a);
    else beam_select_kernel<__nv_bfloat16><<<a.batch, kThreads, 0, s>>>(a);
    check_launch("beam_select");
}

}  // namespace gpt
