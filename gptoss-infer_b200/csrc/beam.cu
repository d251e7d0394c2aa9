// Beam selection: the best `picks` of beams x vocab candidates of each request.
//
// score(r, v) = s_r + x_rv - lse_r with lse_r = log sum_v exp(x_rv), ranked by (score in fp64, lower flattened index
// r * vocab + v first); a NaN logit counts as -inf, and candidates of score -inf or NaN are never picked. A finished
// row's only candidate is done_token at the row's own score.
//
// Bound: the logits' bytes, read once. A CTA takes up to 16384 logits of one row into registers (16-byte loads, 32 per
// thread, a thread's values 8 or 4 at a time), leaves their maximum and sum of exponentials, and its own best `picks`:
// within a row the score orders as the logit does, so no sum is needed to choose them. A threshold comes from the
// threads' own best values: the least over the 16 warps of the warp's j-th largest, 16 j >= picks, so at least `picks`
// values reach it (about three times as many do when the values are in no particular order: 54 for 16 picks). Those go
// on a list and are ranked exactly. Where they overflow it (sorted or constant rows), the exact picks-th largest of the
// threads' best is taken instead: only the `picks` threads whose best reaches it can hold values that do, at most
// picks x 32. Keys (value, then lower index first) are 64-bit words without ties. The last CTA of a request puts the
// rows' sums together in the order of their parts and ranks the parts' picks in the same way, with scores in fp64: the
// result does not depend on timing.
#include <algorithm>
#include <type_traits>

#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kThreads = 512, kPer = 32, kPart = kThreads * kPer, kWarps = kThreads / 32, kMostPicks = 64;
constexpr int kList = kMostPicks * kPer;

// fp32 bits in an order that compares as unsigned: the larger float is the larger word, both zeros are the same one (the
// sum makes -0 into +0); NaN is not passed in.
__device__ __forceinline__ uint32_t ordered(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float unordered(uint32_t o) {
    return __uint_as_float(o & 0x80000000u ? o & 0x7fffffffu : ~o);
}

template <class T>
__device__ __forceinline__ T from_f32(float x) {
    if constexpr (std::is_same<T, float>::value) return x;
    else if constexpr (std::is_same<T, __half>::value) return __float2half_rn(x);
    else return __float2bfloat16_rn(x);
}

struct Found {               // a part's result: its maximum, sum of exp(x - maximum), and keys in descending order
    float top, sum;
};

// The k-th largest (k from 1) of the block's keys, one per thread, none of them twice except 0 ("nothing"): each warp
// sorts its own, then every key finds its rank. Returns 0 when fewer than k exist.
__device__ __forceinline__ unsigned long long kth_largest(unsigned long long key, int k, unsigned long long* sorted,
                                                          unsigned long long* out) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    // bitonic sort of the warp's 32 keys, descending
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int step = size >> 1; step; step >>= 1) {
            const unsigned long long other = __shfl_xor_sync(kFull, key, step);
            const bool down = (lane & size) == 0, lower = (lane & step) == 0;
            key = (down == lower) == (key > other) ? key : other;
        }
    sorted[warp * 32 + lane] = key;
    if (threadIdx.x == 0) *out = 0;
    __syncthreads();
    // how many keys are larger: in its own warp's order, and by binary search in the other warps'
    if (key) {
        int larger = lane;
#pragma unroll 4
        for (int w = 0; w < kWarps; ++w) {
            if (w == warp) continue;
            int at = 0;
#pragma unroll
            for (int step = 16; step; step >>= 1)
                if (sorted[w * 32 + at + step - 1] > key) at += step;
            larger += at + (sorted[w * 32 + at] > key);
        }
        if (larger == k - 1) *out = key;
    }
    __syncthreads();
    const unsigned long long found = *out;
    __syncthreads();                                  // `sorted` and `out` may be written again
    return found;
}

// Lists of keys by rank: eight lanes count the larger ones for each. f(rank, place in the list).
template <class G, class F>
__device__ __forceinline__ void by_rank(int m, G&& larger_than, F&& f) {
    const int lane8 = threadIdx.x % 8;
    for (int i0 = 0; i0 < m; i0 += kThreads / 8) {    // uniform over the warp: all lanes take part in the sum
        const int i = i0 + threadIdx.x / 8;
        int larger = 0;
        if (i < m)
            for (int j = lane8; j < m; j += 8) larger += larger_than(j, i);
#pragma unroll
        for (int o = 4; o; o >>= 1) larger += __shfl_xor_sync(kFull, larger, o);
        if (i < m && lane8 == 0) f(larger, i);
    }
}

// A warp's j-th largest word (0: fewer than j are not 0), equal ones counted apart.
__device__ __forceinline__ uint32_t warp_jth(uint32_t u, int j) {
    uint32_t w = 0;
    for (int i = 0; i < j; ++i) {
        w = __reduce_max_sync(kFull, u);
        if (w == 0) break;
        if (int(threadIdx.x % 32) == __ffs(__ballot_sync(kFull, u == w)) - 1) u = 0;
    }
    return w;
}

template <class T>
__global__ void __launch_bounds__(kThreads, sizeof(T) == 4 ? 2 : 3)
beam_select_kernel(BeamArgs a, int parts, int size, int* counters, Found* found, unsigned long long* keys) {
    __shared__ unsigned long long list[kList];
    __shared__ unsigned long long threshold;
    __shared__ int flat_list[kList];                  // of the request's candidates: row of the request * vocab + token
    __shared__ float red[2 * kWarps];
    __shared__ uint32_t low[kWarps];
    __shared__ double lse[64];
    __shared__ int count, last;
    unsigned long long* sorted = list;                // the threshold is found before the list is filled
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int row = blockIdx.x / parts, part = blockIdx.x % parts, req = row / a.beams;
    const bool done = a.done && a.done[row];
    const int v0 = part * size, n = max(0, min(size, a.vocab - v0));
    if (threadIdx.x == 0) count = 0;
    if (!done) {
        // --- the part's values, in registers as they are stored (16-bit ones in half the registers: three CTAs share
        // an SM), -inf past the end
        constexpr int W = 16 / int(sizeof(T));        // values of a 16-byte load
        const T* src = static_cast<const T*>(a.logits) + (long long)row * a.row_stride + v0;
        const auto index = [&](int i) { return (i / W * kThreads + int(threadIdx.x)) * W + i % W; };
        union {
            uint4 quad[kPer / W];
            T value[kPer];
        } raw;
        if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
#pragma unroll
            for (int i = 0; i < kPer / W; ++i)
                if (index(i * W) + W <= n) raw.quad[i] = __ldcs(reinterpret_cast<const uint4*>(src + index(i * W)));
#pragma unroll
            for (int i = 0; i < kPer / W; ++i)
                if (index(i * W) + W > n) {
#pragma unroll
                    for (int e = 0; e < W; ++e)
                        raw.value[i * W + e] = index(i * W) + e < n ? src[index(i * W) + e] : from_f32<T>(-INFINITY);
                }
        } else {
#pragma unroll
            for (int i = 0; i < kPer; ++i) raw.value[i] = index(i) < n ? src[index(i)] : from_f32<T>(-INFINITY);
        }
        const auto x = [&](int i) { return fmaxf(to_f32(raw.value[i]), -INFINITY); };   // NaN counts as -inf
        // --- maximum, threshold, sum
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < kPer; i += 2) top = fmaxf(fmaxf(top, x(i)), x(i + 1));
        const auto key_of = [&](float value, int i) {
            return value == -INFINITY ? 0ull
                                      : (unsigned long long)ordered(value) << 32 | (0xffffffffu - uint32_t(v0 +
                                          index(i)));
        };
        float all = top;
#pragma unroll
        for (int o = 16; o; o >>= 1) all = fmaxf(all, __shfl_xor_sync(kFull, all, o));
        const int holders = min(kWarps, (n + 32 * W - 1) / (32 * W));       // warps that have values
        const uint32_t word = top == -INFINITY ? 0u : ordered(top);
        const uint32_t jth = warp < holders ? warp_jth(word, (a.picks + holders - 1) / holders) : 0xffffffffu;
        if (lane == 0) {
            red[warp] = all;
            low[warp] = jth;
        }
        __syncthreads();
        uint32_t reach = low[0];
#pragma unroll
        for (int w = 0; w < kWarps; ++w) {
            all = fmaxf(all, red[w]);
            reach = min(reach, low[w]);
        }
        // --- values that reach the threshold (read again: a register cannot be picked by number)
        const auto collect = [&](unsigned long long least) {
            if (word && word >= uint32_t(least >> 32)) {
                const float floor_value = least == 0 ? -INFINITY : unordered(uint32_t(least >> 32));
                uint32_t hits = 0;
#pragma unroll
                for (int i = 0; i < kPer; ++i) hits |= uint32_t(x(i) >= floor_value) << i;
                for (; hits; hits &= hits - 1) {
                    const int i = __ffs(hits) - 1, at = index(i);
                    if (at >= n) continue;
                    const unsigned long long k = key_of(fmaxf(to_f32(src[at]), -INFINITY), i);
                    if (k && k >= least) {
                        const int to = atomicAdd(&count, 1);
                        if (to < kList) list[to] = k;
                    }
                }
            }
        };
        collect((unsigned long long)reach << 32);
        const float base = all == -INFINITY || all == INFINITY ? 0.f : all;
        float sum4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < kPer; ++i) sum4[i & 3] += __expf(x(i) - base);
        const float sum = warp_sum((sum4[0] + sum4[1]) + (sum4[2] + sum4[3]));
        if (lane == 0) red[kWarps + warp] = sum;
        __syncthreads();
        if (threadIdx.x == 0) {
            float z = 0.f;
            for (int w = 0; w < kWarps; ++w) z += red[kWarps + w];
            found[blockIdx.x] = {all, z};
        }
        int m = count;
        if (m > kList) {
            int best = 0;                             // the first of the thread's largest values
#pragma unroll
            for (int i = kPer - 1; i >= 0; --i)
                if (x(i) == top) best = i;
            const unsigned long long least = kth_largest(key_of(top, best), a.picks, sorted, &threshold);
            if (threadIdx.x == 0) count = 0;
            __syncthreads();
            collect(least);
            __syncthreads();
            m = count;
        }
        // rank of each listed key: how many are larger (keys differ from one another)
        by_rank(m, [&](int j, int i) { return list[j] > list[i]; }, [&](int rank, int i) {
            if (rank < a.picks) keys[(long long)blockIdx.x * a.picks + rank] = list[i];
        });
        for (int i = m + threadIdx.x; i < a.picks; i += kThreads) keys[(long long)blockIdx.x * a.picks + i] = 0;
    } else {
        if (threadIdx.x == 0) found[blockIdx.x] = {0.f, 1.f};
        for (int i = threadIdx.x; i < a.picks; i += kThreads)
            keys[(long long)blockIdx.x * a.picks + i] =
                part == 0 && i == 0 ? (unsigned long long)ordered(0.f) << 32 | (0xffffffffu - uint32_t(a.done_token)) : 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        const int c = arrive(&counters[req]);
        last = c == a.beams * parts - 1;
        if (last) counters[req] = 0;
    }
    __syncthreads();
    if (!last) return;

    // --- the request: log-sum-exp of its rows, then the best of all parts' picks
    const int first = req * a.beams * parts;
    for (int r = warp; r < a.beams; r += kWarps) {
        const Found* f = found + first + r * parts;
        float top = -INFINITY;
        for (int p = lane; p < parts; p += 32) top = fmaxf(top, __ldcg(&f[p].top));
#pragma unroll
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
        double sum = 0.0;
        for (int p = lane; p < parts; p += 32) {
            const float t = __ldcg(&f[p].top);
            if (t > -INFINITY) sum += double(__ldcg(&f[p].sum)) * (t == INFINITY ? 1.0 : exp(double(t) - double(top)));
        }
        sum = warp_sum(sum);
        // a finished row's candidate has the key of 0: its score is the row's own
        if (lane == 0) lse[r] = a.done && a.done[req * a.beams + r] ? 0.0 : double(top) + log(sum);
    }
    if (threadIdx.x == 0) count = 0;
    __syncthreads();
    const int total = a.beams * parts * a.picks;
    const unsigned long long* mine = keys + (long long)first * a.picks;
    // score of a candidate, and its order word: fp64 in an order that compares as unsigned, 0: none
    const auto score_of = [&](int i, unsigned long long k, int& flat) {
        const int r = i / (parts * a.picks);
        flat = r * a.vocab + int(0xffffffffu - uint32_t(k));
        return double(a.scores[req * a.beams + r]) + (double(unordered(uint32_t(k >> 32))) - lse[r]);
    };
    const auto order_of = [&](int i, unsigned long long k) {
        int flat;
        if (k == 0) return 0ull;
        const double s = score_of(i, k, flat);
        if (!(s > -INFINITY)) return 0ull;
        const unsigned long long b = __double_as_longlong(s + 0.0);
        return b & 0x8000000000000000ull ? ~b : b | 0x8000000000000000ull;
    };
    // The threshold is the picks-th largest of the threads' best words, made different from one another by the thread's
    // number in the 9 lowest bits (which only lowers it). If the list does not hold what reaches it (equal scores by
    // the hundred), the candidates are ranked where they lie.
    unsigned long long best = 0;
    for (int i = threadIdx.x; i < total; i += kThreads) best = max(best, order_of(i, __ldcg(mine + i)));
    const unsigned long long least = kth_largest(best ? (best & ~511ull) | threadIdx.x : 0, a.picks, sorted,
        &threshold) & ~511ull;
    const auto collect = [&](unsigned long long least) {
        if (best && best >= least)
            for (int i = threadIdx.x; i < total; i += kThreads) {
                const unsigned long long k = __ldcg(mine + i), o = order_of(i, k);
                if (o && o >= least) {
                    const int to = atomicAdd(&count, 1);
                    if (to < kList) {
                        list[to] = o;
                        score_of(i, k, flat_list[to]);
                    }
                }
            }
    };
    collect(least);
    __syncthreads();
    const int m = count;
    const int out = req * a.picks;
    const auto put = [&](int at, double score, int flat) {
        a.out_scores[out + at] = float(score);
        a.rows[out + at] = req * a.beams + flat / a.vocab;
        a.tokens[out + at] = flat % a.vocab;
    };
    if (m <= kList) {
        by_rank(m, [&](int j, int i) { return list[j] > list[i] || (list[j] == list[i] &&
            flat_list[j] < flat_list[i]); },
                [&](int rank, int i) {
                    const unsigned long long o = list[i];
                    if (rank < a.picks)
                        put(rank, __longlong_as_double(o & 0x8000000000000000ull ? o & 0x7fffffffffffffffull : ~o),
                            flat_list[i]);
                });
    } else {
        for (int i = warp; i < total; i += kWarps) {
            const unsigned long long ki = __ldcg(mine + i), oi = order_of(i, ki);
            if (!oi || oi < least) continue;
            int fi;
            const double si = score_of(i, ki, fi);
            int larger = 0;
            for (int j = lane; j < total; j += 32) {
                const unsigned long long kj = __ldcg(mine + j), oj = order_of(j, kj);
                if (!oj || oj < oi) continue;
                int fj;
                score_of(j, kj, fj);
                larger += oj > oi || fj < fi;
            }
            larger = __reduce_add_sync(kFull, larger);
            if (lane == 0 && larger < a.picks) put(larger, si, fi);
        }
    }
    for (int i = min(m, a.picks) + threadIdx.x; i < a.picks; i += kThreads) {
        a.out_scores[out + i] = -INFINITY;
        a.rows[out + i] = a.tokens[out + i] = -1;
    }
}

int parts_of(const BeamArgs& a) { return (a.vocab + kPart - 1) / kPart; }
size_t counter_bytes(const BeamArgs& a) { return (size_t(a.batch) * sizeof(int) + 255) / 256 * 256; }
size_t found_bytes(const BeamArgs& a) {
    return (size_t(a.batch) * a.beams * parts_of(a) * sizeof(Found) + 255) / 256 * 256;
}

template <class T>
void launch(const BeamArgs& a, void* ws, cudaStream_t s) {
    char* p = static_cast<char*>(ws);
    // equal parts, of whole 64-byte runs
    const int parts = parts_of(a), size = ((a.vocab + parts - 1) / parts + 31) / 32 * 32;
    beam_select_kernel<T><<<a.batch * a.beams * parts, kThreads, 0, s>>>(
        a, parts, size, reinterpret_cast<int*>(p), reinterpret_cast<Found*>(p + kBeamCounters),
        reinterpret_cast<unsigned long long*>(p + kBeamCounters + found_bytes(a)));
    check_launch("beam_select");
}

}  // namespace

size_t beam_ws_bytes(const BeamArgs& a) {
    require(counter_bytes(a) <= kBeamCounters, "beam_select: too many requests in one call");
    return kBeamCounters + found_bytes(a) + size_t(a.batch) * a.beams * parts_of(a) * a.picks * 8;
}

void launch_beam_select(const BeamArgs& a, void* ws, cudaStream_t s) {
    if (a.type == kF32) launch<float>(a, ws, s);
    else if (a.type == kF16) launch<__half>(a, ws, s);
    else launch<__nv_bfloat16>(a, ws, s);
}

}  // namespace gpt
