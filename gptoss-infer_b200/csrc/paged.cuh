// Device helpers of the paged cache kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "paged.h"

namespace gpt {
namespace paged {

__device__ __forceinline__ void report(int* err, int code) { atomicCAS(err, 0, code); }

// The sequence that row t of the batch belongs to: the last b with cu[b] <= t, by a 32-way search of one warp (two
// dependent reads for up to 1024 sequences). Reads cu[0 .. seqs - 1] only, whatever the values.
__device__ __forceinline__ int find_sequence(const int* __restrict__ cu, int seqs, int t, int lane) {
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + lane * step;
        const unsigned below = __ballot_sync(kFull, at < hi && cu[at] <= t);
        const int n = below ? 32 - __clz(below) : 1;
        lo += (n - 1) * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

// A length forced into 0 .. most (with an error word).
__device__ __forceinline__ int safe_len(int len, int most, int* err) {
    if (unsigned(len) <= unsigned(most)) return len;
    report(err, kKvBadLength);
    return len < 0 ? 0 : most;
}

// Sequence b's rows and cache length, forced into range (with an error word) whatever the arrays hold.
struct Seq {
    int row0, n, len;        // first row, new tokens, cache length with them
};
__device__ __forceinline__ Seq load_seq(const KvBatch& b, int i, int* err) {
    int r0 = b.cu[i], r1 = b.cu[i + 1];
    if (r0 < 0 || r1 < r0 || r1 > b.tokens) {
        report(err, kKvBadBatch);
        r0 = min(max(r0, 0), b.tokens);
        r1 = min(max(r1, r0), b.tokens);
    }
    return {r0, r1 - r0, safe_len(b.lens[i], b.most, err)};
}

__device__ __forceinline__ int safe_page(int id, const KvView& c) {
    if (unsigned(id) < unsigned(c.num_pages)) return id;
    report(c.err, kKvBadPage);
    return 0;
}

// One more arrival at a counter, after everything this CTA wrote (the caller has passed a barrier since); what the
// earlier arrivals wrote is visible to the CTA after its next barrier.
__device__ __forceinline__ int arrive(int* counter) {
    int old;
    asm volatile("atom.add.acq_rel.gpu.global.s32 %0, [%1], 1;" : "=r"(old) : "l"(counter) : "memory");
    return old;
}

template <class T>
__device__ __forceinline__ float to_f32(T x);
template <>
__device__ __forceinline__ float to_f32(float x) { return x; }
template <>
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// Stores one value rounded to nearest in the given type.
__device__ __forceinline__ void store_as(void* base, long long i, float x, int type) {
    if (type == kF32) static_cast<float*>(base)[i] = x;
    else if (type == kF16) static_cast<__half*>(base)[i] = __float2half_rn(x);
    else static_cast<__nv_bfloat16*>(base)[i] = __float2bfloat16_rn(x);
}

__device__ __forceinline__ uint32_t pack2(float a, float b, bool half) {
    if (half) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
}

// Weights are exp2(score - m) with a reference m that moves when a score passes it by kLift + kSlack, and then to kLift
// below the largest score so far: a row's largest weight is stored as 2^kLift .. 2^(kLift + kSlack), the factor falls out
// of the quotient. fp16 ends at 2^-24 whatever the weights' scale, so they are stored near its upper end (65504): what is
// lost of a weight is at most 2^-38 of the row's largest, below its own rounding (2^-12; 2^-23 in two parts) down to
// 2^-26 (2^-15) of the largest. With kLift 0 and kSlack 8 the many small weights beside a dominant key vanished: 0.11 %
// of the weight over 16384 keys came out 1 % wrong. (The narrower slack costs rescaling: a chunk of 511 with a window of
// 1000, fp16, 70.4 us before, 71.9 us now; 73 us with kSlack 2.) bf16 has fp32's exponents and needs no lift.
template <class C>
struct Weights {
    static constexpr bool kHalf = std::is_same<C, __half>::value;
    static constexpr float kLift = kHalf ? 13.f : 0.f, kSlack = kHalf ? 2.9f : 8.f;
};

// Eight consecutive values as loaded: one 16-byte word of 16-bit ones, two of fp32.
template <class T, int Q>
__device__ __forceinline__ void unpack8(const uint4 (&a)[Q], float (&x)[8]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            x[4 * i] = __uint_as_float(a[i].x);
            x[4 * i + 1] = __uint_as_float(a[i].y);
            x[4 * i + 2] = __uint_as_float(a[i].z);
            x[4 * i + 3] = __uint_as_float(a[i].w);
        }
    } else {
        const uint32_t w[4] = {a[0].x, a[0].y, a[0].z, a[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                x[2 * i] = f.x;
                x[2 * i + 1] = f.y;
            } else {
                x[2 * i] = __uint_as_float(w[i] << 16);
                x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
            }
        }
    }
}

__device__ __forceinline__ void store8(char* p, const float (&x)[8], int type) {
    if (type == kF32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
    } else {
        const bool h = type == kF16;
        *reinterpret_cast<uint4*>(p) = make_uint4(pack2(x[0], x[1], h), pack2(x[2], x[3], h), pack2(x[4], x[5], h),
                                                  pack2(x[6], x[7], h));
    }
}

}  // namespace paged
}  // namespace gpt
