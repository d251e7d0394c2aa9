// Attention of new tokens over the paged cache: few rows per key/value head (decode).
//
// out = sum_j w_j v_j / (sum_j w_j [+ exp(sink)]), w_j = exp(scale q.k_j) over the positions max(0, p - window + 1) ..
// p of the token at p; one pass with a running maximum and sum (base 2, fp32).
//
// Bound: the keys' and values' bytes, read once. A CTA is four warps that never wait for one another inside an item:
// each warp owns every fourth group of keys, copies it into its own ring of shared memory (16-byte asynchronous copies,
// page ids looked up one group ahead) and keeps its own statistics and accumulators for all R = 8 NT rows of the item;
// the four are put together at the item's end. The ring runs ahead across item boundaries, so memory stays busy while
// items are finished.
//
// Products are transposed, so that keys (16 at a time) and not the few rows fill the m16n8k16 instructions' long side:
// S^T [keys x rows] = K Q^T, O^T [dims x rows] += V^T P^T; P^T is S^T's own fragment with its 8 x 8 blocks turned by
// movmatrix. The running maximum is a reference that all lanes share and that moves (with a rescaling of O) only when a
// weight would pass what its type is used for (Weights in paged.cuh): most groups need no exchange between lanes at all.
//
// Measured: 64 sequences of 4K to 8K positions, one token each, 64 query heads over 8 of 64, bf16: 149 us, 5.5 TB/s
// (0.84 of the measured copy) with slot-major pages, whose rows of one head are 1 KB apart, 135 us, 6.1 TB/s with
// head-major ones; 32 heads over 4 of 128: 130 us, 6.3 TB/s. With rows along the instructions' long side, 16 keys at a
// time, 203 us.
//
// fp32 queries: a row is scaled by a power of two into [2^10, 2^11) and split into two fp16 parts (22 bits, exact
// products with fp16 keys); the weights are split the same way for the second product.
#include <algorithm>
#include <type_traits>

#include "paged_schedule.cuh"
#include "device_once.h"
#include "kernels.h"
#include "tc.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kWarps = 4, kThreads = kWarps * 32;
constexpr int kHalfSm = 113 * 1024;   // shared memory of a CTA when two share an SM
constexpr int kAhead = 10;       // pieces read at a time when an item is put together
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_trans(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <class C>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (std::is_same<C, __half>::value)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
            "{%0, %1, %2, %3};"
            : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Byte offset of 16-byte chunk c of row r in a tile of D-element rows: chunks permuted within each 128 bytes so that
// eight rows' equal chunks fall into eight different bank groups (ldmatrix without conflicts).
template <int D>
__device__ __forceinline__ uint32_t tile_off(int r, int c) {
    return uint32_t(r * D * 2 + ((c ^ (r & 7)) << 4));
}

// Whether either 16-bit value of a word is NaN or infinite (all exponent bits set).
template <class C>
__device__ __forceinline__ bool not_finite2(uint32_t w) {
    constexpr uint32_t e = std::is_same<C, __half>::value ? 0x7c00u : 0x7f80u;
    return (w & e) == e || (w >> 16 & e) == e;
}

// Transposes an 8 x 8 block of 16-bit values held one row pair per lane.
__device__ __forceinline__ uint32_t turn8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

template <class T, int D, int NT>
struct Shape {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int R = 8 * NT;
    static constexpr int kKeys = 2048 / D;                               // keys of a group: 32 or 16
    static constexpr int kStage = kKeys * D * 4;                         // its keys and values: 8 KB
    static constexpr int kQ = R * D * 2 * (kSplit ? 2 : 1);
    static constexpr int kPitch = D + 4;                                 // of a slab's row: no bank conflicts
    static constexpr int kSlab = kWarps * R * kPitch * 4;
    static constexpr int kRest = kQ + kSlab + (2 * kWarps + 1) * R * 4 + 64;
    static constexpr int kRing = kWarps * kStage;
    static constexpr int kStages = kRest + 3 * kRing <= kHalfSm ? 3 : 2;
    static constexpr int kSmem = kStages * kRing + kRest;
    static constexpr int kPerSm = kSmem <= kHalfSm ? 2 : 1;
};

// A piece's place in the workspace: R rows of D sums, then R maxima and R sums of weights.
template <int R, int D>
__host__ __device__ constexpr int slot_floats() {
    return R * D + 2 * R;
}

template <class T, class C, int D, int NT>
__global__ void __launch_bounds__(kThreads, Shape<T, D, NT>::kPerSm)
paged_rows_kernel(KvView c, KvBatch b, PagedAttnArgs a, FastDiv group, int* counters, float* slots) {
    using S = Shape<T, D, NT>;
    using W = Weights<C>;
    constexpr int R = S::R, NS = S::kStages, CH = D / 8, kGroup = S::kKeys, KT = kGroup / 16, PITCH = S::kPitch;
    extern __shared__ __align__(128) char smem[];
    char* ring = smem;
    char* q_tile = ring + kWarps * NS * S::kStage;
    float* slab = reinterpret_cast<float*>(q_tile + S::kQ);
    float* row_m = slab + kWarps * R * PITCH;             // [warp][row]
    float* row_l = row_m + kWarps * R;
    float* row_scale = row_l + kWarps * R;            // [row]
    int* flags = reinterpret_cast<int*>(row_scale + R);   // [0] poisoned, [1] last
    __shared__ long long scratch[kWarps + 2];

    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const Schedule<R, kGroup> sch{c, b, a.window, group, 1, a.rows_from, a.rows_to, a.check};
    const Span sp = find_span<kThreads>(sch, kWarps, scratch);
    if (sp.len == 0) return;
    const int G = int(group.d);

    // --- loader: this warp's groups (span indices warp, warp + 4, ...), NS - 1 ahead of the consumer
    Item li = sp.it;
    int lg = sp.g, left = sp.len > warp ? (sp.len - warp + kWarps - 1) / kWarps : 0;
    sch.step(li, lg, warp);
    int slot_in = 0;
    int next_id = 0, next_pos = 0;
    bool next_ok = false;
    const uint32_t ring0 = tc::smem_u32(ring) + warp * NS * S::kStage;
    const auto look_up = [&] {                        // lane l: the page of key l of the group to load next
        next_pos = li.lo + lg * kGroup + (lane & (kGroup - 1));
        next_ok = left > 0 && next_pos < li.hi;
        if (next_ok) next_id = __ldg(b.tables + (long long)li.b * b.table_stride + c.page.div(next_pos));
    };
    const auto issue = [&] {
        if (left > 0) {
            long long off = 0;
            if (next_ok)
                off = safe_page(next_id, c) * c.page_stride +
                      (next_pos - int(c.page.div(next_pos) * c.page.d)) * c.token_stride + li.h * c.head_stride;
            const unsigned okm = __ballot_sync(kFull, next_ok);
            const uint32_t dst = ring0 + slot_in * S::kStage;
#pragma unroll
            for (int i = 0; i < kGroup * CH / 32; ++i) {
                const int r = i * (32 / CH) + lane / CH, ch = lane % CH;
                const long long o = __shfl_sync(kFull, off, r) + ch * 16;
                const bool ok = okm >> r & 1;
                cp_async16_zfill(dst + tile_off<D>(r, ch), c.k + o, ok);
                cp_async16_zfill(dst + kGroup * D * 2 + tile_off<D>(r, ch), c.v + o, ok);
            }
            --left;
            sch.step(li, lg, kWarps);
            look_up();
        }
        cp_async_commit();
        slot_in = slot_in + 1 == NS ? 0 : slot_in + 1;
    };
    const auto stage_q = [&](const Item& it) {        // an item's queries to shared memory
        const int r0 = it.t * R;
        if constexpr (S::kSplit) {
            for (int r = warp; r < R; r += kWarps) {
                float x[D / 32], top = 0.f;
                const int tok = int(group.div(r0 + r));
                const float* src = static_cast<const float*>(a.q) + (long long)(it.s.row0 + tok) * a.q_stride +
                                   (it.h * G + (r0 + r - tok * G)) * D + lane * (D / 32);
#pragma unroll
                for (int e = 0; e < D / 32; ++e) {
                    x[e] = r < it.rows ? src[e] : 0.f;
                    top = fmaxf(top, fabsf(x[e]));
                }
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
                int ex = 0;
                if (top > 0.f && top < INFINITY) frexpf(top, &ex);      // top = f 2^ex, f in [1/2, 1)
                const float up = ldexpf(1.f, min(max(11 - ex, -126), 126));
#pragma unroll
                for (int e = 0; e < D / 32; ++e) {
                    const float y = x[e] * up;
                    const __half hi = __float2half_rn(y);
                    const int d = lane * (D / 32) + e;
                    char* p = q_tile + tile_off<D>(r, d / 8) + d % 8 * 2;
                    *reinterpret_cast<__half*>(p) = hi;
                    *reinterpret_cast<__half*>(p + R * D * 2) = __float2half_rn(y - __half2float(hi));
                }
                if (lane == 0) row_scale[r] = a.scale * kLog2e / up;
            }
        } else {
            for (int u = threadIdx.x; u < R * CH; u += kThreads) {
                const int r = u / CH, ch = u % CH, tok = int(group.div(r0 + r));
                uint4 x = make_uint4(0, 0, 0, 0);
                if (r < it.rows)
                    x = __ldg(reinterpret_cast<const uint4*>(
                        static_cast<const T*>(a.q) + (long long)(it.s.row0 + tok) * a.q_stride +
                        (it.h * G + (r0 + r - tok * G)) * D + ch * 8));
                *reinterpret_cast<uint4*>(q_tile + tile_off<D>(r, ch)) = x;
            }
        }
    };
    look_up();                                        // its latency passes while the first queries are fetched
    stage_q(sp.it);
#pragma unroll
    for (int i = 0; i < NS - 1; ++i) issue();

    int slot_out = 0, at = 0;                         // at: span index of the current piece's first group
    Item it = sp.it;
    int g0 = sp.g;
    if (threadIdx.x == 0) flags[0] = 0;
    while (at < sp.len) {
        const int g1 = min(it.n, g0 + sp.len - at);   // this piece: groups [g0, g1) of the item
        const int r0 = it.t * R;
        const int lo_last = a.window ? max(0, it.p1 - a.window + 1) : 0;
        if (at > 0) {
            __syncthreads();
            stage_q(it);
        }
        __syncthreads();
        float o[D / 16][NT][4], m[NT][2], l[NT][2], sc[NT][2];
        constexpr bool kHold = NT <= 2 && !(S::kSplit && D == 128);      // queries stay in registers
        uint32_t qf[kHold ? NT : 1][kHold ? D / 16 : 1][2], qg[kHold && S::kSplit ? NT : 1][kHold ? D / 16 : 1][2];
        const uint32_t q0 = tc::smem_u32(q_tile);
        const auto load_q = [&](int nt, int k, uint32_t (&x)[4]) {       // B fragments of dims 16 k .. 16 k + 31
            ldsm4(q0 + tile_off<D>(nt * 8 + lane % 8, 2 * k + lane / 8), x);
        };
        const auto load_q_low = [&](int nt, int k, uint32_t (&x)[4]) {
            ldsm4(q0 + R * D * 2 + tile_off<D>(nt * 8 + lane % 8, 2 * k + lane / 8), x);
        };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                m[nt][e] = -INFINITY;
                l[nt][e] = 0.f;
                sc[nt][e] = S::kSplit ? row_scale[nt * 8 + lane % 4 * 2 + e] : a.scale * kLog2e;
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[n][nt][e] = 0.f;
            if constexpr (kHold) {
#pragma unroll
                for (int k = 0; k < D / 16; k += 2) {
                    uint32_t x[4];
                    load_q(nt, k, x);
                    qf[nt][k][0] = x[0]; qf[nt][k][1] = x[1]; qf[nt][k + 1][0] = x[2]; qf[nt][k + 1][1] = x[3];
                    if constexpr (S::kSplit) {
                        load_q_low(nt, k, x);
                        qg[nt][k][0] = x[0]; qg[nt][k][1] = x[1]; qg[nt][k + 1][0] = x[2]; qg[nt][k + 1][1] = x[3];
                    }
                }
            }
        }
        // --- this warp's groups: span indices i = warp mod 4 in [at, at + g1 - g0)
        bool poisoned = false;
        for (int i = at + ((warp - at) & (kWarps - 1)); i < at + g1 - g0; i += kWarps) {
            const int k0 = it.lo + (g0 + i - at) * kGroup;
            const bool edge = k0 + kGroup > it.p0 + 1 || k0 < lo_last;
            issue();                                  // into the slot read in the previous step
            cp_async_wait_group<NS - 1>();
            __syncwarp();
            const uint32_t kt = ring0 + slot_out * S::kStage, vt = kt + kGroup * D * 2;
            slot_out = slot_out + 1 == NS ? 0 : slot_out + 1;
            float s[KT][NT][4];
#pragma unroll
            for (int x = 0; x < KT; ++x)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[x][nt][e] = 0.f;
#pragma unroll
            for (int k = 0; k < D / 16; k += 2) {
                uint32_t ka[KT][2][4];
#pragma unroll
                for (int x = 0; x < KT; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) ldsm4(kt + tile_off<D>(x * 16 + lane % 16, 2 * (k + y) + lane / 16),
                        ka[x][y]);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    uint32_t q[4];
                    if constexpr (kHold) {
                        q[0] = qf[nt][k][0]; q[1] = qf[nt][k][1]; q[2] = qf[nt][k + 1][0]; q[3] = qf[nt][k + 1][1];
                    } else {
                        load_q(nt, k, q);
                    }
#pragma unroll
                    for (int y = 0; y < 2; ++y)
#pragma unroll
                        for (int x = 0; x < KT; ++x) mma16816<C>(s[x][nt], ka[x][y], q[2 * y], q[2 * y + 1]);
                    if constexpr (S::kSplit) {
                        if constexpr (kHold) {
                            q[0] = qg[nt][k][0]; q[1] = qg[nt][k][1]; q[2] = qg[nt][k + 1][0]; q[3] = qg[nt][k + 1][1];
                        } else {
                            load_q_low(nt, k, q);
                        }
#pragma unroll
                        for (int y = 0; y < 2; ++y)
#pragma unroll
                            for (int x = 0; x < KT; ++x) mma16816<C>(s[x][nt], ka[x][y], q[2 * y], q[2 * y + 1]);
                    }
                }
            }
            // scores in base 2; element (x, nt, 2 y + e): key x * 16 + lane / 4 + 8 y, row nt * 8 + lane % 4 * 2 + e
            float top[NT][2];
            bool past = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int x = 0; x < KT; ++x)
#pragma unroll
                        for (int y = 0; y < 2; ++y) s[x][nt][2 * y + e] *= sc[nt][e];
                    if (edge) {
                        const int row = min(nt * 8 + lane % 4 * 2 + e, it.rows - 1);
                        const int p = it.s.len - it.s.n + int(group.div(r0 + row));
                        const int first = a.window ? p - a.window + 1 : 0;
#pragma unroll
                        for (int x = 0; x < KT; ++x)
#pragma unroll
                            for (int y = 0; y < 2; ++y) {
                                const int key = k0 + x * 16 + lane / 4 + 8 * y;
                                if (key > p || key < first) s[x][nt][2 * y + e] = -INFINITY;
                            }
                    }
                    top[nt][e] = fmaxf(s[0][nt][e], s[0][nt][2 + e]);
#pragma unroll
                    for (int x = 1; x < KT; ++x) top[nt][e] = fmaxf(top[nt][e], fmaxf(s[x][nt][e], s[x][nt][2 + e]));
                    past |= top[nt][e] - m[nt][e] > W::kLift + W::kSlack;
                }
            // (as the weights' exponents are computed, and the reference rounded up: no weight is larger than meant)
            if (__any_sync(kFull, past)) {            // move the references: kLift below the rows' maxima so far
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        float mm = fmaxf(m[nt][e], __fsub_ru(top[nt][e], W::kLift));
#pragma unroll
                        for (int z = 4; z < 32; z <<= 1) mm = fmaxf(mm, __shfl_xor_sync(kFull, mm, z));
                        const float f = ex2(m[nt][e] - (mm == -INFINITY ? 0.f : mm));
                        m[nt][e] = mm;
                        l[nt][e] *= f;
#pragma unroll
                        for (int n = 0; n < D / 16; ++n) {
                            o[n][nt][e] *= f;
                            o[n][nt][2 + e] *= f;
                        }
                    }
            }
            constexpr bool half = std::is_same<C, __half>::value;
            uint32_t pa[KT][NT][2], pb[S::kSplit ? KT : 1][NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                const float b0 = m[nt][0] == -INFINITY ? 0.f : m[nt][0], b1 = m[nt][1] == -INFINITY ? 0.f : m[nt][1];
#pragma unroll
                for (int x = 0; x < KT; ++x)
#pragma unroll
                    for (int y = 0; y < 2; ++y) {
                        const float u = ex2(s[x][nt][2 * y] - b0), v = ex2(s[x][nt][2 * y + 1] - b1);
                        l[nt][0] += u;
                        l[nt][1] += v;
                        const uint32_t w = pack2(u, v, half);
                        pa[x][nt][y] = turn8x8(w);
                        if constexpr (S::kSplit) {
                            const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&w));
                            pb[x][nt][y] = turn8x8(pack2(u - r.x, v - r.y, half));
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < D / 16; ++n)
#pragma unroll
                for (int x = 0; x < KT; ++x) {
                    uint32_t va[4];
                    ldsm4_trans(vt + tile_off<D>(x * 16 + lane % 8 + lane / 16 * 8, 2 * n + lane / 8 % 2), va);
                    if (edge)
                        poisoned |= not_finite2<C>(va[0]) | not_finite2<C>(va[1]) | not_finite2<C>(va[2]) |
                                    not_finite2<C>(va[3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma16816<C>(o[n][nt], va, pa[x][nt][0], pa[x][nt][1]);
                        if constexpr (S::kSplit) mma16816<C>(o[n][nt], va, pb[x][nt][0], pb[x][nt][1]);
                    }
                }
            __syncwarp();                             // all lanes have read the slot before it is filled again
        }
        // --- the four warps together
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
                for (int z = 4; z < 32; z <<= 1) l[nt][e] += __shfl_xor_sync(kFull, l[nt][e], z);
                if (lane < 4) {
                    row_m[warp * R + nt * 8 + lane * 2 + e] = m[nt][e];
                    row_l[warp * R + nt * 8 + lane * 2 + e] = l[nt][e];
                }
            }
        if (poisoned) flags[0] = 1;
        __syncthreads();
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = nt * 8 + lane % 4 * 2 + e;
                float top = row_m[row];
#pragma unroll
                for (int w = 1; w < kWarps; ++w) top = fmaxf(top, row_m[w * R + row]);
                const float f = top == -INFINITY ? 0.f : ex2(m[nt][e] - top);
#pragma unroll
                for (int n = 0; n < D / 16; ++n) {
                    slab[(warp * R + row) * PITCH + n * 16 + lane / 4] = o[n][nt][e] * f;
                    slab[(warp * R + row) * PITCH + n * 16 + lane / 4 + 8] = o[n][nt][2 + e] * f;
                }
            }
        __syncthreads();
        const bool whole = g0 == 0 && g1 == it.n;
        if (flags[0]) {                               // redo the piece without products of masked values
            const int klo = it.lo + g0 * kGroup, khi = min(it.hi, it.lo + g1 * kGroup);
            for (int r = warp; r < it.rows; r += kWarps) {
                const int tok = int(group.div(r0 + r)), p = it.s.len - it.s.n + tok;
                float mm, ll, oo[D / 32];
                careful_row<T, C, D>(c, b, a, it.b, it.h,
                                     (long long)(it.s.row0 + tok) * a.q_stride + (it.h * G + (r0 + r - tok * G)) * D,
                                     max(klo, a.window ? p - a.window + 1 : 0), min(khi, p + 1), &mm, &ll, oo);
                for (int e = 0; e < D / 32; ++e) {
                    slab[r * PITCH + lane * (D / 32) + e] = oo[e];
                    for (int w = 1; w < kWarps; ++w) slab[(w * R + r) * PITCH + lane * (D / 32) + e] = 0.f;
                }
                if (lane < kWarps) {
                    row_m[lane * R + r] = lane ? -INFINITY : mm;
                    row_l[lane * R + r] = lane ? 0.f : ll;
                }
            }
            __syncthreads();
            if (threadIdx.x == 0) flags[0] = 0;
        }
        // piece of an item: my slot is 2 c (the item began before my span) or 2 c + 1 (it goes on past it)
        const int mine = 2 * blockIdx.x + (g0 > 0 ? 0 : 1);
        float* my = slots + (long long)mine * slot_floats<R, D>();
        for (int u = threadIdx.x; u < it.rows * (D / 4); u += kThreads) {
            const int r = u / (D / 4), d = u % (D / 4) * 4;
            float top = row_m[r];
#pragma unroll
            for (int w = 1; w < kWarps; ++w) top = fmaxf(top, row_m[w * R + r]);
            float z = 0.f;
            float4 x = make_float4(0, 0, 0, 0);
#pragma unroll
            for (int w = 0; w < kWarps; ++w) {
                z += top == -INFINITY ? 0.f : row_l[w * R + r] * ex2(row_m[w * R + r] - top);
                const float4 y = *reinterpret_cast<const float4*>(slab + (w * R + r) * PITCH + d);
                x.x += y.x; x.y += y.y; x.z += y.z; x.w += y.w;
            }
            if (whole) {
                const int tok = int(group.div(r0 + r)), head = it.h * G + (r0 + r - tok * G);
                if (a.sinks && z > 0.f) z += ex2(a.sinks[head] * kLog2e - top);
                const float inv = z == 0.f ? 0.f : 1.f / z;
                T* dst = static_cast<T*>(a.out) + (long long)(it.s.row0 + tok) * a.out_stride + head * D + d;
                if constexpr (S::kSplit) {
                    *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                } else {
                    constexpr bool half = std::is_same<T, __half>::value;
                    *reinterpret_cast<uint2*>(dst) =
                        make_uint2(pack2(x.x * inv, x.y * inv, half), pack2(x.z * inv, x.w * inv, half));
                }
            } else {
                *reinterpret_cast<float4*>(my + r * D + d) = x;
                if (d == 0) {
                    my[R * D + r] = top;
                    my[R * D + R + r] = z;
                }
            }
        }
        if (!whole) {
            // the item's first CTA and the number of its pieces follow from where its groups lie
            const long long first = sp.start + at - g0;
            const int c0 = blockIdx.x - (first < sp.start ? ceil_div(sp.start - first, sp.per) : 0);
            const int c1 = blockIdx.x + int(unsigned(first + it.n - 1 - sp.start) / unsigned(sp.per));
            __syncthreads();
            if (threadIdx.x == 0) {
                const int done = arrive(&counters[c0]);
                flags[1] = done == c1 - c0;
                if (done == c1 - c0) counters[c0] = 0;
            }
            __syncthreads();
            if (flags[1]) {
                for (int u = threadIdx.x; u < it.rows * (D / 4); u += kThreads) {
                    const int r = u / (D / 4), d = u % (D / 4) * 4;
                    float top = -INFINITY, z = 0.f;
                    float4 x = make_float4(0, 0, 0, 0);
                    for (int i0 = c0; i0 <= c1; i0 += kAhead) {      // kAhead pieces' reads in flight at a time
                        float pm[kAhead], pz[kAhead];
                        float4 y[kAhead];
#pragma unroll
                        for (int e = 0; e < kAhead; ++e) {
                            const int i = min(i0 + e, c1);
                            const float* ps = slots + (long long)(2 * i + (i == c0)) * slot_floats<R, D>();
                            pm[e] = i0 + e <= c1 ? __ldcg(ps + R * D + r) : -INFINITY;
                            pz[e] = __ldcg(ps + R * D + R + r);
                            y[e] = __ldcg(reinterpret_cast<const float4*>(ps + r * D + d));
                        }
                        float mm = top;
#pragma unroll
                        for (int e = 0; e < kAhead; ++e) mm = fmaxf(mm, pm[e]);
                        const float base = mm == -INFINITY ? 0.f : mm, f0 = ex2(top - base);
                        z *= f0;
                        x.x *= f0; x.y *= f0; x.z *= f0; x.w *= f0;
                        top = mm;
#pragma unroll
                        for (int e = 0; e < kAhead; ++e) {
                            const float f = ex2(pm[e] - base);
                            z += pz[e] * f;
                            x.x += y[e].x * f; x.y += y[e].y * f; x.z += y[e].z * f; x.w += y[e].w * f;
                        }
                    }
                    const int tok = int(group.div(r0 + r)), head = it.h * G + (r0 + r - tok * G);
                    if (a.sinks && z > 0.f) z += ex2(a.sinks[head] * kLog2e - top);
                    const float inv = z == 0.f ? 0.f : 1.f / z;
                    T* dst = static_cast<T*>(a.out) + (long long)(it.s.row0 + tok) * a.out_stride + head * D + d;
                    if constexpr (S::kSplit) {
                        *reinterpret_cast<float4*>(dst) = make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv);
                    } else {
                        constexpr bool half = std::is_same<T, __half>::value;
                        *reinterpret_cast<uint2*>(dst) =
                            make_uint2(pack2(x.x * inv, x.y * inv, half), pack2(x.z * inv, x.w * inv, half));
                    }
                }
            }
        }
        at += g1 - g0;
        g0 = 0;
        if (at < sp.len) sch.next(it);
    }
}

constexpr int kMaxCtas = 2 * 160;                     // two CTAs per SM, SMs rounded up
static_assert(kMaxCtas * sizeof(int) <= kCounterBytes, "one counter per CTA");
constexpr int kSlotFloats = std::max(slot_floats<32, 64>(), slot_floats<16, 128>());

template <class T, class C, int D, int NT>
void launch(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws, cudaStream_t s) {
    using S = Shape<T, D, NT>;
    static DeviceOnce once;
    int dev = 0;
    GPT_CHECK(cudaGetDevice(&dev));
    once.run(dev, [] {
        GPT_CHECK(cudaFuncSetAttribute(paged_rows_kernel<T, C, D, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       S::kSmem));
    });
    const int grid = std::min(kMaxCtas, num_sms() * S::kPerSm);
    PagedAttnArgs args = a;
    args.check = many_groups(b, c, a, S::kKeys, S::R);
    paged_rows_kernel<T, C, D, NT><<<grid, kThreads, S::kSmem, s>>>(
        c, b, args, FastDiv::of(uint32_t(a.q_heads / c.kv_heads)), static_cast<int*>(ws),
        reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes));
    check_launch("paged_attention");
}

template <class T, class C>
void by_shape(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws, cudaStream_t s) {
    const long long rows = (long long)b.max_new * (a.q_heads / c.kv_heads);
    if (c.dim == 64) {
        if (rows <= 8) launch<T, C, 64, 1>(c, b, a, ws, s);
        else if (rows <= 16) launch<T, C, 64, 2>(c, b, a, ws, s);
        else launch<T, C, 64, 4>(c, b, a, ws, s);
    } else {
        if (rows <= 8) launch<T, C, 128, 1>(c, b, a, ws, s);
        else launch<T, C, 128, 2>(c, b, a, ws, s);
    }
}

// Query rows per key/value head up to which the kernel of this file takes a sequence. Both sides, 64 sequences of 4K to
// 8K positions / 2 of them, 64 query heads over 8: 64 rows of heads of 64 (as two tiles of 32) 296 / 28 us here, 285 /
// 42 us on the 128-row tiles; 32 rows 170 / 24 us here, 254 / 43 us there. Heads of 128 (32 over 4): 32 rows 283 us
// here, 259 us there, 64 rows 492 us and 211 us.
int few_rows_of(int dim) { return dim == 64 ? 64 : 16; }

void few_rows(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws, cudaStream_t s) {
    if (a.type == kF32) by_shape<float, __half>(c, b, a, ws, s);
    else if (a.type == kF16) by_shape<__half, __half>(c, b, a, ws, s);
    else by_shape<__nv_bfloat16, __nv_bfloat16>(c, b, a, ws, s);
}

}  // namespace

size_t paged_attention_ws_bytes(int dim) {
    return std::max(kCounterBytes + kMaxCtas * 2 * sizeof(float) * kSlotFloats, paged_tiles_ws_bytes(dim));
}

void launch_paged_attention(const KvMaps& maps, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws,
    cudaStream_t s) {
    const long long most = (long long)b.max_new * (a.q_heads / c.kv_heads);
    const int few_at_most = few_rows_of(c.dim);
    if (most <= few_at_most) return few_rows(c, b, a, ws, s);
    // Chunks go to the tensor-core tiles. Where sequences differ in length (the batch's tokens say so), those of few
    // rows, decoding beside a chunk, are left out of that launch and take one of their own.
    const bool mixed = b.tokens < (long long)b.seqs * b.max_new && b.seqs > 1;
    PagedAttnArgs part = a;
    if (mixed) part.rows_from = few_at_most + 1;
    launch_paged_tiles(maps, c, b, part, ws, s);
    if (!mixed) return;
    part.rows_from = 0;
    part.rows_to = few_at_most;
    KvBatch few = b;
    // (their mean length, the longest sequence aside, steers the choice of tile)
    few.max_new = std::max(1, (b.tokens - b.max_new + b.seqs - 2) / (b.seqs - 1));
    few_rows(c, few, part, ws, s);
}

}  // namespace gpt
