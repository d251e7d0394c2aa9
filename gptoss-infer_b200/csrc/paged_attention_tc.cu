// Attention of new tokens over the paged cache: many rows per key/value head (prompt chunks), on tcgen05 tensor cores.
//
// The same sum as in paged_attention.cu. An item is 256 query rows (row = token * group + head of the group: all query
// heads of a key/value head share its tiles) against tiles of 128 keys. Per tile and half of 128 rows:
//   S = Q K^T            tcgen05.mma kind::f16, both operands in shared memory, K-major, accumulator in TMEM
//   P = exp2(S - m)      one thread per row, no exchange between threads
//   O += P V             A operand P read from TMEM, V in shared memory as stored (rows = keys)
// S is taken in tiles of 64 keys (128 for 16-bit heads of 64, whose P has columns of its own), read into registers and
// released at once, so the next scores are made while this tile's exponentials run; the products are issued in the
// order in which two halves half a step apart need them.
//
// Bound: the exponentials: 16 a clock and SM, 2048 cycles for 256 rows x 128 keys, against 1024 (heads of 64) and
// 2560 (heads of 128) of products. Measured, 2048 new tokens over 16384 positions, 64 query heads over 8, bf16:
// heads of 64 691 us in a graph of 20 calls, 745 TFLOP/s, 45 % of the measured matrix rate (677 us at its best):
// about 3100 cycles a step. Two warps of rows per scheduler do not keep the special-function unit busy alone (a
// warp's 128 exponentials take about 1800 cycles by themselves), and waits for products (about 600 cycles from
// weights written to their product seen) fall between. 32 heads of 128 over 4: 538 us, 958 TFLOP/s (510 us alone).
// Tried: reading the scores twice instead of holding them (1110 us), halves taking strict turns at the exponentials
// (974 us), polling for whatever product is ready (735 us), 3 and 4 of 8 exponentials on the fp32 pipes.
//
// Warps: 0-3 and 4-7 the rows of the two halves (softmax, rescaling, output); the next two copy keys and values through
// a ring of tiles with TMA (a box per run of slots in a page; page sizes that are multiples of 8), or the next four
// with 16-byte asynchronous copies (any page size); one more issues the products. The weights' reference moves only
// when the maximum has grown past kSlack (Weights in paged.cuh), so the accumulator in TMEM is rescaled rarely.
//
// fp32 queries: two fp16 parts of a row scaled by a power of two, and two of the weights, as in paged_attention.cu.
// (2048 over 16384, heads of 64: 1.13 ms, 456 TFLOP/s of the sum's own operations, twice that in products.)
#include <algorithm>
#include <type_traits>

#include "paged_schedule.cuh"
#include "device_once.h"
#include "kernels.h"
#include "tc.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kRows = 256, kHalf = 128, kTile = 128;
// Threads that bring in keys, values and queries: two warps with TMA, four without; one warp more issues the products.
constexpr int copy_threads(bool tma) { return tma ? 64 : 128; }
constexpr int block_threads(bool tma) { return tma ? 384 : 512; }
// Of 8 pairs of exponentials, those computed on the fp32 pipes beside the special-function unit (2048 tokens over
// 16384, heads of 64, bf16: 0 of 8 747 us, 2 748, 3 790; heads of 128: 551, 540, 546).
constexpr int kMixed = 2;
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void cp_async16_zfill(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
// 5-D tiled TMA load: 64 dims (128 bytes, swizzled) x slots of one head, page and layer.
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int d, int h, int slot, int page,
                                            int layer, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, "
        "%6}], [%7];" ::"r"(dst),
        "l"(map), "r"(d), "r"(h), "r"(slot), "r"(page), "r"(layer), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Instruction descriptor of tcgen05.mma kind::f16: fp32 accumulator (bit 4), A and B both fp16 (0) or both bf16 (1) in
// bits 7-9 and 10-12, B rows = K when `turned` (bit 16), N >> 3 in bits 17-22, M >> 4 in bits 24-28.
__host__ __device__ constexpr uint32_t idesc_f16(bool bf16, bool turned, int M, int N) {
    return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(turned) << 16) |
           (uint32_t(N >> 3) << 17) | (uint32_t(M >> 4) << 24);
}
// Shared-memory descriptors in the 128-byte swizzled layout: the high word (stride between 8-row groups 1024 bytes,
// version 1, layout 2) is common to all, the low word is the address and the leading offset, both in 16-byte units.
__device__ __forceinline__ uint64_t desc_of(uint32_t low) {
    constexpr uint32_t high = (1024u >> 4) | (1u << 14) | (2u << 29);
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(low), "r"(high));
    return d;
}
// D (+)= A B^T, A and B in shared memory. Issued by one thread; M = 128, K = 16 takes 48, 64 and 128 cycles for N = 64,
// 128 and 256.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}
// D (+)= A B, A in TMEM (one lane per row, two 16-bit values per column): 32 and 64 cycles for N = 64 and 128.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(uint32_t(accumulate))
        : "memory");
}
__device__ __forceinline__ void tmem_st_x16(uint32_t taddr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
        "%15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// A wait's outcome as the whole warp's.
__device__ __forceinline__ bool all_ok(bool ok) { return __all_sync(kFull, ok); }
// One arrival for the whole warp, after all its lanes' work (32 arrivals on one barrier take turns).
__device__ __forceinline__ void arrive_warp(uint64_t* bar) {
    __syncwarp();
    if (threadIdx.x % 32 == 0) tc::mbar_arrive(bar);
}
template <int N>
__device__ __forceinline__ void bar_copies() { asm volatile("bar.sync 2, %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void bar_rows() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Scores outside [from, to] become -infinity: a word of bits per run of 32, tested bit by bit (branches around the
// scores' registers made them spill).
template <int N>
__device__ __forceinline__ void mask(uint32_t (&x)[N], int from, int to) {
#pragma unroll
    for (int r = 0; r < N; r += 32) {
        const int lo = min(max(from - r, 0), 32), hi = min(max(to - r + 1, 0), 32);      // seen: [lo, hi)
        const uint32_t below_hi = hi == 32 ? ~0u : (1u << hi) - 1, below_lo = lo == 32 ? ~0u : (1u << lo) - 1;
        const uint32_t seen = below_hi & ~below_lo;
#pragma unroll
        for (int i = 0; i < 32; ++i)
            if (!(seen & (1u << i))) x[r + i] = 0xff800000u;
    }
}

// Two fp32 values in a register pair: one instruction for both.
__device__ __forceinline__ uint64_t pair(uint32_t x, uint32_t y) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(x), "r"(y));
    return r;
}
__device__ __forceinline__ void unpair(uint64_t p, float& x, float& y) {
    asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(p));
}
__device__ __forceinline__ uint64_t fma2(uint64_t x, uint64_t y, uint64_t z) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(x), "l"(y), "l"(z));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t x, uint64_t y) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(x), "l"(y));
    return r;
}

// The largest of three, NaN if one of them is.
__device__ __forceinline__ float max3_nan(float x, float y, float z) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}

// 2^x of two values on the fp32 pipes: x = n + f with n = round(x), |f| <= 1/2 (the sum with 1.5 * 2^23 leaves n in the
// low mantissa bits), 2^f by the polynomial of least largest relative error on [-1/2, 1/2] (weighted least squares
// iterated to equal ripple; degree 3: 7.5e-5, degree 4: 2.6e-6), n added to its exponent. x below -126 counts as
// -126, and so does NaN: not for scores that are not finite.
template <int DEGREE>
__device__ __forceinline__ void exp2_pair(uint64_t x2, float& u, float& v) {
    const auto both = [](float c) { return pair(__float_as_uint(c), __float_as_uint(c)); };
    float a, b;
    unpair(x2, a, b);
    x2 = pair(__float_as_uint(fmaxf(a, -126.f)), __float_as_uint(fmaxf(b, -126.f)));
    const uint64_t r = add2(x2, both(12582912.f)), f = fma2(add2(r, both(-12582912.f)), both(-1.f), x2);
    uint64_t y;
    if constexpr (DEGREE == 3) {
        y = fma2(both(0.0551716685f), f, both(0.242611125f));
        y = fma2(y, f, both(0.693260968f));
        y = fma2(y, f, both(0.999928057f));
    } else {
        y = fma2(both(0.0095701022f), f, both(0.0559178591f));
        y = fma2(y, f, both(0.240247443f));
        y = fma2(y, f, both(0.693121791f));
        y = fma2(y, f, both(0.999999285f));
    }
    float ya, yb, ra, rb;
    unpair(y, ya, yb);
    unpair(r, ra, rb);
    u = __uint_as_float(__float_as_uint(ya) + (__float_as_uint(ra) << 23));
    v = __uint_as_float(__float_as_uint(yb) + (__float_as_uint(rb) << 23));
}

// Weights exp2(score * sc + shift) as 16-bit values, two a TMEM column, to p_at; SPLIT: what rounding took from them to
// p_low. Returns the fp32 weights' sum. MIX: kMixed of every 8 pairs on the fp32 pipes.
template <class C, bool SPLIT, bool MIX, int N>
__device__ __forceinline__ float weights(const uint32_t (&x)[N], float sc, float shift, uint32_t p_at, uint32_t p_low) {
    constexpr bool half = std::is_same<C, __half>::value;
    const uint64_t sc2 = pair(__float_as_uint(sc), __float_as_uint(sc)),
                   shift2 = pair(__float_as_uint(shift), __float_as_uint(shift));
    uint64_t sum[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; i += 32) {
        uint32_t hi[16], low[SPLIT ? 16 : 1];
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const uint64_t x2 = fma2(pair(x[i + 2 * e], x[i + 2 * e + 1]), sc2, shift2);
            float u, v;
            if (MIX && e * kMixed % 8 < kMixed) {
                exp2_pair<half ? 4 : 3>(x2, u, v);
            } else {
                unpair(x2, u, v);
                u = ex2(u);
                v = ex2(v);
            }
            sum[e & 1] = add2(sum[e & 1], pair(__float_as_uint(u), __float_as_uint(v)));
            hi[e] = pack2(u, v, half);
            if constexpr (SPLIT) {
                const float2 r = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
                low[e] = pack2(u - r.x, v - r.y, true);
            }
        }
        tmem_st_x16(p_at + i / 2, hi);
        if constexpr (SPLIT) tmem_st_x16(p_low + i / 2, low);
    }
    float a, b, c, d;
    unpair(sum[0], a, b);
    unpair(sum[1], c, d);
    return (a + b) + (c + d);
}

// Shared-memory image of 128 rows of D 16-bit values: halves of 64 columns, each in the 128-byte swizzled layout. As a
// K-major operand the rows are M or N; as V the rows are K (8-row groups 1024 bytes apart, 64-column halves 16 KB
// apart).
template <int D>
__device__ __forceinline__ uint32_t image_off(int r, int chunk) {
    return uint32_t((chunk >> 3) * (128 * 128) + r * 128 + (((chunk & 7) ^ (r & 7)) << 4));
}

template <class T, int D, bool TMA>
struct Layout {
    static constexpr bool kSplit = sizeof(T) == 4;
    static constexpr int kScores = TMA && D == 64 && !kSplit ? 128 : 64;        // keys of a score tile in TMEM
    static constexpr int kTileBytes = 128 * D * 2;                       // a tile of keys or of values
    static constexpr int kQ = 2 * kTileBytes * (kSplit ? 2 : 1);         // [half][part]
    static constexpr int kSlots = D == 64 ? 8 : (kSplit ? 3 : 5);
    static constexpr int kSmem = kQ + kSlots * kTileBytes + 2 * kRows + 2 * kTile * 8 + 512;
};

template <int D>
__host__ __device__ constexpr int slot_floats() {
    return kRows * D + 2 * kRows;                                        // sums [dim][row], maxima, sums of weights
}

enum Bars { kTileFull = 0, kFree = 8, kSFull = 16, kSFree = 18, kPFull = 20, kPvDone = 22, kQFull = 24, kQFree = 25,
    kDrain = 26, kEdge = 27, kBars = 28 };

template <class T, class C, int D, bool TMA>
__global__ void __launch_bounds__(block_threads(TMA), 1)
paged_tiles_kernel(const __grid_constant__ KvMaps maps, KvView c, KvBatch b, PagedAttnArgs a, FastDiv group,
    int* counters,
                   float* slots) {
    using L = Layout<T, D, TMA>;
    using W = Weights<C>;
    constexpr int kThreads = block_threads(TMA), kCopy = copy_threads(TMA);
    constexpr int NS = L::kSlots, CH = D / 8, SK = L::kScores, SUB = kTile / SK;
    constexpr bool kBf16 = std::is_same<C, __nv_bfloat16>::value;
    constexpr int kMma = 8 + kCopy / 32;              // the warp that issues the products
    extern __shared__ __align__(1024) char smem[];
    char* q_tile = smem;
    char* ring = smem + L::kQ;
    int8_t* row_exp = reinterpret_cast<int8_t*>(ring + NS * L::kTileBytes);     // [piece parity][row]: scaled by 2^exp
    long long* row_off = reinterpret_cast<long long*>(row_exp + 2 * kRows);     // [2][key of the tile]
    uint64_t* bars = reinterpret_cast<uint64_t*>(row_off + 2 * kTile);
    int* flags = reinterpret_cast<int*>(bars + kBars);                   // [0..7] poisoned piece, [8] last, [9] TMEM
    long long* scratch = reinterpret_cast<long long*>(reinterpret_cast<char*>(bars) + 352);

    const int warp = int(threadIdx.x / 32), lane = threadIdx.x % 32;
    int* err = c.err;
    const Schedule<kRows, kTile> sch{c, b, a.window, group, TMA ? 1 << c.box_log : 1, a.rows_from, a.rows_to, a.check};
    const Span sp = find_span<kThreads>(sch, 4, scratch);
    if (sp.len == 0) return;
    const int G = int(group.d);

    if (threadIdx.x == 0) {
        for (int i = 0; i < NS; ++i) {
            tc::mbar_init(&bars[kTileFull + i], TMA ? 1 : kCopy / 32);
            tc::mbar_init(&bars[kFree + i], 1);
        }
        for (int t = 0; t < 2; ++t) {
            tc::mbar_init(&bars[kSFull + t], 1);
            tc::mbar_init(&bars[kSFree + t], 4);
            tc::mbar_init(&bars[kPFull + t], 4);
            tc::mbar_init(&bars[kPvDone + t], 1);
        }
        tc::mbar_init(&bars[kQFull], kCopy / 32);
        tc::mbar_init(&bars[kQFree], 1);
        tc::mbar_init(&bars[kDrain], 1);
        tc::mbar_init(&bars[kEdge], 1);
        tc::fence_barrier_init();
        for (int i = 0; i < 8; ++i) flags[i] = 0;
    }
    if (warp == kMma) {
        tc::tmem_alloc(reinterpret_cast<uint32_t*>(&flags[9]), 512);
        tc::tmem_relinquish();
    }
    tc::tc_fence_before();
    __syncthreads();
    tc::tc_fence_after();
    const uint32_t tmem = uint32_t(flags[9]);
    // TMEM columns of half t, from 256 t: S [0, SK), P [SK, SK + SK / 2), its low parts the next SK / 2, O the last D
    const auto s_col = [&](int t) { return tmem + 256 * t; };
    const auto p_col = [&](int t, int part) { return tmem + 256 * t + SK + part * (SK / 2); };
    const auto o_col = [&](int t) { return tmem + 256 * t + 256 - D; };

    if (warp >= 8 && warp < kMma) {
        // ------------------------------------------------------------------------------------------- copies
        const int tid = threadIdx.x - 256;
        const uint32_t ring0 = tc::smem_u32(ring);
        int issued = 0, piece = 0, at = 0, g0 = sp.g;
        Item it = sp.it;
        bool good = true;
        // queries of a piece, once the previous piece's products have read theirs
        const auto load_queries = [&] {
                if (piece > 0 && good) good = all_ok(tc::mbar_wait(&bars[kQFree], (piece - 1) & 1, err, kKvWait + 1));
                const int r0 = it.t * kRows;
                const auto query = [&](int r) {       // row r's query
                    const int tok = int(group.div(r0 + r));
                    return static_cast<const T*>(a.q) + (long long)(it.s.row0 + tok) * a.q_stride + (it.h * G + (r0 +
                        r - tok * G)) * D;
                };
                const auto q_off = [&](int r, int ch) { return (r / kHalf) * L::kTileBytes + image_off<D>(r % kHalf,
                    ch); };
                if constexpr (L::kSplit) {
                    // eight lanes a row, 8 values of each 16-byte chunk to a lane
                    constexpr int N = CH / 8;         // chunks of a lane
#pragma unroll 2
                    for (int r0w = (warp - 8) * 4; r0w < kRows; r0w += kCopy / 8) {
                        const int r = r0w + lane / 8;
                        const float4* src = reinterpret_cast<const float4*>(query(r < it.rows ? r : 0));
                        float4 x[N][2];
                        float top = 0.f;
#pragma unroll
                        for (int n = 0; n < N; ++n)
#pragma unroll
                            for (int e = 0; e < 2; ++e) {
                                x[n][e] = __ldg(src + (n * 8 + lane % 8) * 2 + e);
                                if (r >= it.rows) x[n][e] = make_float4(0, 0, 0, 0);
                                top = fmaxf(top, fmaxf(fmaxf(fabsf(x[n][e].x), fabsf(x[n][e].y)),
                                                       fmaxf(fabsf(x[n][e].z), fabsf(x[n][e].w))));
                            }
#pragma unroll
                        for (int o = 4; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(kFull, top, o));
                        // 2^ex brings the largest value into [2^10, 2^11)
                        const int ex = min(max(11 + 126 - int(__float_as_uint(top) >> 23), -126), 126);
                        const float by = __int_as_float((127 + ex) << 23) * (a.scale < 0.f ? -1.f : 1.f);
#pragma unroll
                        for (int n = 0; n < N; ++n) {
                            const float y[8] = {x[n][0].x * by, x[n][0].y * by, x[n][0].z * by, x[n][0].w * by,
                                                x[n][1].x * by, x[n][1].y * by, x[n][1].z * by, x[n][1].w * by};
                            uint32_t hi[4], lo[4];
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                hi[e] = pack2(y[2 * e], y[2 * e + 1], true);
                                const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&hi[e]));
                                lo[e] = pack2(y[2 * e] - h.x, y[2 * e + 1] - h.y, true);
                            }
                            char* to = q_tile + (r / kHalf) * 2 * L::kTileBytes +
                                image_off<D>(r % kHalf, n * 8 + lane % 8);
                            *reinterpret_cast<uint4*>(to) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
                            *reinterpret_cast<uint4*>(to + L::kTileBytes) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
                        }
                        if (lane % 8 == 0) row_exp[(piece & 1) * kRows + r] = int8_t(ex);
                    }
                } else {
                    if (a.scale < 0.f) {
                        // the sign goes to the queries, so that the largest product is the largest score
                        for (int u = tid; u < kRows * CH; u += kCopy) {
                            uint4 x = make_uint4(0, 0, 0, 0);
                            if (u / CH < it.rows) x = *reinterpret_cast<const uint4*>(query(u / CH) + u % CH * 8);
                            x.x ^= 0x80008000u; x.y ^= 0x80008000u; x.z ^= 0x80008000u; x.w ^= 0x80008000u;
                            *reinterpret_cast<uint4*>(q_tile + q_off(u / CH, u % CH)) = x;
                        }
                    } else {
                        const uint32_t q_at = tc::smem_u32(q_tile);
#pragma unroll 8
                        for (int u = tid; u < kRows * CH; u += kCopy) {
                            const bool ok = u / CH < it.rows;
                            cp_async16_zfill(q_at + q_off(u / CH, u % CH), query(ok ? u / CH : 0) + u % CH * 8, ok);
                        }
                        cp_async_commit();
                        cp_async_wait_group<0>();
                    }
                }
                tc::fence_proxy_async_smem();
                arrive_warp(&bars[kQFull]);
        };
        // Bits 15 and 31 of the result: one of the eight values is NaN or infinite (an exponent of all ones, which one
        // more carries into the sign's place). Values that some row must not see are checked: a product would carry
        // them there.
        const auto exponents = [](const uint4& x) {
            constexpr uint32_t one = kBf16 ? 0x00800080u : 0x04000400u, rest = 0x7fff7fffu;
            return ((x.x & rest) + one) | ((x.y & rest) + one) | ((x.z & rest) + one) | ((x.w & rest) + one);
        };
        const auto wait_free = [&] {                  // until the ring's next place is free
            if (issued >= NS) good = all_ok(good && tc::mbar_wait(&bars[kFree + issued % NS], (issued / NS - 1) & 1,
                err, kKvWait));
        };
        if constexpr (TMA) {
            // lane x of the first copying warp brings box x of a tile: 2^box_log slots of one page, one copy per 64
            // dims
            const int box = 1 << c.box_log, boxes = kTile >> c.box_log;
            int id = -1, edges = 0;
            const auto look_up = [&](int k0) {
                const int pos = k0 + lane * box;
                id = lane < boxes && pos < it.hi ? __ldg(b.tables + (long long)it.b * b.table_stride +
                    c.page.div(pos)) : -1;
            };
            const auto issue = [&](const CUtensorMap* map, int k0, int page, uint64_t* bar) {
                // (the second warp must not wait here: nothing holds it within a phase of the first)
                if (warp == 8) wait_free();
                if (good && warp == 8) {
                    const int pos = k0 + lane * box;
                    const bool mine = lane < boxes && pos < it.hi;
                    const int n = __popc(__ballot_sync(kFull, mine));
                    if (lane == 0) tc::mbar_arrive_expect_tx(bar, uint32_t(n * box * D * 2));
                    __syncwarp();
                    if (mine) {
                        const int slot = pos - int(c.page.div(pos) * c.page.d);
#pragma unroll
                        for (int h = 0; h < D / 64; ++h)
                            tma_load_5d(ring0 + issued % NS * L::kTileBytes + h * (128 * 128) + lane * box * 128, map,
                                h * 64,
                                        it.h, slot, page, c.layer, tc::smem_u32(bar));
                    }
                    __syncwarp();
                }
                ++issued;
            };
            while (at < sp.len) {                     // after a failed wait: barriers only
                const int g1 = min(it.n, g0 + sp.len - at);
                const int lo_last = a.window ? max(0, it.p1 - a.window + 1) : 0;
                const auto page_of = [&](int k0) {
                    return lane < boxes && k0 + lane * box < it.hi ? safe_page(id, c) : 0;
                };
                look_up(it.lo + g0 * kTile);
                int page = page_of(it.lo + g0 * kTile);
                issue(&maps.k, it.lo + g0 * kTile, page, &bars[kTileFull + issued % NS]);
                if (g0 + 1 < g1) look_up(it.lo + (g0 + 1) * kTile);
                load_queries();
                for (int g = g0; g < g1; ++g) {
                    const int k0 = it.lo + g * kTile, slot = issued % NS;
                    const bool edge = k0 + kTile > it.p0 + 1 || k0 < lo_last;
                    issue(&maps.v, k0, page, &bars[edge ? int(kEdge) : kTileFull + slot]);
                    if (g + 1 < g1) {                 // the next keys are on their way while the values are checked
                        page = page_of(k0 + kTile);
                        issue(&maps.k, k0 + kTile, page, &bars[kTileFull + issued % NS]);
                        if (g + 2 < g1) look_up(k0 + 2 * kTile);
                    }
                    if (edge) {
                        // some row does not see all of these values: slots past the sequence's end (whatever they hold)
                        // become zeros, and the others are checked
                        if (good) good = all_ok(tc::mbar_wait(&bars[kEdge], edges & 1, err, kKvWait + 1));
                        ++edges;
                        char* v = ring + slot * L::kTileBytes;
                        const int valid = min(kTile, it.hi - k0);
                        uint32_t seen = 0;
                        if (good) {
                            for (int i = tid + valid * CH; i < kTile * CH; i += kCopy)
                                *reinterpret_cast<uint4*>(v + image_off<D>(i / CH, i % CH)) = make_uint4(0, 0, 0, 0);
#pragma unroll 8
                            for (int i = tid; i < valid * CH; i += kCopy)
                                seen |= exponents(*reinterpret_cast<const uint4*>(v + image_off<D>(i / CH, i % CH)));
                        }
                        if (seen & 0x80008000u) flags[piece & 7] = piece + 1;
                        tc::fence_proxy_async_smem();
                        bar_copies<kCopy>();
                        if (tid == 0 && good) tc::mbar_arrive(&bars[kTileFull + slot]);
                    }
                }
                at += g1 - g0;
                g0 = 0;
                ++piece;
                if (at < sp.len) sch.next(it);
            }
        } else {
        int done = 0;
        constexpr int kLag = NS >= 5 ? 3 : 2;
        int check0 = 0, check1 = 0, check2 = 0;       // newest to oldest in flight: piece + 1 if its values are checked
        const auto complete = [&](int check) {        // the oldest tile in flight is complete for all threads
            tc::fence_proxy_async_smem();
            const int slot = done % NS;
            if (check) {
                uint32_t seen = 0;
                for (int i = 0; i < kTile * CH / kCopy; ++i) {
                    const int r = i * (kCopy / CH) + tid / CH, ch = tid % CH;
                    seen |= exponents(*reinterpret_cast<const uint4*>(ring + slot * L::kTileBytes + image_off<D>(r,
                        ch)));
                }
                if (seen & 0x80008000u) flags[(check - 1) & 7] = check;
            }
            arrive_warp(&bars[kTileFull + slot]);
            ++done;
        };
        // thread k finds keys k and k + 64 of a tile: page ids are read a tile ahead, byte offsets shared through
        // row_off (K and V lie at the same offsets); -1: no such key, filled with zeros
        int id[kTile / kCopy], pos0 = 0;
        const auto look_up = [&](int k0) {
            pos0 = k0 + tid;
#pragma unroll
            for (int i = 0; i < kTile / kCopy; ++i) {
                const int pos = pos0 + i * kCopy;
                id[i] = pos < it.hi ? __ldg(b.tables + (long long)it.b * b.table_stride + c.page.div(pos)) : -1;
            }
        };
        const auto share = [&](int buf) {
#pragma unroll
            for (int i = 0; i < kTile / kCopy; ++i) {
                const int pos = pos0 + i * kCopy;
                long long off = -1;
                if (pos < it.hi) {
                    if (unsigned(id[i]) >= unsigned(c.num_pages)) {
                        report(err, kKvBadPage);
                        id[i] = 0;
                    }
                    off = id[i] * c.page_stride + (pos - int(c.page.div(pos) * c.page.d)) * c.token_stride +
                          it.h * c.head_stride;
                }
                row_off[buf * kTile + tid + i * kCopy] = off;
            }
            bar_copies<kCopy>();
        };
        const uint32_t my_dst = image_off<D>(tid / CH, tid % CH);
        const auto issue = [&](int buf, bool values, int check) {
            wait_free();
            if (!good) return;
            const char* base = (values ? c.v : c.k) + tid % CH * 16;
            // rows kCopy / CH apart: a chunk's place repeats every 8 rows
            constexpr int kStep = kCopy / CH;
            const uint32_t dst = ring0 + (issued % NS) * L::kTileBytes + my_dst;
            const long long* offs = row_off + buf * kTile + tid / CH;
#pragma unroll
            for (int i = 0; i < kTile / kStep; ++i) {
                const long long off = offs[i * kStep];
                const uint32_t to = kStep % 8 == 0 || i % 2 == 0 ? dst : dst ^ 64;   // four rows on: chunk ^ 4
                cp_async16_zfill(to + i * kStep * 128, base + (off < 0 ? 0 : off), off >= 0);
            }
            cp_async_commit();
            check2 = check1;
            check1 = check0;
            check0 = check;
            ++issued;
            if (issued - done == kLag) {
                cp_async_wait_group<kLag - 1>();
                complete(kLag == 3 ? check2 : check1);
            }
        };
        while (at < sp.len) {                         // after a failed wait: barriers only
            const int g1 = min(it.n, g0 + sp.len - at);
            const int lo_last = a.window ? max(0, it.p1 - a.window + 1) : 0;
            for (int g = g0; g < g1; ++g) {
                const int k0 = it.lo + g * kTile;
                const bool edge = k0 + kTile > it.p0 + 1 || k0 < lo_last;
                if (g == g0) look_up(k0);
                share(g & 1);
                if (g + 1 < g1) look_up(k0 + kTile);
                issue(g & 1, false, 0);
                if (g == g0) load_queries();
                issue(g & 1, true, edge ? piece + 1 : 0);
            }
            bar_copies<kCopy>();                             // row_off is read before the next piece writes it
            at += g1 - g0;
            g0 = 0;
            ++piece;
            if (at < sp.len) sch.next(it);
        }
        cp_async_wait_group<0>();
        if (good && issued - done == 2) complete(check1);
        if (good && issued - done == 1) complete(check0);
        }
    } else if (warp >= kMma) {
        // ------------------------------------------------------------------------------------------- products
        if (warp == kMma && tc::elect_one()) {
            constexpr uint32_t id_qk = idesc_f16(kBf16, false, 128, SK), id_pv = idesc_f16(kBf16, true, 128, D);
            // low descriptor words; leading offset: unused (1) for the K-major ones, between 64-dim halves for V
            const uint32_t q0 = tc::smem_u32(q_tile) >> 4 | 1u << 16, ring0 = tc::smem_u32(ring) >> 4;
            constexpr uint32_t k_lead = 1u << 16, v_lead = (D == 64 ? 1024u : 128u * 128u) >> 4 << 16;
            int at = 0, g0 = sp.g, piece = 0, tile = 0;           // tile: ring position of the piece's first keys
            int made[2] = {0, 0}, used[2] = {0, 0};               // score tiles and weight tiles issued per half
            Item it = sp.it;
            bool good = true;
            const auto wait = [&](int bar, int parity, int code) {
                good = good && tc::mbar_wait(&bars[bar], parity & 1, err, code);
                tc::tc_fence_after();
            };
            while (at < sp.len && good) {
                const int n = min(it.n, g0 + sp.len - at) - g0, steps = n * SUB;
                const bool two = it.rows > kHalf;
                // ring positions: keys of tile j at tile + 2 j, values at tile + 2 j + 1
                const auto qk = [&](int t, int u) {               // scores of keys SK u .. of the piece
                    const int pos = tile + u / SUB * 2;
                    if (t == 0 && u % SUB == 0) wait(kTileFull + pos % NS, pos / NS, kKvWait + 3);
                    if (made[t] > 0) wait(kSFree + t, made[t] - 1, kKvWait + 4);
                    if (!good) return;
                    const uint32_t kt = (ring0 | k_lead) + (pos % NS * L::kTileBytes + u % SUB * (SK * 128)) / 16;
#pragma unroll
                    for (int part = 0; part < (L::kSplit ? 2 : 1); ++part) {
                        const uint32_t q = q0 + (t * (L::kSplit ? 2 : 1) + part) * (L::kTileBytes / 16);
#pragma unroll
                        for (int k = 0; k < D / 16; ++k) {
                            const uint32_t off = ((k / 4) * (128 * 128) + (k % 4) * 32) / 16;
                            mma_ss(s_col(t), desc_of(q + off), desc_of(kt + off), id_qk, part + k > 0);
                        }
                    }
                    tc::mma_commit(&bars[kSFull + t]);
                    ++made[t];
                    if (t == int(two)) {
                        if (u % SUB == SUB - 1) tc::mma_commit(&bars[kFree + pos % NS]);
                        if (u == steps - 1) tc::mma_commit(&bars[kQFree]);
                    }
                };
                const auto pv = [&](int t, int u) {
                    const int pos = tile + u / SUB * 2 + 1;
                    if (t == 0 && u % SUB == 0) wait(kTileFull + pos % NS, pos / NS, kKvWait + 5);
                    wait(kPFull + t, used[t], kKvWait + 6);
                    if (!good) return;
                    const uint32_t vt = (ring0 | v_lead) + (pos % NS * L::kTileBytes + u % SUB * (SK * 128)) / 16;
#pragma unroll
                    for (int part = 0; part < (L::kSplit ? 2 : 1); ++part)
#pragma unroll
                        for (int k = 0; k < SK / 16; ++k)
                            mma_ts(o_col(t), p_col(t, part) + k * 8, desc_of(vt + k * 2048 / 16), id_pv, u > 0 ||
                                part + k > 0);
                    tc::mma_commit(&bars[kPvDone + t]);
                    ++used[t];
                    if (t == int(two) && u % SUB == SUB - 1) tc::mma_commit(&bars[kFree + pos % NS]);
                };
                wait(kQFull, piece, kKvWait + 2);
                qk(0, 0);
                if (two) qk(1, 0);
                // the halves half a step apart: one's products run while the other's weights are computed
                for (int u = 0; u < steps && good; ++u) {
                    if (u + 1 < steps) qk(0, u + 1);
                    if (two && u > 0) pv(1, u - 1);
                    if (two && u + 1 < steps) qk(1, u + 1);
                    pv(0, u);
                }
                if (two && good) pv(1, steps - 1);
                tile += 2 * n;
                at += n;
                g0 = 0;
                ++piece;
                if (at < sp.len) sch.next(it);
            }
            tc::mma_commit(&bars[kDrain]);
            tc::mbar_wait(&bars[kDrain], 0, err, kKvWait + 9);
        }
    } else {
        // ------------------------------------------------------------------------------------------- rows
        const int t = warp / 4, row = t * kHalf + (warp % 4) * 32 + lane;
        const uint32_t lanes = uint32_t((warp % 4) * 32) << 16;
        int at = 0, g0 = sp.g, piece = 0, step = 0;
        Item it = sp.it;
        bool good = true;
        while (at < sp.len) {
            const int g1 = min(it.n, g0 + sp.len - at), halves = it.rows > kHalf ? 2 : 1;
            const int r0 = it.t * kRows, rr = min(row, it.rows - 1), tok = int(group.div(r0 + rr));
            const int head = it.h * G + (r0 + rr - tok * G);
            const int p = it.s.len - it.s.n + tok, first = a.window ? p - a.window + 1 : 0;
            const bool mine = t < halves && good, valid = row < it.rows && good;   // after a failed wait: barriers only
            const float sink = a.sinks ? a.sinks[head] * kLog2e : -INFINITY;
            float m = -INFINITY, l = 0.f, sc = fabsf(a.scale) * kLog2e;
            if (mine) {
                // first and last position of this half's rows: between them some tiles are partly masked
                const int pa = it.s.len - it.s.n + int(group.div(r0 + t * kHalf));
                const int pz = it.s.len - it.s.n + int(group.div(r0 + min(it.rows, (t + 1) * kHalf) - 1));
                const int lo_last = a.window ? max(0, pz - a.window + 1) : 0;
                for (int g = g0 * SUB; g < g1 * SUB && good; ++g, ++step) {
                    const int k0 = it.lo + g * SK;
                    const bool edge = k0 + SK > pa + 1 || k0 < lo_last;
                    good = all_ok(tc::mbar_wait(&bars[kSFull + t], step & 1, err, kKvWait));
                    if (!good) break;
                    tc::tc_fence_after();
                    uint32_t x[SK];
#pragma unroll
                    for (int i = 0; i < SK; i += 32)
                        tc::tmem_ld_32x32b_x32(s_col(t) + lanes + i, *reinterpret_cast<uint32_t(*)[32]>(x + i));
                    tc::tmem_ld_wait();
                    tc::tc_fence_before();
                    arrive_warp(&bars[kSFree + t]);       // the next scores may be written
                    if (L::kSplit && g == g0 * SUB) sc *= __int_as_float((127 - row_exp[(piece & 1) * kRows +
                        row]) << 23);
                    if (edge) mask<SK>(x, first - k0, p - k0);
                    float top4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                    for (int i = 0; i < SK; i += 2)
                        top4[i / 2 & 3] = max3_nan(top4[i / 2 & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    const float top = max3_nan(top4[0], top4[1], max3_nan(top4[2], top4[3], top4[3]));
                    // as the weights' own exponents are computed, and the reference rounded up: no weight is larger
                    // than meant, however large the scores
                    const bool past = fmaf(top, sc, -m) > W::kLift + W::kSlack;
                    if (__any_sync(kFull, past)) {
                        const float mm = past ? __fmaf_ru(top, sc, -W::kLift) : m, f = past ? ex2(m - mm) : 1.f;
                        if (g > g0 * SUB) {
                            good = all_ok(tc::mbar_wait(&bars[kPvDone + t], (step - 1) & 1, err, kKvWait + 1));
                            if (!good) break;
                            tc::tc_fence_after();
#pragma unroll 1
                            for (int i = 0; i < D / 16; ++i) {
                                uint32_t o[16];
                                tc::tmem_ld_32x32b_x16(o_col(t) + lanes + i * 16, o);
                                tc::tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tmem_st_x16(o_col(t) + lanes + i * 16, o);
                            }
                        }
                        m = mm;
                        l *= f;
                    }
                    const float base = m == -INFINITY ? 0.f : m;
                    if (step > 0) good = all_ok(tc::mbar_wait(&bars[kPvDone + t], (step - 1) & 1, err, kKvWait + 1));
                    if (!good) break;
                    tc::tc_fence_after();             // the products have read the previous weights
                    const uint32_t p_at = p_col(t, 0) + lanes, p_low = p_col(t, 1) + lanes;
                    // a row without a key so far needs exact zeros, and one with a score of NaN or +infinity (which make
                    // it NaN) the exponential that keeps them
                    if (L::kSplit || edge || __any_sync(kFull, m == -INFINITY || !(top * sc < INFINITY)))
                        l += weights<C, L::kSplit, false, SK>(x, sc, -base, p_at, p_low);
                    else
                        l += weights<C, L::kSplit, true, SK>(x, sc, -base, p_at, p_low);
                    tmem_st_wait();
                    tc::tc_fence_before();
                    arrive_warp(&bars[kPFull + t]);
                }
                if (good) good = all_ok(tc::mbar_wait(&bars[kPvDone + t], (step - 1) & 1, err, kKvWait + 1));
                tc::tc_fence_after();
            }
            // ---- the piece's result
            const bool whole = g0 == 0 && g1 == it.n;
            const int at_slot = 2 * blockIdx.x + (g0 > 0 ? 0 : 1);
            float* my = slots + (long long)at_slot * slot_floats<D>();
            T* dst = static_cast<T*>(a.out) + (long long)(it.s.row0 + tok) * a.out_stride + head * D;
            const auto put = [&](int d, const float (&y)[8], float inv) {     // eight finished values of this row
                if constexpr (L::kSplit) {
                    reinterpret_cast<float4*>(dst + d)[0] = make_float4(y[0] * inv, y[1] * inv, y[2] * inv, y[3] * inv);
                    reinterpret_cast<float4*>(dst + d)[1] = make_float4(y[4] * inv, y[5] * inv, y[6] * inv, y[7] * inv);
                } else {
                    *reinterpret_cast<uint4*>(dst + d) =
                        make_uint4(pack2(y[0] * inv, y[1] * inv, !kBf16), pack2(y[2] * inv, y[3] * inv, !kBf16),
                                   pack2(y[4] * inv, y[5] * inv, !kBf16), pack2(y[6] * inv, y[7] * inv, !kBf16));
                }
            };
            const auto inverse = [&](float mm, float z) {
                if (z > 0.f) z += ex2(sink - mm);
                return z == 0.f ? 0.f : 1.f / z;
            };
            if (mine && good && flags[piece & 7] == piece + 1) {
                // a value that some row must not see is NaN or infinite: the piece again, without products of masked
                // values
                const int klo = it.lo + g0 * kTile, khi = min(it.hi, it.lo + g1 * kTile);
                for (int i = 0; i < 32; ++i) {
                    const int r = t * kHalf + (warp % 4) * 32 + i;
                    if (r >= it.rows) break;
                    const int tk = int(group.div(r0 + r)), pp = it.s.len - it.s.n + tk, hd = it.h * G + (r0 +
                        r - tk * G);
                    float mm, ll, oo[D / 32];
                    careful_row<T, C, D>(c, b, a, it.b, it.h, (long long)(it.s.row0 + tk) * a.q_stride + hd * D,
                                         max(klo, a.window ? pp - a.window + 1 : 0), min(khi, pp + 1), &mm, &ll, oo);
                    float z = ll;
                    if (a.sinks && z > 0.f) z += ex2(a.sinks[hd] * kLog2e - mm);
                    const float inv = z == 0.f ? 0.f : 1.f / z;
                    for (int e = 0; e < D / 32; ++e) {
                        const int d = lane * (D / 32) + e;
                        if (whole) store_as(a.out, (long long)(it.s.row0 + tk) * a.out_stride + hd * D + d,
                            oo[e] * inv, a.type);
                        else my[d * kRows + r] = oo[e];
                    }
                    if (!whole && lane == 0) {
                        my[kRows * D + r] = mm;
                        my[kRows * D + kRows + r] = ll;
                    }
                }
            } else if (mine && good) {
                const float inv = inverse(m, l);
#pragma unroll
                for (int i = 0; i < D / 32; ++i) {
                    uint32_t o[32];
                    __syncwarp();
                    tc::tmem_ld_32x32b_x32(o_col(t) + lanes + i * 32, o);
                    tc::tmem_ld_wait();
                    if (!valid) {
                    } else if (whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            float y[8];
#pragma unroll
                            for (int k = 0; k < 8; ++k) y[k] = l == 0.f ? 0.f : __uint_as_float(o[e + k]);
                            put(i * 32 + e, y, inv);
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < 32; ++e) my[(i * 32 + e) * kRows + row] = __uint_as_float(o[e]);
                    }
                }
                if (!whole && valid) {
                    my[kRows * D + row] = m;
                    my[kRows * D + kRows + row] = l;
                }
            }
            tc::tc_fence_before();
            if (!whole) {
                const long long start = sp.start + at - g0;
                const int c0 = blockIdx.x - (start < sp.start ? ceil_div(sp.start - start, sp.per) : 0);
                const int c1 = blockIdx.x + int(unsigned(start + it.n - 1 - sp.start) / unsigned(sp.per));
                bar_rows();
                if (threadIdx.x == 0) {
                    const int n = arrive(&counters[c0]);
                    flags[8] = n == c1 - c0;
                    if (n == c1 - c0) counters[c0] = 0;
                }
                bar_rows();
                if (flags[8] && valid) {
                    float mm = -INFINITY, z = 0.f;
                    for (int i = c0; i <= c1; ++i)
                        mm = fmaxf(mm, __ldcg(slots + (long long)(2 * i + (i == c0)) * slot_floats<D>() + kRows * D +
                            row));
                    const float base = mm == -INFINITY ? 0.f : mm;
                    for (int i = c0; i <= c1; ++i) {
                        const float* ps = slots + (long long)(2 * i + (i == c0)) * slot_floats<D>() + kRows * D;
                        z += __ldcg(ps + kRows + row) * ex2(__ldcg(ps + row) - base);
                    }
                    const float inv = inverse(mm, z);
                    for (int d = 0; d < D; d += 8) {
                        float y[8] = {};
                        for (int i = c0; i <= c1; ++i) {
                            const float* ps = slots + (long long)(2 * i + (i == c0)) * slot_floats<D>();
                            const float f = ex2(__ldcg(ps + kRows * D + row) - base);
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] += __ldcg(ps + (d + e) * kRows + row) * f;
                        }
                        put(d, y, inv);
                    }
                }
                bar_rows();                           // flags[8] is read before the next piece sets it
            }
            at += g1 - g0;
            g0 = 0;
            ++piece;
            if (at < sp.len) sch.next(it);
        }
    }
    tc::tc_fence_before();
    __syncthreads();
    if (warp == kMma) tc::tmem_dealloc(tmem, 512);
}

constexpr int kMaxCtas = 160;

template <class T, class C, int D, bool TMA>
void launch(const KvMaps& maps, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws, cudaStream_t s) {
    using L = Layout<T, D, TMA>;
    static DeviceOnce once;
    int dev = 0;
    GPT_CHECK(cudaGetDevice(&dev));
    once.run(dev, [] {
        GPT_CHECK(cudaFuncSetAttribute(paged_tiles_kernel<T, C, D, TMA>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       L::kSmem));
    });
    PagedAttnArgs args = a;
    args.check = many_groups(b, c, a, kTile, kRows);
    paged_tiles_kernel<T, C, D, TMA><<<std::min(kMaxCtas, num_sms()), block_threads(TMA), L::kSmem, s>>>(
        maps, c, b, args, FastDiv::of(uint32_t(a.q_heads / c.kv_heads)), static_cast<int*>(ws),
        reinterpret_cast<float*>(static_cast<char*>(ws) + kCounterBytes));
    check_launch("paged_attention");
}

template <class T, class C, int D>
void by_copy(const KvMaps& maps, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws, cudaStream_t s) {
    if (c.box_log >= 3) launch<T, C, D, true>(maps, c, b, a, ws, s);
    else launch<T, C, D, false>(maps, c, b, a, ws, s);
}

}  // namespace

size_t paged_tiles_ws_bytes(int dim) {
    return kCounterBytes + kMaxCtas * 2 * sizeof(float) * (dim == 64 ? slot_floats<64>() : slot_floats<128>());
}

void launch_paged_tiles(const KvMaps& m, const KvView& c, const KvBatch& b, const PagedAttnArgs& a, void* ws,
                        cudaStream_t s) {
    if (c.dim == 64) {
        if (a.type == kF32) by_copy<float, __half, 64>(m, c, b, a, ws, s);
        else if (a.type == kF16) by_copy<__half, __half, 64>(m, c, b, a, ws, s);
        else by_copy<__nv_bfloat16, __nv_bfloat16, 64>(m, c, b, a, ws, s);
    } else {
        if (a.type == kF32) by_copy<float, __half, 128>(m, c, b, a, ws, s);
        else if (a.type == kF16) by_copy<__half, __half, 128>(m, c, b, a, ws, s);
        else by_copy<__nv_bfloat16, __nv_bfloat16, 128>(m, c, b, a, ws, s);
    }
}

}  // namespace gpt
