// Work items of the paged attention kernels and their split over the grid.
//
// An item is (sequence, key/value head, tile of R query rows), row = token * group + head of the group; its work is the
// key range [lo, hi) that its rows see together, in groups of UNIT keys (at least one). All items laid end to end are
// cut into one contiguous span of groups per CTA, so every CTA gets the same number of groups whatever the lengths: a
// span may begin or end inside an item. An item cut into pieces is put together by the CTA that finishes last, from the
// pieces in their order, so the result does not depend on timing. Each CTA leaves at most two pieces (the item it
// starts in and the item it ends in), which bounds the workspace by the grid alone. Every CTA finds its span itself
// from the lengths in device memory: the host needs none of them.
#pragma once
#include <algorithm>

#include "paged.cuh"

namespace gpt {
namespace paged {

struct Item {
    int b, h, t, nt;         // sequence, key/value head, row tile, the sequence's row tiles
    Seq s;
    int rows;                // valid rows of this tile
    int p0, p1;              // positions of its first and last row
    int lo, hi;              // keys any of its rows sees (lo <= hi)
    int n;                   // groups
};

// A head's groups are counted in 32 bits: n, a sequence's new tokens, or 0 (with an error word) where they would not fit.
inline __device__ __noinline__ int countable(int n, int len, int tiles, int window, int unit, int tile_rows, int* err) {
    const int keys = window ? min(len, min(window, 1 << 30) + tile_rows) : len;
    if ((long long)tiles * (keys / unit + 3) < 1ll << 31) return n;
    report(err, kKvTooMuch);
    return 0;
}
// Whether tokens and tables allow a head of 2^31 groups, or so many groups for a CTA (then the kernel looks).
inline bool many_groups(const KvBatch& b, const KvView& c, const PagedAttnArgs& a, int unit, int tile_rows) {
    const double rows = std::min(double(b.tokens) * (a.q_heads / c.kv_heads), double(a.rows_to));
    const double keys = std::min(double(b.most), a.window ? double(a.window) + tile_rows : 2147483648.0);
    return (rows / tile_rows + b.seqs) * (keys / unit + 3) * c.kv_heads >= 2147483648.0;
}

template <int R, int UNIT>
struct Schedule {
    const KvView& c;
    const KvBatch& b;
    int window;
    FastDiv group;
    int align;               // lo is a multiple of this (a power of two)
    int rows_from, rows_to;  // only sequences with so many rows (new tokens x group) have items
    bool check;              // the host could not rule out a head of 2^31 groups (many_groups)

    __device__ __forceinline__ Seq seq(int i) const {
        Seq s = load_seq(b, i, c.err);
        const int rows = s.n * int(group.d);
        if (rows < rows_from || rows > rows_to) s.n = 0;
        if (check) s.n = countable(s.n, s.len, row_tiles(s.n), window, UNIT, R, c.err);
        return s;
    }
    __device__ __forceinline__ int row_tiles(int n) const { return (n * int(group.d) + R - 1) / R; }

    __device__ __forceinline__ void fill(Item& it) const {
        const int r0 = it.t * R;
        it.rows = min(R, it.s.n * int(group.d) - r0);
        it.p0 = it.s.len - it.s.n + int(group.div(r0));
        it.p1 = it.s.len - it.s.n + int(group.div(r0 + it.rows - 1));
        it.lo = window ? max(0, max(it.p0, 0) - (window - 1)) & -align : 0;   // (p0 may be negative, window 2^31 - 1)
        it.hi = max(it.lo, it.p1 + 1);
        it.n = max(1, (it.hi - it.lo + UNIT - 1) / UNIT);
    }

    // Groups of tile t of a sequence, rounded up to a multiple of pad.
    __device__ __forceinline__ int tile_groups(const Seq& s, int t, int pad) const {
        Item it;
        it.s = s;
        it.t = t;
        fill(it);
        return pad == 1 ? it.n : (it.n + pad - 1) / pad * pad;
    }
    // Groups of one key/value head of each lane's sequence: a few tiles by the lane itself, more by the whole warp, a
    // lane per tile (64 tiles by one lane took 4 us). All lanes call it.
    __device__ __forceinline__ int head_groups(const Seq& s, int pad) const {
        const int lane = threadIdx.x % 32, nt = row_tiles(s.n);
        int sum = 0;
        if (nt <= 2)
            for (int t = 0; t < nt; ++t) sum += tile_groups(s, t, pad);
        for (unsigned many = __ballot_sync(kFull, nt > 2); many; many &= many - 1) {
            const int src = __ffs(many) - 1;
            const Seq q{__shfl_sync(kFull, s.row0, src), __shfl_sync(kFull, s.n, src), __shfl_sync(kFull, s.len, src)};
            int part = 0;
            for (int t = lane; t < row_tiles(q.n); t += 32) part += tile_groups(q, t, pad);
            part = __reduce_add_sync(kFull, part);
            if (lane == src) sum = part;
        }
        return sum;
    }
    // The tile of the item's head that holds group `off` of it; off becomes the group within the tile. All lanes call
    // it.
    __device__ __forceinline__ void find_tile(Item& it, int& off, int pad) const {
        const int lane = threadIdx.x % 32;
        for (int t0 = 0;; t0 += 32) {
            const int n = t0 + lane < it.nt ? tile_groups(it.s, t0 + lane, pad) : 0;
            int end = n;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(kFull, end, o);
                if (lane >= o) end += y;
            }
            const unsigned holds = __ballot_sync(kFull, off < end);
            if (holds || t0 + 32 >= it.nt) {
                const int src = holds ? __ffs(holds) - 1 : 0;
                it.t = t0 + src;
                off -= __shfl_sync(kFull, end - n, src);
                break;
            }
            off -= __shfl_sync(kFull, end, 31);
        }
        fill(it);
    }

    // First item at or after (b, 0, 0); false past the last sequence.
    __device__ __forceinline__ bool open(Item& it, int i) const {
        for (; i < b.seqs; ++i) {
            it.s = seq(i);
            it.nt = row_tiles(it.s.n);
            if (it.nt > 0) {
                it.b = i;
                it.h = it.t = 0;
                fill(it);
                return true;
            }
        }
        it.b = b.seqs;
        it.n = 0x7fffffff;
        return false;
    }
    __device__ __forceinline__ void next(Item& it) const {
        if (++it.t < it.nt) {
            fill(it);
        } else if (++it.h < c.kv_heads) {
            it.t = 0;
            fill(it);
        } else {
            open(it, it.b + 1);
        }
    }
    // Steps k groups on from group g of the item.
    __device__ __forceinline__ void step(Item& it, int& g, int k) const {
        g += k;
        while (g >= it.n && it.b < b.seqs) {
            g -= it.n;
            next(it);
        }
    }
};

// What a CTA works on: groups [start, start + len) of all, `per` groups per CTA; the item and group it starts in.
struct Span {
    long long start;
    int len, per, g;
    Item it;
};

__device__ __forceinline__ int ceil_div(long long a, int b) {
    return a >> 31 ? int((a + b - 1) / b) : int((unsigned(a) + unsigned(b) - 1) / unsigned(b));
}

// Sum over the block in thread order and each thread's exclusive prefix; NT threads, two barriers.
template <int NT>
__device__ __forceinline__ long long block_prefix(long long v, long long* warp_sums, long long* total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    long long before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < NT / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return before + x - v;
}

// Whether a CTA's share of all groups would not fit.
inline __device__ __noinline__ bool too_much(long long total, int grid, int* err) {
    if (total >> 30 < grid) return false;
    report(err, kKvTooMuch);
    return true;
}

// Finds this CTA's span; all NT threads call it. scratch: NT / 32 + 2 words of shared memory.
//
// With few items (an eighth of the grid at most) a span never crosses from one item into the next: items are laid out
// padded to whole spans of `per` groups, per = total / (grid - items), which costs at most a seventh of the grid and
// saves the CTAs in between a second item's fixed cost (4K positions, 8 heads, one token: 17.9 us with spans cut
// anywhere, 14.2 us without). least: the fewest groups worth a CTA of its own then.
template <int NT, int R, int UNIT>
__device__ __forceinline__ Span find_span(const Schedule<R, UNIT>& sch, int least, long long* scratch) {
    const int seqs = sch.b.seqs, kvh = sch.c.kv_heads, grid = int(gridDim.x);
    Span sp;
    sp.g = 0;
    if (seqs <= 32) {                                 // each warp for itself, a lane per sequence
        const int lane = threadIdx.x % 32;
        Seq s{0, 0, 0};
        if (lane < seqs) s = sch.seq(lane);
        int units = sch.head_groups(s, 1);
        long long total = (long long)units * kvh;
        int items = sch.row_tiles(s.n) * kvh;
#pragma unroll
        for (int o = 16; o; o >>= 1) {
            total += __shfl_xor_sync(kFull, total, o);
            items += __shfl_xor_sync(kFull, items, o);
        }
        const bool whole = items * 8 <= grid;
        if (sch.check && too_much(total, grid, sch.c.err)) total = 0;
        sp.per = whole ? max(least, ceil_div(total, grid - items)) : ceil_div(total, grid);
        sp.start = (long long)blockIdx.x * sp.per;
        sp.len = 0;
        if (sp.per == 0) return sp;
        const int pad = whole ? sp.per : 1;
        if (whole) units = sch.head_groups(s, pad);
        const long long mine = (long long)units * kvh;
        long long end = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const long long y = __shfl_up_sync(kFull, end, o);
            if (lane >= o) end += y;
        }
        const unsigned holds = __ballot_sync(kFull, sp.start >= end - mine && sp.start < end);
        if (holds == 0) return sp;
        const int src = __ffs(holds) - 1;
        total = __shfl_sync(kFull, end, 31);
        const long long in_seq = sp.start - __shfl_sync(kFull, end - mine, src);
        units = __shfl_sync(kFull, units, src);
        Item& it = sp.it;
        it.b = src;
        it.s = {__shfl_sync(kFull, s.row0, src), __shfl_sync(kFull, s.n, src), __shfl_sync(kFull, s.len, src)};
        it.nt = sch.row_tiles(it.s.n);
        it.h = in_seq >> 31 ? int(in_seq / units) : int(unsigned(in_seq) / unsigned(units));
        int off = int(in_seq - (long long)it.h * units);
        sch.find_tile(it, off, pad);
        sp.g = off;
        sp.len = whole ? min(sp.per, it.n - off) : int(min((long long)sp.per, total - sp.start));
        return sp;
    }
    long long total = 0, mine = 0, before = 0;
    for (int i0 = 0; i0 < seqs; i0 += NT) {
        const int i = i0 + threadIdx.x;
        mine = (long long)sch.head_groups(i < seqs ? sch.seq(i) : Seq{0, 0, 0}, 1) * kvh;
        long long sum;
        before = total + block_prefix<NT>(mine, scratch, &sum);
        total += sum;
    }
    if (sch.check && too_much(total, grid, sch.c.err)) total = 0;
    sp.per = ceil_div(total, grid);
    sp.start = (long long)blockIdx.x * sp.per;
    sp.len = int(max(0ll, min((long long)sp.per, total - sp.start)));
    if (sp.len == 0) return sp;
    // the sequence that holds group `start`: its thread knows the prefix (with many sequences, a second pass)
    long long* found = scratch + NT / 32;
    if (seqs > NT) {
        long long base = 0;
        for (int i0 = 0; i0 < seqs; i0 += NT) {
            const int i = i0 + threadIdx.x;
            mine = (long long)sch.head_groups(i < seqs ? sch.seq(i) : Seq{0, 0, 0}, 1) * kvh;
            long long sum;
            before = base + block_prefix<NT>(mine, scratch, &sum);
            base += sum;
            if (sp.start >= before && sp.start < before + mine) {
                found[0] = i;
                found[1] = before;
            }
        }
    } else if (sp.start >= before && sp.start < before + mine) {
        found[0] = threadIdx.x;
        found[1] = before;
    }
    __syncthreads();
    sch.open(sp.it, int(found[0]));
    const long long in_seq = sp.start - found[1];
    const int per_head = sch.head_groups(sp.it.s, 1);
    sp.it.h = in_seq >> 31 ? int(in_seq / per_head) : int(unsigned(in_seq) / unsigned(per_head));
    int off = int(in_seq - (long long)sp.it.h * per_head);
    sch.find_tile(sp.it, off, 1);
    sp.g = off;
    return sp;
}

// One query row over keys [k0, k1) of a sequence, by one warp, in plain fp32 arithmetic and with masked keys never
// multiplied: the path taken when a value that some row of a tile must not see is NaN or infinite (a matrix product
// would carry it into every row as 0 * NaN). m (base-2 logarithm), l and o (dims lane * E ..) are left unnormalised.
template <class T, class C, int D>
__device__ __noinline__ void careful_row(const KvView& c, const KvBatch& b, const PagedAttnArgs& a, int seq, int kh,
                                         long long q_at, int lo, int hi, float* m_out, float* l_out, float* o_out) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x % 32;
    float q[E], o[E] = {};
    for (int e = 0; e < E; ++e) q[e] = to_f32(static_cast<const T*>(a.q)[q_at + lane * E + e]);
    const float sc = a.scale * 1.4426950408889634f;
    float m = -INFINITY, z = 0.f;
    for (int j = lo; j < hi; ++j) {
        const int pg = c.page.div(j);
        const int id = safe_page(b.tables[(long long)seq * b.table_stride + pg], c);
        const long long off = id * c.page_stride + (j - pg * int(c.page.d)) * c.token_stride + kh * c.head_stride;
        const C* k = reinterpret_cast<const C*>(c.k + off) + lane * E;
        const C* v = reinterpret_cast<const C*>(c.v + off) + lane * E;
        float x = 0.f;
        for (int e = 0; e < E; ++e) x += q[e] * to_f32(k[e]);
        x = warp_sum(x) * sc;
        const float mm = fmaxf(m, x);
        const float f = mm == -INFINITY ? 1.f : exp2f(m - mm), w = x == -INFINITY ? 0.f : exp2f(x - mm);
        z = z * f + w;
        for (int e = 0; e < E; ++e) o[e] = o[e] * f + w * to_f32(v[e]);
        m = mm;
    }
    *m_out = m;
    *l_out = z;
    for (int e = 0; e < E; ++e) o_out[e] = o[e];
}

}  // namespace paged
}  // namespace gpt
