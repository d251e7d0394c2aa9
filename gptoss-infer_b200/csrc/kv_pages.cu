// Pages of the paged cache: fork (reorder, share, grow and free sequences with reference counts) and compaction.
//
// fork:    refs' = refs - (references from the given tables) + (references from the children's tables). A child shares
//          its parent's full pages. A part-filled last page to which no reference would be left (the given tables'
//          dropped, the children's full pages counted) stays with the first child of the sequences that hold it; every
//          other child gets a copy in a fresh page, in all layers. Fresh pages are the lowest free ones (count 0 after
//          that), in the order of the children. So a page that is copied from always keeps a reference and is never a
//          fresh page of the same call: the copies may run in any order.
// compact: live pages (count > 0) at or past the number of live pages move into the free pages below it, both in
//          ascending order, so sources and destinations never overlap.
//
// The counting is whole-number arithmetic: atomics in any order give the same result.
//
// Bound: the copied pages' bytes, read and written; for a few beams, latency. Each is one cooperative launch whose
// phases are separated by grid-wide barriers (four launches in a row took 23.9 us for a fork of four beams, most of it
// on the host): fork counts references into a zeroed array, one CTA then gives out the free pages (8192 a step), and
// all CTAs copy; compact plans on one CTA, then all copy and rewrite the tables.
#include <algorithm>

#include "paged.cuh"
#include "kernels.h"
#include "tc.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kThreads = 512, kPer = 16, kScan = kThreads * kPer;    // pages of a scan step

constexpr int kNoChild = 0x7fffffff;

size_t up256(size_t n) { return (n + 255) / 256 * 256; }

// All CTAs of a cooperative launch meet. Bounded; after a wait that gave up the error word is set and the kernel goes
// on (the arrays it reads are within bounds whatever they hold). The last to arrive sets the arrivals back to 0 and
// lets the others go by a new number, so launches of any size follow one another.
__device__ __forceinline__ void grid_barrier(int* barrier, int* err) {
    __syncthreads();
    if (threadIdx.x == 0) {
        const auto number = [&] {
            int n;
            asm volatile("ld.acquire.gpu.global.s32 %0, [%1];" : "=r"(n) : "l"(barrier + 1) : "memory");
            return n;
        };
        const int before = number();
        if (arrive(barrier) == int(gridDim.x) - 1) {
            barrier[0] = 0;
            arrive(barrier + 1);
        } else {
            uint32_t i = 0;
            while (number() == before && i < tc::kSpinLimit) ++i;
            if (i == tc::kSpinLimit) report(err, kKvWait + 9);
        }
    }
    __syncthreads();
}

// Exclusive prefix sum over the block; *total gets the sum. Three barriers.
template <class V>
__device__ __forceinline__ V block_scan(V v, V* warp_sums, V* total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    V x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const V y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    V before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += warp_sums[w];
        all += warp_sums[w];
    }
    *total = all;
    return before + x - v;
}

__device__ __forceinline__ int pages_of(int len, int page) {
    return int((unsigned(len) + unsigned(page) - 1) / unsigned(page));        // (len may be close to 2^31)
}

// Copies the pages of `moves` in all layers, K and V: pieces of 32 KB, one per CTA and step, four 16-byte loads of a
// thread in flight. Where a page is one run of memory (slot-major or head-major without gaps) a piece is a part of the
// run, otherwise rows.
__device__ __forceinline__ void copy_pages(const KvPages& p, int n, const int2* moves) {
    const int rows = p.page_size * p.kv_heads, chunks = p.row_bytes / 16;
    const bool run = (p.head_stride == p.row_bytes && p.token_stride == (long long)p.row_bytes * p.kv_heads) ||
                     (p.token_stride == p.row_bytes && p.head_stride == (long long)p.row_bytes * p.page_size);
    const long long total = (long long)rows * chunks;               // 16-byte chunks of a page
    constexpr int kPiece = kThreads * 4;
    const long long pieces = (total + kPiece - 1) / kPiece;
    const long long work = n * 2ll * p.layers * pieces;
    for (long long it = blockIdx.x; it < work; it += gridDim.x) {
        const long long mv = it / pieces;
        const int piece = int(it - mv * pieces), plane = int(mv % (2 * p.layers)), m = int(mv / (2 * p.layers));
        const int2 move = __ldcg(moves + m);
        char* base = (plane & 1 ? p.v : p.k) + (plane >> 1) * p.layer_stride;
        const char* src = base + move.x * p.page_stride;
        char* dst = base + move.y * p.page_stride;
        uint4 x[4];
        long long off[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const long long u = (long long)piece * kPiece + i * kThreads + threadIdx.x;
            if (run) {
                off[i] = u * 16;
            } else {
                const int row = int(u / chunks), h = row % p.kv_heads, t = row / p.kv_heads;
                off[i] = t * p.token_stride + h * p.head_stride + u % chunks * 16;
            }
            if (u < total) x[i] = __ldcs(reinterpret_cast<const uint4*>(src + off[i]));
            else off[i] = -1;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (off[i] >= 0) __stcs(reinterpret_cast<uint4*>(dst + off[i]), x[i]);
    }
}

__global__ void __launch_bounds__(kThreads, 2) kv_fork_kernel(KvPages p, ForkArgs a, PageWs w) {
    __shared__ int sums[kThreads / 32];
    __shared__ long long wide_sums[kThreads / 32];
    const long long step = (long long)gridDim.x * kThreads, t0 = (long long)blockIdx.x * kThreads + threadIdx.x;
    // --- references dropped and added (full pages), the first child of each part-filled last page
    for (long long i = t0, n = (long long)a.seqs * a.stride; i < n; i += step) {
        const int s = int(i / a.stride), j = int(i - (long long)s * a.stride);
        if (j >= pages_of(safe_len(a.lens[s], a.most, p.err), p.page_size)) continue;
        const int id = a.tables[i];
        if (unsigned(id) < unsigned(p.num_pages)) atomicSub(&w.delta[id], 1);
        else report(p.err, kKvBadPage);
    }
    for (long long i = t0, n = (long long)a.children * a.stride; i < n; i += step) {
        const int m = int(i / a.stride), j = int(i - (long long)m * a.stride), par = a.parents[m];
        int id = -1;
        if (par >= 0 && par < a.seqs && j < safe_len(a.lens[par], a.most, p.err) / p.page_size) {
            id = a.tables[(long long)par * a.stride + j];
            if (unsigned(id) < unsigned(p.num_pages)) atomicAdd(&w.delta[id], 1);
        }
        a.tables_out[i] = id;
    }
    for (long long m = step - 1 - t0; m < a.children; m += step) {      // by the threads that have no table entries
        const int par = a.parents[m];
        if (par >= 0 && par < a.seqs) {
            const int len = safe_len(a.lens[par], a.most, p.err);
            if (len % p.page_size == 0) continue;
            const int id = a.tables[(long long)par * a.stride + len / p.page_size];
            if (unsigned(id) < unsigned(p.num_pages)) atomicMin(&w.first[id], int(m));
        } else if (par != -1) {
            report(p.err, kKvBadParent);
        }
    }
    grid_barrier(w.barrier, p.err);
    if (blockIdx.x == 0) {
        // --- the last pages that stay (only a page's first child looks at its count here, and adds to it)
        for (int m = threadIdx.x; m < a.children; m += kThreads) {
            const int par = a.parents[m];
            if (par < 0 || par >= a.seqs) continue;
            const int len = safe_len(a.lens[par], a.most, p.err), full = len / p.page_size;
            if (len % p.page_size == 0) continue;
            const int id = a.tables[(long long)par * a.stride + full];
            if (unsigned(id) < unsigned(p.num_pages) && __ldcg(&w.first[id]) == m &&
                a.refs[id] + __ldcg(&w.delta[id]) == 0) {
                atomicAdd(&w.delta[id], 1);
                a.tables_out[(long long)m * a.stride + full] = id;
            }
        }
        __syncthreads();
        // --- new counts, free pages in ascending order
        int free_pages = 0;
        for (int i0 = 0; i0 < p.num_pages; i0 += kScan) {
            const int i = i0 + threadIdx.x * kPer;
            unsigned is_free = 0;
            int r[kPer];
#pragma unroll
            for (int e = 0; e < kPer; ++e) r[e] = i + e < p.num_pages ? a.refs[i + e] : 1;
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (i + e < p.num_pages) r[e] += __ldcg(&w.delta[i + e]);
#pragma unroll
            for (int e = 0; e < kPer; ++e)
                if (i + e < p.num_pages) {
                    w.delta[i + e] = 0;
                    a.refs_out[i + e] = r[e];
                    is_free |= unsigned(r[e] == 0) << e;
                }
            int total;
            int at = free_pages + block_scan(__popc(is_free), sums, &total);
            for (unsigned f = is_free; f; f &= f - 1) w.free_page[at++] = i + __ffs(f) - 1;
            free_pages += total;
        }
        __syncthreads();
        // --- fresh pages, in the order of the children (what they ask for together may pass 2^31)
        long long used = 0;
        int copies = 0;
        for (int m0 = 0; m0 < a.children; m0 += kThreads) {
            const int m = m0 + threadIdx.x;
            int have = 0, want_len = 0, src = -1;
            if (m < a.children) {
                const int par = a.parents[m];
                if (par >= 0 && par < a.seqs) {
                    const int len = safe_len(a.lens[par], a.most, p.err);
                    have = len / p.page_size;
                    if (len % p.page_size) {
                        const int id = a.tables[(long long)par * a.stride + have];
                        if (unsigned(id) < unsigned(p.num_pages)) {
                            w.first[id] = kNoChild;
                            if (__ldcg(&a.tables_out[(long long)m * a.stride + have]) >= 0) ++have;
                            else src = id;
                        } else {
                            report(p.err, kKvBadPage);
                        }
                    }
                    const long long want = (long long)len + (a.extra ? max(a.extra[m], 0) : 0);
                    if (want > a.most) report(p.err, kKvBadLength);
                    want_len = int(min(want, (long long)a.most));
                }
            }
            const int n = max(0, pages_of(want_len, p.page_size) - have);
            long long total;
            int total_copies;
            const long long at = used + block_scan((long long)n, wide_sums, &total);
            const int got = int(max(0ll, min((long long)n, free_pages - at)));
            const bool copy = src >= 0 && got > 0;
            const int slot = copies + block_scan(int(copy), sums, &total_copies);
            if (m < a.children) {
                if (got < n) report(p.err, kKvOutOfPages);
                for (int i = 0; i < got; ++i) {
                    const int id = w.free_page[at + i];
                    a.tables_out[(long long)m * a.stride + have + i] = id;
                    a.refs_out[id] = 1;
                }
                a.lens_out[m] = got < n ? int(min((long long)want_len, (long long)(have +
                    got) * p.page_size)) : want_len;
                if (copy) w.moves[slot] = make_int2(src, w.free_page[at]);
            }
            used += total;
            copies += total_copies;
        }
        if (threadIdx.x == 0) *w.count = copies;
    }
    grid_barrier(w.barrier, p.err);
    copy_pages(p, __ldcg(w.count), w.moves);
}

__global__ void __launch_bounds__(kThreads, 2) kv_compact_kernel(KvPages p, CompactArgs a, PageWs w) {
    __shared__ int sums[kThreads / 32];
    if (blockIdx.x == 0) {
        int live = 0;
        for (int i = threadIdx.x; i < p.num_pages; i += kThreads) live += a.refs[i] > 0;
        int total;
        block_scan(live, sums, &total);
        live = total;
        // holes below the live count and live pages from it on, both in ascending order: as many of the one as of the
        // other
        int holes = 0, movers = 0;
        for (int i0 = 0; i0 < p.num_pages; i0 += kScan) {
            const int i = i0 + threadIdx.x * kPer;
            unsigned hole = 0, mover = 0;
#pragma unroll
            for (int e = 0; e < kPer; ++e) {
                const int r = i + e < p.num_pages ? a.refs[i + e] : 0;
                if (i + e < p.num_pages) a.remap[i + e] = r > 0 ? i + e : -1;
                if (i + e < live) hole |= unsigned(r <= 0) << e;
                else mover |= unsigned(r > 0) << e;
            }
            int n_holes, n_movers;
            int at = holes + block_scan(__popc(hole), sums, &n_holes);
            for (; hole; hole &= hole - 1) w.moves[at++].y = i + __ffs(hole) - 1;
            at = movers + block_scan(__popc(mover), sums, &n_movers);
            for (; mover; mover &= mover - 1) w.moves[at++].x = i + __ffs(mover) - 1;
            holes += n_holes;
            movers += n_movers;
        }
        __syncthreads();
        // counts: the movers' go to their holes; pages past the live count are free
        if (a.refs_out != a.refs)
            for (int i = threadIdx.x; i < min(live, p.num_pages); i += kThreads) a.refs_out[i] = max(a.refs[i], 0);
        __syncthreads();
        for (int i = threadIdx.x; i < movers; i += kThreads) {
            const int2 v = w.moves[i];
            a.remap[v.x] = v.y;
            a.refs_out[v.y] = a.refs[v.x];
        }
        __syncthreads();
        for (int i = live + threadIdx.x; i < p.num_pages; i += kThreads) a.refs_out[i] = 0;
        if (threadIdx.x == 0) {
            *w.count = movers;
            *a.live = live;
        }
    }
    grid_barrier(w.barrier, p.err);
    const long long n = (long long)a.seqs * a.stride;
    for (long long i = (long long)blockIdx.x * kThreads + threadIdx.x; i < n; i += (long long)gridDim.x * kThreads) {
        const int s = int(i / a.stride), j = int(i - (long long)s * a.stride);
        int id = -1;
        if (j < pages_of(safe_len(a.lens[s], a.most, p.err), p.page_size)) {
            const int old = a.tables[i];
            if (unsigned(old) < unsigned(p.num_pages)) id = __ldcg(a.remap + old);
            else report(p.err, kKvBadPage);
        }
        a.tables_out[i] = id;
    }
    copy_pages(p, __ldcg(w.count), w.moves);
}

__global__ void init_first_kernel(int* first, int n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) first[i] = kNoChild;
}

// CTAs for so many table entries and bytes of pages that may have to be copied.
int grid_for(long long entries, long long bytes) {
    const long long want = std::max((entries + 2 * kThreads - 1) / (2 * kThreads), (bytes + 32767) / 32768);
    return int(std::min<long long>(2 * num_sms(), std::max<long long>(1, want)));
}
long long page_bytes(const KvPages& p) { return 2ll * p.layers * p.page_size * p.kv_heads * p.row_bytes; }

}  // namespace

size_t kv_pages_ws_bytes(int num_pages) {
    return 256 + 3 * up256(size_t(num_pages) * 4) + size_t(num_pages) * 8;
}

PageWs make_kv_pages_ws(void* ws, int num_pages) {
    char* p = static_cast<char*>(ws);
    PageWs w;
    w.barrier = reinterpret_cast<int*>(p);
    w.count = reinterpret_cast<int*>(p + 128);
    w.delta = reinterpret_cast<int*>(p += 256);
    w.free_page = reinterpret_cast<int*>(p += up256(size_t(num_pages) * 4));
    w.first = reinterpret_cast<int*>(p += up256(size_t(num_pages) * 4));
    w.moves = reinterpret_cast<int2*>(p + up256(size_t(num_pages) * 4));
    init_first_kernel<<<std::min(1024, (num_pages + 255) / 256), 256>>>(w.first, num_pages);
    check_launch("kv_pages workspace");
    return w;
}

void launch_kv_fork(const KvPages& p, const ForkArgs& a, const PageWs& w, cudaStream_t s) {
    const int grid = grid_for((long long)std::max(a.seqs, a.children) * a.stride, a.children * page_bytes(p));
    KvPages pp = p;
    ForkArgs aa = a;
    PageWs ww = w;
    void* args[] = {&pp, &aa, &ww};
    GPT_CHECK(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kv_fork_kernel), dim3(grid), dim3(kThreads),
        args, 0, s));
}

void launch_kv_compact(const KvPages& p, const CompactArgs& a, const PageWs& w, cudaStream_t s) {
    const int grid = grid_for((long long)a.seqs * a.stride, p.num_pages * page_bytes(p) / 4);
    KvPages pp = p;
    CompactArgs aa = a;
    PageWs ww = w;
    void* args[] = {&pp, &aa, &ww};
    GPT_CHECK(cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(kv_compact_kernel), dim3(grid),
        dim3(kThreads), args, 0, s));
}

}  // namespace gpt
