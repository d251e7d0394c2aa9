// Pages of the paged cache: fork (reorder, share, grow and free sequences with reference counts) and compaction.
//
// fork:    refs' = refs - (references from the given tables) + (references from the children's tables). A child shares
//          its parent's full pages. A part-filled last page stays with the parent's first child if nobody else holds it
//          (its count was 1), and is copied into a fresh page for every other child, in all layers. Fresh pages are the
//          lowest free ones (count 0 after the given tables' references and the children's shared ones are counted), in
//          the order of the children.
// compact: live pages (count > 0) at or past the number of live pages move into the free pages below it, both in
//          ascending order, so sources and destinations never overlap.
//
// The counting is whole-number arithmetic: atomics in any order give the same result.
#include <algorithm>

#include "paged.cuh"

namespace gpt {
namespace {

using namespace paged;

constexpr int kScan = 1024;

// Workspace words: [0] copies, [1] live pages / holes; then per-page ranks or moves, then per-child words.
struct PageWs {
    int* head;
    int* page;               // free list, or movers' destinations
    int2* moves;             // (source, destination)
    int* first;              // first child of each parent is found through the children's own words
    int4* child;             // per child: base length, kept pages, wanted pages, last page or -1
};

__host__ __device__ inline PageWs carve(void* ws, int num_pages, int children) {
    char* p = static_cast<char*>(ws);
    PageWs w;
    w.head = reinterpret_cast<int*>(p);
    p += 256;
    w.page = reinterpret_cast<int*>(p);
    p += (size_t(num_pages) * 4 + 255) / 256 * 256;
    w.moves = reinterpret_cast<int2*>(p);
    p += (size_t(num_pages > children ? num_pages : children) * 8 + 255) / 256 * 256;
    w.child = reinterpret_cast<int4*>(p);
    p += (size_t(children) * 16 + 255) / 256 * 256;
    w.first = reinterpret_cast<int*>(p);
    return w;
}

// Exclusive prefix sum over a block of kScan threads; *total gets the sum. Two barriers.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(kFull, x, o);
        if (lane >= o) x += y;
    }
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(kFull, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    const int before = warp ? warp_sums[warp - 1] : 0;
    *total = warp_sums[31];
    return before + x - v;
}

__device__ __forceinline__ int pages_of(int len, int page) { return (len + page - 1) / page; }

__device__ __forceinline__ int table_len(const int* lens, int i, int stride, int page, int* err) {
    const int len = lens[i];
    const long long cap = (long long)stride * page;
    if (len < 0 || len > cap) {
        report(err, kKvBadLength);
        return len < 0 ? 0 : int(cap);
    }
    return len;
}

__global__ void fork_counts_kernel(KvPages p, ForkArgs a, void* ws, int pass) {
    const PageWs w = carve(ws, p.num_pages, a.children);
    const long long stride = (long long)gridDim.x * blockDim.x, t0 = (long long)blockIdx.x * blockDim.x + threadIdx.x;
    if (pass == 0) {
        if (a.refs_out != a.refs)
            for (long long i = t0; i < p.num_pages; i += stride) a.refs_out[i] = a.refs[i];
        for (long long m = t0; m < a.children; m += stride) {
            // the first child of each parent: the lowest m among those that name it
            const int par = a.parents[m];
            int4 c = make_int4(0, 0, 0, -1);
            if (par >= a.seqs || par < -1) report(p.err, kKvBadParent);
            if (par >= 0 && par < a.seqs) {
                const int len = table_len(a.lens, par, a.stride, p.page_size, p.err), full = len / p.page_size;
                bool first = true;
                for (int i = 0; i < m; ++i) first = first && a.parents[i] != par;
                c.x = len;
                c.y = full;
                if (len % p.page_size) {
                    const int id = a.tables[(long long)par * a.stride + full];
                    if (unsigned(id) >= unsigned(p.num_pages)) report(p.err, kKvBadPage);
                    else if (first && a.refs[id] == 1) c.y = full + 1;
                    else c.w = id;
                }
                long long want = (long long)len + (a.extra ? max(a.extra[m], 0) : 0);
                const long long cap = (long long)a.stride * p.page_size;
                if (want > cap) {
                    report(p.err, kKvBadLength);
                    want = cap;
                }
                c.z = int(want);
            }
            w.child[m] = c;
        }
        return;
    }
    const long long n_in = (long long)a.seqs * a.stride, n_out = (long long)a.children * a.stride;
    for (long long i = t0; i < n_in; i += stride) {
        const int s = int(i / a.stride), j = int(i % a.stride);
        if (j >= pages_of(table_len(a.lens, s, a.stride, p.page_size, p.err), p.page_size)) continue;
        const int id = a.tables[i];
        if (unsigned(id) < unsigned(p.num_pages)) atomicSub(&a.refs_out[id], 1);
        else report(p.err, kKvBadPage);
    }
    for (long long i = t0; i < n_out; i += stride) {
        const int m = int(i / a.stride), j = int(i % a.stride);
        int id = -1;
        if (j < w.child[m].y) {
            id = a.tables[(long long)a.parents[m] * a.stride + j];
            if (unsigned(id) < unsigned(p.num_pages)) atomicAdd(&a.refs_out[id], 1);
        }
        a.tables_out[i] = id;
    }
}

__global__ void __launch_bounds__(kScan) fork_alloc_kernel(KvPages p, ForkArgs a, void* ws) {
    __shared__ int sums[32];
    const PageWs w = carve(ws, p.num_pages, a.children);
    int free_pages = 0;
    for (int i0 = 0; i0 < p.num_pages; i0 += kScan) {
        const int i = i0 + threadIdx.x;
        const bool f = i < p.num_pages && a.refs_out[i] == 0;
        int total;
        const int at = block_scan(f, sums, &total);
        if (f) w.page[free_pages + at] = i;
        free_pages += total;
        __syncthreads();
    }
    int used = 0, copies = 0;
    for (int m0 = 0; m0 < a.children; m0 += kScan) {
        const int m = m0 + threadIdx.x;
        int4 c = m < a.children ? w.child[m] : make_int4(0, 0, 0, -1);
        const int want = pages_of(c.z, p.page_size), n = max(0, want - c.y);
        int total;
        const int at = used + block_scan(n, sums, &total);
        __syncthreads();
        const int got = max(0, min(n, free_pages - at));
        const bool copy = c.w >= 0 && got > 0;
        int total_copies;
        const int slot = copies + block_scan(copy, sums, &total_copies);
        if (m < a.children) {
            if (got < n) report(p.err, kKvOutOfPages);
            for (int i = 0; i < got; ++i) {
                const int id = w.page[at + i];
                a.tables_out[(long long)m * a.stride + c.y + i] = id;
                a.refs_out[id] = 1;
            }
            a.lens_out[m] = got < n ? min((long long)c.z, (long long)(c.y + got) * p.page_size) : c.z;
            if (copy) w.moves[slot] = make_int2(c.w, w.page[at]);
        }
        used += total;
        copies += total_copies;
        __syncthreads();
    }
    if (threadIdx.x == 0) w.head[0] = copies;
}

// One CTA column per (layer, K or V); rows of row_bytes (128 or 256), 16 bytes per thread.
__global__ void copy_pages_kernel(KvPages p, const int* count, const int2* moves) {
    const int n = *count, chunks = p.row_bytes / 16;
    const long long per_page = (long long)p.page_size * p.kv_heads * chunks;
    const int plane = blockIdx.y, layer = plane >> 1;
    char* base = (plane & 1 ? p.v : p.k) + layer * p.layer_stride;
    for (int i = blockIdx.x; i < n; i += gridDim.x) {
        const char* src = base + moves[i].x * p.page_stride;
        char* dst = base + moves[i].y * p.page_stride;
        for (long long u = threadIdx.x; u < per_page; u += blockDim.x) {
            const int c = int(u % chunks), h = int(u / chunks % p.kv_heads), t = int(u / chunks / p.kv_heads);
            const long long off = t * p.token_stride + h * p.head_stride + c * 16;
            *reinterpret_cast<uint4*>(dst + off) = *reinterpret_cast<const uint4*>(src + off);
        }
    }
}

__global__ void __launch_bounds__(kScan) compact_plan_kernel(KvPages p, CompactArgs a, void* ws) {
    __shared__ int sums[32];
    const PageWs w = carve(ws, p.num_pages, 0);
    int live = 0;
    for (int i0 = 0; i0 < p.num_pages; i0 += kScan) {
        const int i = i0 + threadIdx.x;
        int total;
        block_scan(i < p.num_pages && a.refs[i] > 0, sums, &total);
        live += total;
        __syncthreads();
    }
    int holes = 0;
    for (int i0 = 0; i0 < live; i0 += kScan) {
        const int i = i0 + threadIdx.x;
        const bool f = i < live && a.refs[i] <= 0;
        int total;
        const int at = holes + block_scan(f, sums, &total);
        if (f) w.moves[at].y = i;
        holes += total;
        __syncthreads();
    }
    int movers = 0;
    for (int i0 = live; i0 < p.num_pages; i0 += kScan) {
        const int i = i0 + threadIdx.x;
        const int r = i < p.num_pages ? a.refs[i] : 0;
        int total;
        const int at = movers + block_scan(r > 0, sums, &total);
        if (r > 0) w.moves[at].x = i;
        movers += total;
        __syncthreads();
    }
    for (int i = threadIdx.x; i < p.num_pages; i += kScan) {
        const int r = a.refs[i];
        a.remap[i] = r > 0 ? i : -1;
        a.refs_out[i] = r > 0 && i < live ? r : i < live ? 0 : (a.refs_out == a.refs ? r : 0);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < movers; i += kScan) {
        const int2 v = w.moves[i];
        a.remap[v.x] = v.y;
        a.refs_out[v.y] = a.refs[v.x];
    }
    __syncthreads();
    if (a.refs_out == a.refs)
        for (int i = live + threadIdx.x; i < p.num_pages; i += kScan) a.refs_out[i] = 0;
    if (threadIdx.x == 0) {
        w.head[0] = movers;
        *a.live = live;
    }
}

__global__ void compact_tables_kernel(KvPages p, CompactArgs a) {
    const long long n = (long long)a.seqs * a.stride;
    for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < n; i += (long long)gridDim.x * blockDim.x) {
        const int s = int(i / a.stride), j = int(i % a.stride);
        int id = -1;
        if (j < pages_of(table_len(a.lens, s, a.stride, p.page_size, p.err), p.page_size)) {
            const int old = a.tables[i];
            if (unsigned(old) < unsigned(p.num_pages)) id = a.remap[old];
            else report(p.err, kKvBadPage);
        }
        a.tables_out[i] = id;
    }
}

int grid_for(long long n) { return int(std::min<long long>(592, std::max<long long>(1, (n + 255) / 256))); }

}  // namespace

size_t kv_pages_ws_bytes(int num_pages, int children) {
    return 256 + (size_t(num_pages) * 4 + 256) + (size_t(std::max(num_pages, children)) * 8 + 256) +
           (size_t(children) * 20 + 512);
}

void launch_kv_fork(const KvPages& p, const ForkArgs& a, void* ws, cudaStream_t s) {
    const PageWs w = carve(ws, p.num_pages, a.children);
    fork_counts_kernel<<<grid_for(std::max(p.num_pages, a.children)), 256, 0, s>>>(p, a, ws, 0);
    fork_counts_kernel<<<grid_for((long long)std::max(a.seqs, a.children) * a.stride), 256, 0, s>>>(p, a, ws, 1);
    fork_alloc_kernel<<<1, kScan, 0, s>>>(p, a, ws);
    copy_pages_kernel<<<dim3(std::min(std::max(1, a.children), 256), 2 * p.layers), 256, 0, s>>>(p, w.head, w.moves);
    check_launch("kv_fork");
}

void launch_kv_compact(const KvPages& p, const CompactArgs& a, void* ws, cudaStream_t s) {
    const PageWs w = carve(ws, p.num_pages, 0);
    compact_plan_kernel<<<1, kScan, 0, s>>>(p, a, ws);
    copy_pages_kernel<<<dim3(std::min(p.num_pages, 1024), 2 * p.layers), 256, 0, s>>>(p, w.head, w.moves);
    compact_tables_kernel<<<grid_for((long long)a.seqs * a.stride), 256, 0, s>>>(p, a);
    check_launch("kv_compact");
}

}  // namespace gpt
