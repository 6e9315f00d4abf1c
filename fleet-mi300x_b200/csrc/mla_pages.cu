// The life of cache pages: requests that become copies of others (fork), release,
// reservation of pages for new rows, compaction, and plain copies of pages, for the
// caches of all layers of a model at once (they share the block table).
//
// State, all on the device, so that a decode loop or a CUDA graph needs no host in
// between: refs[page] = block-table entries that hold the page (0 = free), held[b] =
// pages of request b. Pages are taken lowest number first and every list is built in
// order, so the outcome does not depend on how the threads ran; the counts change by
// integer atomics, whose order does not matter.
//
// A forked request shares its parent's full pages and gets a copy of the last page's
// rows if that page is not full, so that the rows either of them appends are its own.
//
// What bounds these: the copies HBM (2 bytes moved per byte copied); the planning one
// CTA's passes over refs (4 bytes per page, 16 pages per thread and step) and the
// launches, so that a fork is three: plan, share + copy, switch the tables.
#include "mla_kv8.cuh"

namespace mla {

namespace pages {

constexpr int kPlanThreads = 1024;
constexpr int kCopyThreads = 256;
constexpr int kPageBytes = kPage * kRow * 2;  // a bf16 page

// Scratch of a pool: control words, per pair or request {rows, page, owner}, a list of
// page numbers per page, a second one (compaction), block-table rows of a fork.
struct Scratch {
    uint64_t ctl, rows, fresh, owner, ids, ids2, table, total;
};
__host__ __device__ inline Scratch scratch_layout(int batch, int n_pages, int max_blocks) {
    Scratch s;
    uint64_t off = 0;
    s.ctl = off;   off = align256(off + 16);
    s.rows = off;  off = align256(off + (uint64_t)batch * 4);
    s.fresh = off; off = align256(off + (uint64_t)batch * 4);
    s.owner = off; off = align256(off + (uint64_t)batch * 4);
    s.ids = off;   off = align256(off + (uint64_t)n_pages * 4);
    s.ids2 = off;  off = align256(off + (uint64_t)n_pages * 4);
    s.table = off; off = align256(off + (uint64_t)batch * max_blocks * 4);
    s.total = off;
    return s;
}
struct View {
    int32_t *ctl, *rows, *fresh, *owner, *ids, *ids2, *table;
    __device__ explicit View(const MlaPagePool& p) {
        const Scratch s = scratch_layout(p.batch, p.n_pages, p.max_blocks);
        char* b = static_cast<char*>(p.scratch);
        ctl = reinterpret_cast<int32_t*>(b + s.ctl);
        rows = reinterpret_cast<int32_t*>(b + s.rows);
        fresh = reinterpret_cast<int32_t*>(b + s.fresh);
        owner = reinterpret_cast<int32_t*>(b + s.owner);
        ids = reinterpret_cast<int32_t*>(b + s.ids);
        ids2 = reinterpret_cast<int32_t*>(b + s.ids2);
        table = reinterpret_cast<int32_t*>(b + s.table);
    }
};

__device__ __forceinline__ ErrSink sink(const MlaPagePool& p) { return ErrSink{p.error_word, p.error_host}; }
__device__ __forceinline__ bool page_ok(const MlaPagePool& p, int page) { return page >= 0 && page < p.n_pages; }

// Exclusive prefix sum over the CTA (all threads call); total in the last argument.
__device__ int block_scan(int v, int* warp_tot, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    __syncthreads();  // warp_tot of the previous scan has been read
    if (lane == 31) warp_tot[warp] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / 32; ++w) {
        if (w < warp) before += warp_tot[w];
        total += warp_tot[w];
    }
    return before + incl - v;
}

// Whether some request is named twice among ids[0, n) (numbers outside the batch do not count), by a
// bitmap in shared memory: in the usual case that no owner has to be found through global memory.
__device__ bool named_twice(const MlaPagePool& p, const int32_t* __restrict__ ids, int n, uint32_t* seen) {
    for (int i = threadIdx.x; i < (p.batch + 31) / 32; i += kPlanThreads) seen[i] = 0;
    __syncthreads();
    bool twice = false;
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        const int b = ids[i];
        if (b >= 0 && b < p.batch) twice |= (atomicOr(&seen[b >> 5], 1u << (b & 31)) >> (b & 31)) & 1;
    }
    return __syncthreads_or(twice);
}
// Then: owner[b] = the last i with ids[i] = b.
__device__ void last_named(const MlaPagePool& p, const int32_t* __restrict__ ids, int n, int32_t* owner) {
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (ids[i] >= 0 && ids[i] < p.batch) owner[ids[i]] = -1;
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += kPlanThreads)
        if (ids[i] >= 0 && ids[i] < p.batch) atomicMax(&owner[ids[i]], i);
    __syncthreads();
}

// The pages of [from, to) that are free (live = false) or held, in order, the first
// `want` of them into ids; returns how many were found (the same in every thread).
__device__ int list_pages(const MlaPagePool& p, bool live, int from, int to, int want, int32_t* ids, int* warp_tot) {
    constexpr int kPer = 16;  // consecutive pages per thread and step
    int found = 0;
    for (int base = from & ~(kPer - 1); base < to && found < want; base += kPlanThreads * kPer) {
        const int first = base + (int)threadIdx.x * kPer;
        uint32_t mask = 0;
        if (first + kPer <= to) {
            int4 v[kPer / 4];
#pragma unroll
            for (int i = 0; i < kPer / 4; ++i) v[i] = reinterpret_cast<const int4*>(p.refs + first)[i];
#pragma unroll
            for (int i = 0; i < kPer / 4; ++i)
                mask |= ((v[i].x > 0) | (v[i].y > 0) << 1 | (v[i].z > 0) << 2 | (v[i].w > 0) << 3) << (4 * i);
            if (!live) mask ^= (1u << kPer) - 1;
        } else {
            for (int i = 0; i < kPer && first + i < to; ++i) mask |= (uint32_t)((p.refs[first + i] > 0) == live) << i;
        }
        if (first < from) mask &= from - first < kPer ? ~0u << (from - first) : 0u;
        int total;
        int at = found + block_scan(__popc(mask), warp_tot, total);
        for (; mask; mask &= mask - 1, ++at)
            if (at < want) ids[at] = first + __ffs(mask) - 1;
        found += total;
    }
    return min(found, want);
}

// This CTA's share (part of parts) of a copy of `bytes` (a multiple of 16).
__device__ __forceinline__ void copy_bytes(void* dst, const void* src, int bytes, int part, int parts) {
    constexpr int kUnroll = 6;
    const uint4* s = static_cast<const uint4*>(src);
    uint4* d = static_cast<uint4*>(dst);
    const int n = bytes / 16, step = parts * kCopyThreads;
    int i = part * kCopyThreads + threadIdx.x;
    for (; i + (kUnroll - 1) * step < n; i += kUnroll * step) {
        uint4 v[kUnroll];
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) v[k] = __ldcs(s + i + k * step);
#pragma unroll
        for (int k = 0; k < kUnroll; ++k) __stcs(d + i + k * step, v[k]);
    }
    for (; i < n; i += step) d[i] = s[i];
}

// The first `rows` rows of a page, in one layer.
__device__ __forceinline__ void copy_rows(const MlaPagePool& to, const MlaPagePool& from, int layer, int dst, int src,
                                          int rows, int part, int parts) {
    char* d = static_cast<char*>(to.pages[layer]);
    const char* s = static_cast<const char*>(from.pages[layer]);
    if (!to.kv8) {
        copy_bytes(d + (int64_t)dst * kPageBytes, s + (int64_t)src * kPageBytes, rows * kRow * 2, part, parts);
        return;
    }
    d += (int64_t)dst * kPage8;
    s += (int64_t)src * kPage8;
    copy_bytes(d, s, rows * kLora, part, parts);
    copy_bytes(d + kPage8Rope, s + kPage8Rope, rows * kRope, part, parts);
    if (part == 0 && threadIdx.x == 0)
        static_cast<uint64_t*>(to.scales[layer])[dst] = static_cast<const uint64_t*>(from.scales[layer])[src];
}

// ---------------------------------------------------------------------------- fork
// One CTA: which pairs take part, the rows of each, and the fresh page of each that
// needs one (fresh[i] = page, -1 = none, -2 = the pair takes no part). ctl[0] = 1 if
// the pool cannot give them all: then nothing changes.
__global__ void __launch_bounds__(kPlanThreads) k_fork_plan(const MlaPagePool p, const int32_t* __restrict__ src,
                                                            const int32_t* __restrict__ dst, int n) {
    __shared__ int warp_tot[kPlanThreads / 32];
    __shared__ uint32_t seen[MLA_MAX_BATCH / 32];
    __shared__ int32_t near_ids[kPlanThreads];  // the fresh pages, if they are few
    pdl_wait();
    pdl_trigger();
    const View v(p);
    auto in_range = [&](int b) { return b >= 0 && b < p.batch; };
    const bool twice = named_twice(p, dst, n, seen);  // a destination named twice takes its last pair
    if (twice) last_named(p, dst, n, v.owner);
    int need = 0;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        int fresh = -2, rows = 0;
        if (i < n) {
            const int a = src[i], b = dst[i];
            if (!in_range(a) || !in_range(b) || (twice && v.owner[b] != i)) {
                record_error(sink(p), MLA_DEV_BAD_REQUEST);
            } else if (a != b) {
                rows = p.seq_lens[a];
                const int full = rows / kPage;
                if (rows < 0 || (rows + kPage - 1) / kPage > min(p.held[a], p.max_blocks)) {
                    record_error(sink(p), MLA_DEV_BAD_POSITION);
                } else if (rows % kPage && !page_ok(p, p.block_table[(int64_t)a * p.max_blocks + full])) {
                    record_error(sink(p), MLA_DEV_BAD_PAGE);
                } else {
                    fresh = rows % kPage ? 0 : -1;
                }
            }
        }
        int total;
        const int rank = need + block_scan(fresh == 0, warp_tot, total);
        if (i < n) {
            v.rows[i] = rows;
            v.fresh[i] = fresh == 0 ? rank : fresh;
        }
        need += total;
    }
    int32_t* ids = need <= kPlanThreads ? near_ids : v.ids;
    const int got = list_pages(p, false, 0, p.n_pages, need, ids, warp_tot);
    __syncthreads();  // ids complete
    if (threadIdx.x == 0) v.ctl[0] = got < need;
    if (got < need) {
        if (threadIdx.x == 0) record_error(sink(p), MLA_DEV_NO_PAGE);
        return;
    }
    for (int i = threadIdx.x; i < n; i += kPlanThreads) {
        if (v.fresh[i] < 0) continue;
        const int page = ids[v.fresh[i]];
        v.fresh[i] = page;
        p.refs[page] = 1;
    }
}

// Pair x: block 0 of y keeps a copy of the parent's entries and counts them, block
// 1 + layer copies the rows of the last page in that layer.
__global__ void __launch_bounds__(kCopyThreads) k_fork_share(const MlaPagePool p, const int32_t* __restrict__ src) {
    pdl_wait();
    pdl_trigger();
    const View v(p);
    const int i = blockIdx.x, fresh = v.fresh[i];
    if (v.ctl[0] || fresh == -2) return;
    const int rows = v.rows[i], full = rows / kPage;
    const int32_t* from = p.block_table + (int64_t)src[i] * p.max_blocks;
    if (blockIdx.y == 0) {
        int32_t* keep = v.table + (int64_t)i * p.max_blocks;
        for (int k = threadIdx.x; k < full; k += kCopyThreads) {
            const int page = from[k];
            keep[k] = page;
            if (page_ok(p, page)) atomicAdd(&p.refs[page], 1);
            else record_error(sink(p), MLA_DEV_BAD_PAGE);
        }
    } else if (fresh >= 0) {
        copy_rows(p, p, blockIdx.y - 1, fresh, from[full], rows % kPage, 0, 1);
    }
}

// One page less held by an entry.
__device__ __forceinline__ void drop(const MlaPagePool& p, int page) {
    if (!page_ok(p, page)) { record_error(sink(p), MLA_DEV_BAD_PAGE); return; }
    if (atomicSub(&p.refs[page], 1) <= 0) {
        atomicAdd(&p.refs[page], 1);
        record_error(sink(p), MLA_DEV_BAD_PAGE);
    }
}

// Pair x: the destination lets go of its old pages and takes over. Entries past its new pages
// are emptied, as release does: their pages may be another's soon.
__global__ void __launch_bounds__(kCopyThreads) k_fork_switch(const MlaPagePool p, const int32_t* __restrict__ dst) {
    pdl_wait();
    const View v(p);
    const int i = blockIdx.x, fresh = v.fresh[i];
    if (v.ctl[0] || fresh == -2) return;
    const int b = dst[i], rows = v.rows[i], full = rows / kPage;
    int32_t* row = p.block_table + (int64_t)b * p.max_blocks;
    const int32_t* keep = v.table + (int64_t)i * p.max_blocks;
    const int old = min(p.held[b], p.max_blocks);
    for (int k = threadIdx.x; k < max(old, full); k += kCopyThreads) {
        if (k < old) drop(p, row[k]);
        row[k] = k < full ? keep[k] : -1;
    }
    __syncthreads();  // held and the entry at `full` were read
    if (threadIdx.x == 0) {
        if (fresh >= 0) row[full] = fresh;
        p.held[b] = full + (fresh >= 0);
        p.seq_lens[b] = rows;
    }
}

// ---------------------------------------------------------------------------- release, reserve
__global__ void __launch_bounds__(kCopyThreads) k_release(const MlaPagePool p, const int32_t* __restrict__ requests) {
    const int b = requests[blockIdx.x];
    if (b < 0 || b >= p.batch) {
        if (threadIdx.x == 0) record_error(sink(p), MLA_DEV_BAD_REQUEST);
        return;
    }
    __shared__ int held_s;
    if (threadIdx.x == 0) {  // a request named twice is released once
        held_s = min(atomicExch(&p.held[b], 0), p.max_blocks);
        p.seq_lens[b] = 0;
    }
    __syncthreads();
    for (int k = threadIdx.x; k < held_s; k += kCopyThreads) {
        int32_t& e = p.block_table[(int64_t)b * p.max_blocks + k];
        drop(p, e);
        e = -1;  // the page may be another's soon: a step on this request, unless it reserves, is an error
    }
}

// One CTA: pages for `tokens` more rows of every named request (requests = NULL: all).
__global__ void __launch_bounds__(kPlanThreads) k_reserve(const MlaPagePool p, const int32_t* __restrict__ requests,
                                                          int n, int tokens) {
    __shared__ int warp_tot[kPlanThreads / 32];
    __shared__ uint32_t seen[MLA_MAX_BATCH / 32];
    const View v(p);
    auto request = [&](int i) { return requests ? requests[i] : i; };
    auto in_range = [&](int b) { return b >= 0 && b < p.batch; };
    const bool twice = requests && named_twice(p, requests, n, seen);  // then it gets its pages once
    if (twice) last_named(p, requests, n, v.owner);
    int need = 0;
    for (int base = 0; base < n; base += kPlanThreads) {
        const int i = base + (int)threadIdx.x;
        int more = 0;
        if (i < n) {
            const int b = request(i);
            if (!in_range(b)) {
                record_error(sink(p), MLA_DEV_BAD_REQUEST);
            } else if (!twice || v.owner[b] == i) {
                const int64_t want = ((int64_t)p.seq_lens[b] + tokens + kPage - 1) / kPage;
                if (p.seq_lens[b] < 0 || want > p.max_blocks || p.held[b] < 0) record_error(sink(p), MLA_DEV_BAD_POSITION);
                else more = max(0, (int)want - p.held[b]);
            }
        }
        int total;
        const int before = block_scan(more, warp_tot, total);
        if (total > p.n_pages - need) { need = p.n_pages + 1; break; }  // the same in every thread
        if (i < n) {
            v.rows[i] = more;
            v.fresh[i] = need + before;
        }
        need += total;
    }
    const int got = need > p.n_pages ? 0 : list_pages(p, false, 0, p.n_pages, need, v.ids, warp_tot);
    __syncthreads();  // the lists are complete
    if (got < need) {
        if (threadIdx.x == 0) record_error(sink(p), MLA_DEV_NO_PAGE);
        return;
    }
    for (int i = threadIdx.x / 32; i < n; i += kPlanThreads / 32) {  // a warp per request
        const int more = v.rows[i];
        if (!more) continue;
        const int b = request(i), held = p.held[b], rank = v.fresh[i];
        for (int k = threadIdx.x & 31; k < more; k += 32) {
            const int page = v.ids[rank + k];
            p.block_table[(int64_t)b * p.max_blocks + held + k] = page;
            p.refs[page] = 1;
        }
        __syncwarp();  // held was read
        if ((threadIdx.x & 31) == 0) p.held[b] = held + more;
    }
}

// ---------------------------------------------------------------------------- compact
// One CTA: with L pages held, the held pages from L on (ids2, in order) move to the free
// ones before L (ids); ctl = {L, moves}.
__global__ void __launch_bounds__(kPlanThreads) k_compact_plan(const MlaPagePool p) {
    __shared__ int warp_tot[kPlanThreads / 32];
    const View v(p);
    int mine = 0, live;
    for (int i = threadIdx.x; i < p.n_pages; i += kPlanThreads) mine += p.refs[i] > 0;
    block_scan(mine, warp_tot, live);
    const int n = list_pages(p, false, 0, live, live, v.ids, warp_tot);
    list_pages(p, true, live, p.n_pages, n, v.ids2, warp_tot);
    if (threadIdx.x == 0) { v.ctl[0] = live; v.ctl[1] = n; }
}

__global__ void __launch_bounds__(kCopyThreads) k_compact_move(const MlaPagePool p) {
    const View v(p);
    const int64_t n = (int64_t)v.ctl[1] * p.n_layers;
    for (int64_t i = blockIdx.x; i < n; i += gridDim.x)
        copy_rows(p, p, (int)(i % p.n_layers), v.ids[i / p.n_layers], v.ids2[i / p.n_layers], kPage, 0, 1);
}

// Entries that name a moved page follow it (by its place in ids2, which ascends), and so do the
// counts; neither reads what the other writes.
__global__ void __launch_bounds__(kCopyThreads) k_compact_tables(const MlaPagePool p) {
    const View v(p);
    const int live = v.ctl[0], n = v.ctl[1], b = blockIdx.x;
    const int held = min(p.held[b], p.max_blocks);
    for (int k = threadIdx.x; k < held; k += kCopyThreads) {
        int32_t& e = p.block_table[(int64_t)b * p.max_blocks + k];
        if (e < live || e >= p.n_pages) continue;
        int lo = 0, hi = n;  // first place with ids2 >= e
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (v.ids2[mid] < e) lo = mid + 1; else hi = mid;
        }
        if (lo < n && v.ids2[lo] == e) e = v.ids[lo];
    }
    for (int64_t i = (int64_t)blockIdx.x * kCopyThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kCopyThreads) {
        p.refs[v.ids[i]] = p.refs[v.ids2[i]];
        p.refs[v.ids2[i]] = 0;
    }
}

// ---------------------------------------------------------------------------- copy
__global__ void __launch_bounds__(kCopyThreads) k_copy_pages(const MlaPagePool to, const MlaPagePool from,
                                                             const int32_t* __restrict__ src,
                                                             const int32_t* __restrict__ dst, int parts) {
    pdl_wait();
    const int s = src[blockIdx.x], d = dst[blockIdx.x];
    if (s < 0 || s >= from.n_pages || d < 0 || d >= to.n_pages) {
        if (threadIdx.x == 0) record_error(ErrSink{to.error_word, to.error_host}, MLA_DEV_BAD_PAGE);
        return;
    }
    copy_rows(to, from, blockIdx.y / parts, d, s, kPage, blockIdx.y % parts, parts);
}

}  // namespace pages

using namespace pages;

uint64_t pool_scratch_bytes(int batch, int n_pages, int max_blocks) {
    return scratch_layout(batch, n_pages, max_blocks).total;
}

cudaError_t launch_pool_fork(const MlaPagePool& p, const int32_t* src, const int32_t* dst, int n, cudaStream_t s) {
    cudaError_t e = launch_pdl(k_fork_plan, dim3(1), dim3(kPlanThreads), 0, s, p, src, dst, n);
    if (e == cudaSuccess)
        e = launch_pdl(k_fork_share, dim3(n, 1 + p.n_layers), dim3(kCopyThreads), 0, s, p, src);
    if (e == cudaSuccess) e = launch_pdl(k_fork_switch, dim3(n), dim3(kCopyThreads), 0, s, p, dst);
    return e == cudaSuccess ? cudaGetLastError() : e;
}

cudaError_t launch_pool_release(const MlaPagePool& p, const int32_t* requests, int n, cudaStream_t s) {
    k_release<<<n, kCopyThreads, 0, s>>>(p, requests);
    return cudaGetLastError();
}

cudaError_t launch_pool_reserve(const MlaPagePool& p, const int32_t* requests, int n, int tokens, cudaStream_t s) {
    k_reserve<<<1, kPlanThreads, 0, s>>>(p, requests, n, tokens);
    return cudaGetLastError();
}

cudaError_t launch_pool_compact(const MlaPagePool& p, int sm_count, cudaStream_t s) {
    k_compact_plan<<<1, kPlanThreads, 0, s>>>(p);
    k_compact_move<<<8 * sm_count, kCopyThreads, 0, s>>>(p);
    k_compact_tables<<<p.batch, kCopyThreads, 0, s>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_copy_pages(const MlaPagePool& to, const MlaPagePool& from, const int32_t* src, const int32_t* dst,
                              int n, int sm_count, cudaStream_t s) {
    // few pages: several CTAs per page and layer, so that the copy still fills the GPU
    const int64_t jobs = (int64_t)n * to.n_layers;
    const int parts = jobs >= 4 * sm_count ? 1 : (jobs >= sm_count ? 3 : 9);
    return launch_pdl(k_copy_pages, dim3(n, to.n_layers * parts), dim3(kCopyThreads), 0, s, to, from, src, dst, parts);
}

}  // namespace mla
