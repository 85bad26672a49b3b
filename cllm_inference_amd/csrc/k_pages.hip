// k_pages.hip -- the page work of the paged KV cache: extending sequences (with copies of shared,
// partly filled pages), forking, truncating and freeing them, moving the pages in use to the front
// of the pool, and copying pages. All bookkeeping is on the device: nothing waits for the host.
//
// Every decision follows from the arrays alone (free pages are taken lowest id first, entries in
// the order given), so a call's result does not depend on timing; the atomics on reference counts
// are integer additions, which commute.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device_utils.h"
#include "kv4.h"

namespace cllm_hip {
namespace {

constexpr int kThreads = 1024;   // of the one-workgroup bookkeeping kernels
constexpr int kMaxEntries = 1024;

// Sum of v over the threads before this one; total receives the workgroup's. All threads call it.
__device__ __forceinline__ int block_scan(int v, int& total) {
    __shared__ int sums[kThreads / 64];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int incl = v;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int y = __shfl_up(incl, d, 64);
        if (lane >= d) incl += y;
    }
    __syncthreads();  // the sums of the call before have been read
    if (lane == 63) sums[wave] = incl;
    __syncthreads();
    int before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) before += sums[w];
        total += sums[w];
    }
    return before + incl - v;
}

__device__ __forceinline__ int pages_of(int64_t len, int shift) {
    return (int)((len + ((int64_t)1 << shift) - 1) >> shift);
}

// Puts a key >= 0 into a hash table in LDS (of -1 at first, twice as many places as keys); whether it
// was there.
constexpr int kHash = 2 * kMaxEntries;
__device__ __forceinline__ bool hash_insert(int* table, int key) {
    static_assert(kHash == 1 << 11, "the hash has 11 bits");
    for (uint32_t h = (uint32_t)key * 2654435761u >> 21;; h = (h + 1) & (kHash - 1)) {
        const int old = atomicCAS(&table[h], -1, key);
        if (old == -1) return false;
        if (old == key) return true;
    }
}

// Extends entry i (thread i) by counts[i] tokens. One workgroup, as the entries depend on one another (who
// shares a page, who takes which free one): bound by its chain of loads, 5.4 us for one entry and a new page
// each, 6.7 for 1024; the copies' launch takes 1 to 2 us more without copies, 4.1 for the 7 of a beam step of 32
// layers. Where entries share a last page the comparisons add to it: 16 that share one 6.2 us, 64 7.6, 256 13,
// 1024 36. (Many pages at once are taken one after the other: 64 entries of 128 new pages 40 us, 1024 330.)
// work: [0] copies, then (source, destination) pairs, then the list of taken pages at 1 + 2 * kMaxEntries.
__global__ __launch_bounds__(kThreads) void k_kv4_extend(Kv4View c, const int32_t* __restrict__ slots,
                                                         const int32_t* __restrict__ counts, int n,
                                                         int32_t* __restrict__ status) {
    __shared__ int s_page[kMaxEntries], s_slots[kHash], s_pages[kHash];
    __shared__ int s_bad, s_copies, s_twice;
    const int tid = threadIdx.x;
    if (tid == 0) s_bad = s_copies = s_twice = 0;
    for (int i = tid; i < kHash; i += kThreads) s_slots[i] = s_pages[i] = -1;
    int slot = -1, count = 0, len = 0, old_pages = 0, page = -1;
    int64_t grow = 0;
    bool bad = false;
    if (tid < n) {
        slot = slots ? slots[tid] : tid;
        count = counts[tid];
        bad = (unsigned)slot >= (unsigned)c.max_seqs || count < 0;
        if (!bad) {
            len = c.lens[slot];
            const int64_t cap = (int64_t)c.max_pages << c.page_shift;
            bad = len < 0 || len > cap || len + (int64_t)count > cap;
        }
        if (!bad) {
            old_pages = pages_of(len, c.page_shift);
            grow = pages_of(len + (int64_t)count, c.page_shift) - old_pages;
            if (count > 0 && (len & ((1 << c.page_shift) - 1))) {
                page = c.table[(int64_t)slot * c.max_pages + old_pages - 1];
                bad = (unsigned)page >= (unsigned)c.n_pages;
                if (bad) page = -1;
            }
        }
        s_page[tid] = page;
    }
    __syncthreads();
    if (tid < n) {
        if (!bad) {
            bad = hash_insert(s_slots, slot);
            if (page >= 0 && hash_insert(s_pages, page)) s_twice = 1;
        }
        if (bad) s_bad = 1;
    }
    __syncthreads();
    if (s_bad) {
        if (tid == 0) {
            *status = -1;
            c.work[0] = 0;
        }
        return;
    }
    // entries before this one that hold the same page, which have left it by this one's turn (counted only if a
    // page is named twice: a comparison with every entry before, 29 us for 1024 entries)
    bool copy = false;
    if (tid < n) {
        int same = 0;
        if (s_twice)
            for (int j = 0; j < tid; ++j) same += s_page[j] == page;
        copy = page >= 0 && c.refs[page] - same > 1;
    }
    const int need = tid < n ? (int)grow + (copy ? 1 : 0) : 0;
    int total;
    const int first = block_scan(need, total);
    if (total == 0) {
        if (tid == 0) {
            *status = 0;
            c.work[0] = 0;
        }
        if (tid < n && count > 0) c.lens[slot] = len + count;
        return;
    }
    // the first `total` free pages
    int32_t* taken = c.work + 1 + 2 * kMaxEntries;
    int found = 0;
    for (int base = 0; base < c.n_pages && found < total; base += 4 * kThreads) {
        const int p0 = base + 4 * tid;
        int free[4], k = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            free[i] = p0 + i < c.n_pages && c.refs[p0 + i] == 0;
            k += free[i];
        }
        int here;
        int at = found + block_scan(k, here);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (free[i]) {
                if (at < total) taken[at] = p0 + i;
                ++at;
            }
        }
        found += here;
    }
    if (found < total) {  // nothing has been changed
        if (tid == 0) {
            *status = total - found;
            c.work[0] = 0;
        }
        return;
    }
    __threadfence_block();
    __syncthreads();
    if (tid < n && count > 0) {
        int32_t* row = c.table + (int64_t)slot * c.max_pages;
        int at = first;
        if (copy) {
            const int dst = taken[at++];
            const int i = atomicAdd(&s_copies, 1);
            c.work[1 + 2 * i] = page;
            c.work[2 + 2 * i] = dst;
            row[old_pages - 1] = dst;
            c.refs[dst] = 1;
            atomicSub(&c.refs[page], 1);
        }
        for (int j = 0; j < (int)grow; ++j, ++at) {
            const int dst = taken[at];
            row[old_pages + j] = dst;
            c.refs[dst] = 1;
        }
        c.lens[slot] = len + count;
    }
    __syncthreads();
    if (tid == 0) {
        c.work[0] = s_copies;
        *status = 0;
    }
}

// Copies pages of every layer: pairs src[i * step] -> dst[i * step], i < n (or *n_dev). 16 KB a
// step of a workgroup; a grid that fills the chip walks them, so a call without copies ends at once.
// What bounds it: the HBM copy rate (151 MB out of a pool of 256 pages of 32 layers 47 us, 6.4 TB/s read
// and written; 64 pages of 32 layers by copy_pages, the same bytes, 43 to 45).
constexpr int kCopyChunk = 16384;
__device__ __forceinline__ void copy_pages(const Kv4View& c, const int32_t* src, const int32_t* dst, int step,
                                           int n, int64_t first, int64_t stride) {
    const int64_t chunks = (c.page_bytes + kCopyChunk - 1) / kCopyChunk;
    const int64_t total = (int64_t)n * c.n_layers * chunks;
    for (int64_t u = first; u < total; u += stride) {
        const int64_t chunk = u % chunks, lp = u / chunks;
        const int i = (int)(lp / c.n_layers), layer = (int)(lp % c.n_layers);
        const int s = src[(int64_t)i * step], d = dst[(int64_t)i * step];
        if ((unsigned)s >= (unsigned)c.n_pages || (unsigned)d >= (unsigned)c.n_pages || s == d) continue;
        const int64_t from = ((int64_t)layer * c.n_pages + s) * c.page_bytes + chunk * kCopyChunk;
        const int64_t to = ((int64_t)layer * c.n_pages + d) * c.page_bytes + chunk * kCopyChunk;
        const int bytes = (int)min((int64_t)kCopyChunk, c.page_bytes - chunk * kCopyChunk);
        u32x4 x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = (j * 256 + (int)threadIdx.x) * 16;
            if (at < bytes) x[j] = ld_u32x4_nt(c.pages + from + at);
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int at = (j * 256 + (int)threadIdx.x) * 16;
            if (at < bytes) *(u32x4*)(c.pages + to + at) = x[j];
        }
    }
}

__global__ __launch_bounds__(256) void k_kv4_copy(Kv4View c, const int32_t* src, const int32_t* dst, int step,
                                                  int n, const int32_t* n_dev) {
    copy_pages(c, src, dst, step, n_dev ? *n_dev : n, blockIdx.x, gridDim.x);
}

// Whether an earlier entry names the same slot: the earlier one stands.
__device__ __forceinline__ bool named_before(const int32_t* slots, int i) {
    int found = 0;
    for (int j = threadIdx.x; j < i; j += blockDim.x) found |= slots[j] == slots[i];
    return __syncthreads_or(found);
}

// Fork. Every source is read (its pages and length written to work, and counted once more) before any
// destination is written, so the entries act at once (a beam search's permutation): in two launches with
// a workgroup per entry, or, up to kForkOne table entries, in one workgroup with a barrier between.
__device__ __forceinline__ void fork_read(const Kv4View& c, int i, int s, int first, int step) {
    int32_t* to = c.work + (int64_t)i * (c.max_pages + 1);
    const int32_t* row = c.table + (int64_t)s * c.max_pages;
    for (int p = first; p < c.max_pages; p += step) {
        const int page = row[p];
        to[1 + p] = page;
        if ((unsigned)page < (unsigned)c.n_pages) atomicAdd(&c.refs[page], 1);
    }
    if (first == 0) to[0] = c.lens[s];
}
// The destination leaves its pages and takes those of the source.
__device__ __forceinline__ void fork_write(const Kv4View& c, int i, int d, int first, int step) {
    const int32_t* from = c.work + (int64_t)i * (c.max_pages + 1);
    int32_t* row = c.table + (int64_t)d * c.max_pages;
    for (int p = first; p < c.max_pages; p += step) {
        const int page = row[p];
        if ((unsigned)page < (unsigned)c.n_pages) atomicSub(&c.refs[page], 1);
        row[p] = from[1 + p];
    }
    if (first == 0) c.lens[d] = from[0];
}
__device__ __forceinline__ bool slots_ok(const Kv4View& c, int s, int d) {
    return (unsigned)s < (unsigned)c.max_seqs && (unsigned)d < (unsigned)c.max_seqs;
}

__global__ __launch_bounds__(256) void k_kv4_fork(Kv4View c, const int32_t* __restrict__ src,
                                                  const int32_t* __restrict__ dst, int write) {
    const int i = blockIdx.x, s = src[i], d = dst[i];
    if (!slots_ok(c, s, d) || named_before(dst, i)) return;
    if (write) fork_write(c, i, d, threadIdx.x, 256); else fork_read(c, i, s, threadIdx.x, 256);
}

// A wave per entry, in turns; the entries that stand are found once.
// (us, one launch / two: 8 beams of 40 pages 4.2 / 6.5, 16 of 64 4.6 / 6.2, 16 of 256 7.3 / 6.3, 128 of 128 27 / 7)
constexpr int kForkOne = 2048, kForkEntries = 128;
__global__ __launch_bounds__(kThreads) void k_kv4_fork_one(Kv4View c, const int32_t* __restrict__ src,
                                                           const int32_t* __restrict__ dst, int n) {
    __shared__ int s_src[kForkEntries], s_dst[kForkEntries];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if (tid < n) {
        s_src[tid] = src[tid];
        s_dst[tid] = dst[tid];
    }
    __syncthreads();
    bool ok = false;
    if (tid < n) {
        ok = slots_ok(c, s_src[tid], s_dst[tid]);
        for (int j = 0; j < tid; ++j) ok &= s_dst[j] != s_dst[tid];
    }
    __syncthreads();
    if (tid < n && !ok) s_src[tid] = -1;
    __syncthreads();
    for (int i = wave; i < n; i += kThreads / 64)
        if (s_src[i] >= 0) fork_read(c, i, s_src[i], lane, 64);
    __threadfence_block();
    __syncthreads();
    for (int i = wave; i < n; i += kThreads / 64)
        if (s_src[i] >= 0) fork_write(c, i, s_dst[i], lane, 64);
}

// One launch, a workgroup an entry: 64 entries of 128 pages freed 3.0 us, 1024 3.9.
__global__ __launch_bounds__(256) void k_kv4_truncate(Kv4View c, const int32_t* __restrict__ slots,
                                                      const int32_t* __restrict__ new_lens) {
    const int i = blockIdx.x, slot = slots[i];
    if ((unsigned)slot >= (unsigned)c.max_seqs || named_before(slots, i)) return;
    const int len = min(max(c.lens[slot], 0), max(new_lens ? new_lens[i] : 0, 0));
    int32_t* row = c.table + (int64_t)slot * c.max_pages;
    for (int p = pages_of(len, c.page_shift) + threadIdx.x; p < c.max_pages; p += 256) {
        const int page = row[p];
        if ((unsigned)page < (unsigned)c.n_pages) atomicSub(&c.refs[page], 1);
        row[p] = -1;
    }
    __syncthreads();  // the length has been read by all
    if (threadIdx.x == 0) c.lens[slot] = len;
}

// Compaction, first launch: n = pages in use; the pages in use at ids from n on, ascending, go to
// the free ids below n, ascending. work: [0] moves, (source, destination) pairs, then the new id of
// each page from n on at 1 + 2 n_pages + id.
__global__ __launch_bounds__(kThreads) void k_kv4_compact_plan(Kv4View c, int32_t* __restrict__ n_live) {
    const int tid = threadIdx.x;
    int mine = 0, n;
    for (int p = tid; p < c.n_pages; p += kThreads) mine += c.refs[p] > 0;
    (void)block_scan(mine, n);
    int holes = 0, moves = 0;
    for (int base = 0; base < c.n_pages; base += 4 * kThreads) {
        const int p0 = base + 4 * tid;
        bool live[4];
        int k = 0;  // holes below n in the low half, moved pages in the high half
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i;
            live[i] = p < c.n_pages && c.refs[p] > 0;
            if (p < n && !live[i]) k += 1;
            if (p >= n && live[i]) k += 1 << 16;
        }
        int here;
        const int before = block_scan(k, here);
        int hole = holes + (before & 0xFFFF), move = moves + (before >> 16);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int p = p0 + i;
            if (p < n && !live[i]) c.work[2 + 2 * hole++] = p;
            if (p >= n && live[i]) c.work[1 + 2 * move++] = p;
            if (p >= n && p < c.n_pages && !live[i]) c.work[1 + 2 * (int64_t)c.n_pages + p] = p;
        }
        holes += here & 0xFFFF;
        moves += here >> 16;
    }
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < moves; i += kThreads) {
        const int s = c.work[1 + 2 * i], d = c.work[2 + 2 * i];
        c.work[1 + 2 * (int64_t)c.n_pages + s] = d;
        c.refs[d] = c.refs[s];
        c.refs[s] = 0;
    }
    if (tid == 0) {
        c.work[0] = moves;
        *n_live = n;
    }
}

// Second launch: the tables' ids (the first `remap` workgroups) and the pages themselves. A moved
// page's place is at n or above and its new one below, so no copy reads what another writes.
__global__ __launch_bounds__(256) void k_kv4_compact_move(Kv4View c, const int32_t* __restrict__ n_live, int remap) {
    if ((int)blockIdx.x >= remap) {
        copy_pages(c, c.work + 1, c.work + 2, 2, c.work[0], (int)blockIdx.x - remap, (int)gridDim.x - remap);
        return;
    }
    const int n = *n_live;
    const int64_t entries = (int64_t)c.max_seqs * c.max_pages;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += (int64_t)remap * 256) {
        const int page = c.table[i];
        if (page >= n && page < c.n_pages) c.table[i] = c.work[1 + 2 * (int64_t)c.n_pages + page];
    }
}

int copy_grid(const Kv4View& c, int64_t n) {
    const int64_t units = n * c.n_layers * ((c.page_bytes + kCopyChunk - 1) / kCopyChunk);
    return (int)std::max<int64_t>(1, std::min<int64_t>(units, 2048));
}

}  // namespace

int64_t kv4_work_ints(int n_pages, int max_seqs, int max_pages) {
    const int64_t extend = 1 + 2 * (int64_t)kMaxEntries + n_pages, compact = 1 + 3 * (int64_t)n_pages;
    const int64_t fork = (int64_t)std::min(max_seqs, kMaxEntries) * ((int64_t)max_pages + 1);
    return std::max(fork, std::max(extend, compact));
}

hipError_t launch_kv4_extend(const Kv4View& c, const int32_t* slots, const int32_t* counts, int n,
                             int32_t* status, hipStream_t stream) {
    hipLaunchKernelGGL(k_kv4_extend, dim3(1), dim3(kThreads), 0, stream, c, slots, counts, n, status);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_kv4_copy, dim3((unsigned)copy_grid(c, n)), dim3(256), 0, stream, c, c.work + 1, c.work + 2, 2,
                       0, c.work);
    return hipGetLastError();
}

hipError_t launch_kv4_fork(const Kv4View& c, const int32_t* src, const int32_t* dst, int n, hipStream_t stream) {
    if (n <= kForkEntries && (int64_t)n * c.max_pages <= kForkOne) {
        hipLaunchKernelGGL(k_kv4_fork_one, dim3(1), dim3(kThreads), 0, stream, c, src, dst, n);
        return hipGetLastError();
    }
    hipLaunchKernelGGL(k_kv4_fork, dim3((unsigned)n), dim3(256), 0, stream, c, src, dst, 0);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(k_kv4_fork, dim3((unsigned)n), dim3(256), 0, stream, c, src, dst, 1);
    return hipGetLastError();
}

hipError_t launch_kv4_truncate(const Kv4View& c, const int32_t* slots, const int32_t* new_lens, int n,
                               hipStream_t stream) {
    hipLaunchKernelGGL(k_kv4_truncate, dim3((unsigned)n), dim3(256), 0, stream, c, slots, new_lens);
    return hipGetLastError();
}

hipError_t launch_kv4_compact(const Kv4View& c, int32_t* n_live, hipStream_t stream) {
    hipLaunchKernelGGL(k_kv4_compact_plan, dim3(1), dim3(kThreads), 0, stream, c, n_live);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int64_t entries = (int64_t)c.max_seqs * c.max_pages;
    const int remap = (int)std::min<int64_t>(256, (entries + 255) / 256);
    hipLaunchKernelGGL(k_kv4_compact_move, dim3((unsigned)(remap + copy_grid(c, c.n_pages))), dim3(256), 0, stream, c,
                       n_live, remap);
    return hipGetLastError();
}

hipError_t launch_kv4_copy_pages(const Kv4View& c, const int32_t* src, const int32_t* dst, int n, hipStream_t stream) {
    hipLaunchKernelGGL(k_kv4_copy, dim3((unsigned)copy_grid(c, n)), dim3(256), 0, stream, c, src, dst, 1, n,
                       (const int32_t*)nullptr);
    return hipGetLastError();
}

}  // namespace cllm_hip
