// pages.cu -- the pages of a paged KV cache: reserving (with copy-on-write), forking, freeing and
// compacting, on the device, in the order of the caller's stream.
//
// State: page_table [n_seq][max_pages] (page ids, -1: none) and ref_counts [num_pages] (how many
// table entries name a page; 0: free).  Every result is a function of the state at the call's start:
// counts change by integer atomics (their order does not matter), and what depends on order -- which
// free page goes to which slot, which page moves where -- comes from prefix sums, lowest first.
//
// Reserve and compact are one launch each (the host's cost of a launch is about that of their work):
// block 0 plans, the others wait for it, then all copy pages.  Block 0 waits for nobody and is
// dispatched first, so the wait ends; it is bounded all the same.
//
// All of it is latency: tables and counts are some 100 KB, and what is copied (a few MB) would take HBM
// 1 to 2 us.  Measured: 1024 rows of 257 slots freed in 3.0 us and reserved in 12 us (8 rows of 72: 1.8
// and 8.0 us); compacting 48 rows of some 18 pages after 5 have left 11 us, with 80 pages of 4 layers
// moved or copied.  A plan is read, scanned and written by one block, two passes over the counts, which
// is what a large pool costs: reserving a page for each of 1024 rows takes 12 to 14 us where free pages lie
// among the first 4096, but 32 us behind 89 k live ones packed at the front and 70 us behind 255 k;
// compacting a pool of 100 k, 300 k and 1 M pages takes 100, 284 and 940 us before anything moves.
#include "internal.h"

namespace b2a {
namespace {

constexpr int kPlanThreads = 1024;

// Exclusive prefix sum of v over the block; *total its sum.  All threads.
__device__ __forceinline__ int block_scan(int v, int* warp_sums, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) warp_sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        int s = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    const int off = warp ? warp_sums[warp - 1] : 0;
    *total = warp_sums[(blockDim.x >> 5) - 1];
    __syncthreads();  // warp_sums may be written again
    return off + incl - v;
}

// Words of the workspace that are zero between launches.
struct PlanSync {
    int planned;  // block 0 is done
    int left;     // blocks that are done
};
constexpr unsigned long long kPlanWaitNs = 1000000000ull;

__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}
// After block 0's plan: its writes are visible to all threads of the block.  False (status bit 3) where
// the plan did not come in time.
__device__ __forceinline__ bool plan_ready(const PagePoolParams& p, PlanSync* sync) {
    __shared__ int ok_s;
    __syncthreads();
    if (threadIdx.x == 0) {
        int ok = 1;
        if (blockIdx.x == 0) {
            __threadfence();
            atomicExch(&sync->planned, 1);
        } else {
            const unsigned long long t0 = now_ns();
            while (*reinterpret_cast<volatile int*>(&sync->planned) == 0) {
                if (now_ns() - t0 > kPlanWaitNs) {
                    atomicOr(p.status, 8);
                    ok = 0;
                    break;
                }
                __nanosleep(100);
            }
            __threadfence();
        }
        ok_s = ok;
    }
    __syncthreads();
    return ok_s != 0;
}
// The last block to leave restores the words for the next launch.
__device__ __forceinline__ void leave(PlanSync* sync) {
    __syncthreads();
    if (threadIdx.x == 0 && atomicAdd(&sync->left, 1) == (int)gridDim.x - 1) {
        atomicExch(&sync->left, 0);
        atomicExch(&sync->planned, 0);
    }
}

// Copies page src[i] to page dst[i] in every layer, i < n, where src[i] >= 0; all blocks, all threads.
__device__ __forceinline__ void copy_pages(const PagePoolParams& p, const int* src, const int* dst, int n) {
    const int64_t words = p.page_bytes / 16;
    for (int64_t w = blockIdx.x; w < (int64_t)n * p.n_layers; w += gridDim.x) {
        const int i = (int)(w / p.n_layers);
        const int from = __ldcg(src + i);
        if (from < 0) continue;
        uint8_t* layer = p.pages + (w - (int64_t)i * p.n_layers) * p.layer_stride;
        const uint4* a = reinterpret_cast<const uint4*>(layer + (int64_t)from * p.page_bytes);
        uint4* b = reinterpret_cast<uint4*>(layer + (int64_t)__ldcg(dst + i) * p.page_bytes);
        for (int64_t k = threadIdx.x; k < words; k += blockDim.x) b[k] = a[k];
    }
}

__device__ __forceinline__ bool page_ok(const PagePoolParams& p, int page) {
    if (page < p.num_pages) return true;
    atomicOr(p.status, 16);
    return false;
}

// -------------------------------------------------------------------- free
// A slot that holds no position of [keep_from, keep_to) gives its page back.
__global__ void pages_free_kernel(const PagePoolParams p, const int* keep_from, const int* keep_to, int page_size) {
    const unsigned i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= (unsigned)(p.n_seq * p.max_pages)) return;
    const int row = i / (unsigned)p.max_pages, slot = i - row * p.max_pages;
    int* entry = p.page_table + i;
    const int page = *entry;
    if (page < 0) return;
    const int64_t start = (int64_t)slot * page_size;
    if (start < keep_to[row] && (keep_from == nullptr || start + page_size > keep_from[row])) return;
    if (!page_ok(p, page)) return;
    atomicSub(p.ref_counts + page, 1);
    *entry = -1;
}

// -------------------------------------------------------------------- fork
// Row i becomes what row parents[i] was.  Columns are independent: a block owns `cols` columns of
// all rows and reads them before it writes, so the table changes in place.  It has few columns where
// there are many rows, so that a thread has an entry or two (64 rows of 33: 2.9 us; always 32: 6.0).
__global__ void pages_fork_kernel(const PagePoolParams p, const int* parents, int cols) {
    extern __shared__ int old_s[];  // [n_seq][cols]
    const int c0 = blockIdx.x * cols, nc = min(cols, p.max_pages - c0);
    const int n = p.n_seq * cols;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int row = i / cols, c = i - row * cols;
        old_s[i] = c < nc ? p.page_table[(int64_t)row * p.max_pages + c0 + c] : -1;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const int row = i / cols, c = i - row * cols;
        if (c >= nc) continue;
        const int parent = parents[row];
        if (parent == row) continue;
        if (parent < -1 || parent >= p.n_seq) {
            atomicOr(p.status, 64);
            continue;
        }
        const int was = old_s[i], now = parent < 0 ? -1 : old_s[parent * cols + c];
        if (was == now) continue;
        if (was >= 0 && page_ok(p, was)) atomicSub(p.ref_counts + was, 1);
        if (now >= 0 && page_ok(p, now)) atomicAdd(p.ref_counts + now, 1);
        p.page_table[(int64_t)row * p.max_pages + c0 + c] = now;
    }
}

// -------------------------------------------------------------------- reserve
struct Span {
    int s0, s1;  // slots [s0, s1) that positions [ctx, ctx + new) fall into
};
__device__ __forceinline__ Span written_slots(const PagePoolParams& p, const int* ctx_lens, const int* new_lens,
                                              int row, int page_size) {
    const int ctx = ctx_lens[row], n = new_lens[row];
    if (n <= 0) return Span{0, 0};
    if (ctx < 0 || (int64_t)ctx + n > (int64_t)p.max_pages * page_size) {
        atomicOr(p.status, 1);
        return Span{0, 0};
    }
    const unsigned size = page_size, last = (unsigned)ctx + (unsigned)n - 1;
    return Span{(int)((unsigned)ctx / size), (int)(last / size) + 1};
}
// Whether a written slot needs a page: it has none, or one that other rows hold too.
__device__ __forceinline__ bool wants_page(const PagePoolParams& p, int page) {
    return page < 0 || (page_ok(p, page) && p.ref_counts[page] > 1);
}

// One block: who wants a page, the lowest free pages, who gets which.
// list[i], src[i]: the i-th page given out and the page to copy into it (-1: none); job[0]: how many.
__device__ __forceinline__ void plan_reserve(const PagePoolParams& p, const int* ctx_lens, const int* new_lens,
                                             int page_size, int* list, int* src, int* job, int* counts) {
    __shared__ int sums[32];
    const int tid = threadIdx.x;
    const int per = (p.n_seq + kPlanThreads - 1) / kPlanThreads;
    const int r0 = min(p.n_seq, tid * per), r1 = min(p.n_seq, r0 + per);
    // four consecutive counts a thread; the first ones are requested before the rows are looked at
    int refs[4];
    auto fetch = [&](int base) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const int page = base + 4 * tid + k;
            refs[k] = page < p.num_pages ? p.ref_counts[page] : 1;
        }
    };
    fetch(0);
    // a thread's only row (the usual case) is kept for the assignment below: its span and which of its
    // first 32 slots want a page
    Span kept{0, 0};
    unsigned kept_wants = 0;
    int mine = 0, need = 0;
    for (int row = r0; row < r1; ++row) {
        const Span s = written_slots(p, ctx_lens, new_lens, row, page_size);
        kept = s;
        for (int slot = s.s0; slot < s.s1; ++slot) {
            const bool wants = wants_page(p, p.page_table[(int64_t)row * p.max_pages + slot]);
            mine += wants;
            if (slot - s.s0 < 32) kept_wants |= (unsigned)wants << (slot - s.s0);
        }
    }
    int at = block_scan(mine, sums, &need);
    int found = 0;
    for (int base = 0; base < p.num_pages && found < need; base += 4 * kPlanThreads) {
        if (base > 0) fetch(base);
        int n_free = 0, total;
#pragma unroll
        for (int k = 0; k < 4; ++k) n_free += refs[k] == 0;
        int rank = found + block_scan(n_free, sums, &total);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (refs[k] == 0) {
                if (rank < need) list[rank] = base + 4 * tid + k;
                ++rank;
            }
        found += total;
    }
    __syncthreads();
    if (found < need) {  // too few: nothing changes
        if (tid == 0) {
            job[0] = 0;
            counts[0] = 0;
            counts[1] = need - found;
        }
        return;
    }
    for (int row = r0; row < r1 && mine > 0; ++row) {
        const Span s = per == 1 ? kept : written_slots(p, ctx_lens, new_lens, row, page_size);
        for (int slot = s.s0; slot < s.s1; ++slot) {
            if (per == 1 && slot - s.s0 < 32 && !(kept_wants >> (slot - s.s0) & 1)) continue;
            int* entry = p.page_table + (int64_t)row * p.max_pages + slot;
            const int old = *entry;
            if (!wants_page(p, old)) continue;
            src[at] = old;
            *entry = list[at];
            ++at;
        }
    }
    __syncthreads();  // every decision has read the counts as they were
    for (int i = tid; i < need; i += kPlanThreads) {
        if (src[i] >= 0) atomicSub(p.ref_counts + src[i], 1);
        p.ref_counts[list[i]] = 1;
    }
    if (tid == 0) {
        job[0] = need;
        counts[0] = need;
        counts[1] = 0;
    }
}

__global__ void __launch_bounds__(kPlanThreads) pages_reserve_kernel(const PagePoolParams p, const int* ctx_lens,
                                                                     const int* new_lens, int page_size, int* list,
                                                                     int* src, int* job, PlanSync* sync, int* counts) {
    if (blockIdx.x == 0) plan_reserve(p, ctx_lens, new_lens, page_size, list, src, job, counts);
    if (plan_ready(p, sync)) copy_pages(p, src, list, __ldcg(job));
    leave(sync);
}

// -------------------------------------------------------------------- compact
// One block: n live pages; live ones at n or above (src) go into the free places below n (dst), both
// in order; to[page - n] is where a moved page went.
__device__ __forceinline__ void plan_compact(const PagePoolParams& p, int* src, int* dst, int* to, int* job, int* counts) {
    __shared__ int sums[32];
    const int tid = threadIdx.x;
    int mine = 0, n = 0;
    for (int page = tid; page < p.num_pages; page += kPlanThreads) mine += p.ref_counts[page] > 0;
    block_scan(mine, sums, &n);
    int moves = 0, holes = 0;
    for (int base = 0; base < p.num_pages; base += kPlanThreads) {
        const int page = base + tid;
        const int live = page < p.num_pages && p.ref_counts[page] > 0;
        const int hole = page < n && !live, move = page >= n && live;
        int th, tm;
        const int rh = holes + block_scan(hole, sums, &th), rm = moves + block_scan(move, sums, &tm);
        if (hole) dst[rh] = page;
        if (move) src[rm] = page;
        if (!live && page >= n && page < p.num_pages) to[page - n] = page;  // named by no consistent entry
        holes += th;
        moves += tm;
    }
    __syncthreads();
    for (int i = tid; i < moves; i += kPlanThreads) {
        to[src[i] - n] = dst[i];
        p.ref_counts[dst[i]] = p.ref_counts[src[i]];
        p.ref_counts[src[i]] = 0;
    }
    if (tid == 0) {
        job[0] = moves;
        job[1] = n;
        counts[0] = n;
        counts[1] = moves;
    }
}

__global__ void __launch_bounds__(kPlanThreads) pages_compact_kernel(const PagePoolParams p, int* src, int* dst, int* to,
                                                                     int* job, PlanSync* sync, int* counts) {
    if (blockIdx.x == 0) plan_compact(p, src, dst, to, job, counts);
    if (plan_ready(p, sync)) {
        copy_pages(p, src, dst, __ldcg(job));
        const int n = __ldcg(job + 1);
        const int64_t total = (int64_t)p.n_seq * p.max_pages;
        for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
            const int page = p.page_table[i];
            if (page >= n && page_ok(p, page)) p.page_table[i] = __ldcg(to + page - n);
        }
    }
    leave(sync);
}

}  // namespace

size_t pages_workspace_ints(int num_pages) { return 64 + 3 * (size_t)num_pages; }

cudaError_t launch_pages_free(const PagePoolParams& p, const int* keep_from, const int* keep_to, int page_size,
                              cudaStream_t stream) {
    const unsigned grid = ((unsigned)(p.n_seq * p.max_pages) + 255) / 256;
    pages_free_kernel<<<grid, 256, 0, stream>>>(p, keep_from, keep_to, page_size);
    return cudaGetLastError();
}

cudaError_t launch_pages_fork(const PagePoolParams& p, const int* parents, cudaStream_t stream) {
    int cols = 32;
    while (cols > 4 && (int64_t)p.n_seq * cols > 512) cols >>= 1;  // 4 columns: half a sector of a row
    while (cols > 1 && (int64_t)p.n_seq * cols * 4 > 48 * 1024) cols >>= 1;
    const size_t smem = (size_t)p.n_seq * cols * 4;
    if (smem > 48 * 1024) {
        const cudaError_t e =
            cudaFuncSetAttribute(pages_fork_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
        if (e != cudaSuccess) return e;
    }
    pages_fork_kernel<<<(p.max_pages + cols - 1) / cols, 256, smem, stream>>>(p, parents, cols);
    return cudaGetLastError();
}

cudaError_t launch_pages_reserve(const PagePoolParams& p, const int* ctx_lens, const int* new_lens, int page_size,
                                 int* counts, int* sync, int* ws, int sm_count, cudaStream_t stream) {
    int *list = ws, *src = list + p.num_pages, *job = src + p.num_pages;
    pages_reserve_kernel<<<sm_count, kPlanThreads, 0, stream>>>(p, ctx_lens, new_lens, page_size, list, src, job,
                                                                reinterpret_cast<PlanSync*>(sync), counts);
    return cudaGetLastError();
}

cudaError_t launch_pages_compact(const PagePoolParams& p, int* counts, int* sync, int* ws, int sm_count,
                                 cudaStream_t stream) {
    int *src = ws, *dst = src + p.num_pages, *to = dst + p.num_pages, *job = to + p.num_pages;
    pages_compact_kernel<<<sm_count, kPlanThreads, 0, stream>>>(p, src, dst, to, job, reinterpret_cast<PlanSync*>(sync),
                                                                counts);
    return cudaGetLastError();
}

}  // namespace b2a
