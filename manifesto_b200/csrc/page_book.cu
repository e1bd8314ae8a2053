// page_book.cu -- mf_page_book_fork, mf_page_book_compact, mf_page_copy: page
// tables whose rows share pages.
//
// Fork and compact are a few passes over the rows of the tables and over the
// pages, each of which needs all of the pass before it (who is continued, which
// pages lose their last row, how many of those there are, which row gets which
// page), so one launch runs them with a barrier between: a cluster of up to
// eight CTAs where that is enough work for them (the hardware's barrier, a few
// hundred nanoseconds), else a cooperative grid with a barrier in memory.
// Pages are numbered by prefix sums in ascending order, never by the order in
// which atomics arrive, so results are the same in every run; the atomics add
// to counters (holders) or take a minimum.
//
// Bound: latency, the launch and the chain of passes (a cluster's barrier takes half
// a microsecond to one with the stores before it, the grid's two), then the tables' bytes: 11 us
// for 128 rows of 126 pages, 20 for 2048 rows of 256 over 190 thousand pages (a
// cluster: 26), 31 for a million pages and 2048 rows of 500 compacted (a cluster: 92;
// 7 of them are 776 thousand bits set one by one).  Two barriers are saved by not
// clearing: `first` carries the number of the call, `bits` are zeroed by the call that
// used them.
//
// Copies: HBM.  2001 pages of 32 KB in 8 caches, 1.05 GB read and written: 174 us (160
// at the copy rate).  56 partly filled pages in 16 caches: 6.7 us (4.6).
#include <new>

#include "mf_divisor.cuh"
#include "mf_launch.cuh"
#include "mf_runtime.h"

namespace mf {
namespace {

constexpr int kThreads = 1024;
constexpr int kWarps = kThreads / 32;
constexpr int kCluster = 8;                  // CTAs of a cluster, the portable most (16 were no faster)
constexpr int64_t kClusterShare = 65536;     // entries that a CTA of a cluster has, at most
constexpr int kMostCtas = 256;               // of a grid
constexpr uint64_t kBarrierNs = 2000000000;  // after which a barrier in memory gives up

struct BookArgs {
    const int32_t* table;
    const int32_t* lens;
    const int32_t* parents;
    const int32_t* shares;
    const int32_t* free_pages;
    const int32_t* pool;
    int32_t* table_after;
    int32_t* lens_after;
    int32_t* shares_after;
    int32_t* free_after;
    int32_t* pool_after;
    int32_t* numbers;
    mf_page_move* moves;
    int64_t table_stride;
    int32_t n_before, n_after, n_pages, max_pages, max_requests, limit;
    Divisor page;
    // workspace
    unsigned long long* first;  // [max_requests]: the first row that continues a row, behind the number of the call
    int32_t* rank;       // [max_requests]: which of the new pages a row gets
    int32_t* list;       // [n_pages]: pages set free, or those that pages move to
    int32_t* list2;      // [n_pages]: pages that move
    uint32_t* bits;      // [n_pages / 32]: free pages
    int2* of_cta;        // [CTAs]: what each has counted
    uint32_t* barrier;   // arrivals (zero between barriers), barriers passed; the number of the call; whether bits are zero
    int32_t* status;
};

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Everything that the CTAs of the grid wrote before is visible behind it.  GRID: a barrier in memory (the launch is
// cooperative: every CTA is resident); false where that does not come about in time.  Else the grid is one cluster.
template <bool GRID>
__device__ __forceinline__ bool all_sync(const BookArgs& a) {
    if constexpr (!GRID) {
        asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        return true;
    } else {
        __syncthreads();
        int late = 0;
        if (threadIdx.x == 0) {
            uint32_t round, arrived;
            asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(round) : "l"(a.barrier + 1) : "memory");
            asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(arrived) : "l"(a.barrier) : "memory");
            if (arrived == gridDim.x - 1) {
                *a.barrier = 0;
                asm volatile("red.release.gpu.global.add.u32 [%0], 1;" ::"l"(a.barrier + 1) : "memory");
            } else {
                const uint64_t until = global_ns() + kBarrierNs;
                uint32_t now = round;
                while (now == round) {
                    asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(now) : "l"(a.barrier + 1) : "memory");
                    if (now == round && global_ns() > until) {
                        late = 1;
                        atomicExch(a.status, MF_DEVICE_TIMEOUT);
                        atomicExch(a.barrier, 0u);  // the next launch counts from zero
                        break;
                    }
                }
            }
        }
        return __syncthreads_or(late) == 0;
    }
}

__device__ __forceinline__ int32_t warp_sum(int32_t v) { return static_cast<int32_t>(__reduce_add_sync(0xffffffffu, static_cast<uint32_t>(v))); }

__device__ __forceinline__ int32_t warp_before(int32_t v, int lane) {
    int32_t upto = v;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int32_t x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
    }
    return upto - v;
}

// What the CTAs in front of this one have counted, and all of them.
__device__ __forceinline__ void ctas_before(const BookArgs& a, int2& before, int2& all) {
    const int lane = threadIdx.x & 31;
    before = all = make_int2(0, 0);
    for (int c = lane; c < static_cast<int>(gridDim.x); c += 32) {
        const int2 v = a.of_cta[c];
        all.x += v.x;
        all.y += v.y;
        if (c < static_cast<int>(blockIdx.x)) {
            before.x += v.x;
            before.y += v.y;
        }
    }
    before = make_int2(warp_sum(before.x), warp_sum(before.y));
    all = make_int2(warp_sum(all.x), warp_sum(all.y));
}

// This CTA's share of n things, a multiple of OF each.
template <int OF>
__device__ __forceinline__ void share_of(int32_t n, int32_t& begin, int32_t& end) {
    const int64_t each = (static_cast<int64_t>(n) + OF * gridDim.x - 1) / (OF * gridDim.x) * OF;
    const int64_t b = each * blockIdx.x, e = b + each;
    begin = static_cast<int32_t>(b < n ? b : n);
    end = static_cast<int32_t>(e < n ? e : n);
}

// The list of free pages, and whether it lies in its buffer.
__device__ __forceinline__ void pool_of(const BookArgs& a, int32_t& head, int32_t& count) {
    head = a.pool[0];
    count = a.pool[1];
    const bool wrong = head < 0 || count < 0 || static_cast<int64_t>(head) + count > a.n_pages;
    if (head < 0 || head > a.n_pages) head = count = 0;
    count = max(0, min(count, a.n_pages - head));
    if (wrong && blockIdx.x == 0 && threadIdx.x == 0) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
}

// Tokens of a row, and the entries of its table that hold them.
__device__ __forceinline__ uint32_t row_len(const BookArgs& a, int32_t r) {
    const int64_t reach = static_cast<int64_t>(a.max_pages) * a.page.d;
    const int32_t len = max(a.lens[r], 0);
    return len > reach ? static_cast<uint32_t>(reach) : static_cast<uint32_t>(len);
}
__device__ __forceinline__ uint32_t row_held(const BookArgs& a, uint32_t len) {
    const uint32_t full = len / a.page;
    return full + (full * a.page.d != len);
}

// This warp's share of [begin, end), a multiple of OF each; all warps' together are the CTA's, in order.
template <int OF>
__device__ __forceinline__ void warp_share(int32_t begin, int32_t end, int32_t& from, int32_t& to) {
    const int32_t each = ((end - begin + OF * kWarps - 1) / (OF * kWarps)) * OF, warp = threadIdx.x >> 5;
    from = min(end, begin + each * warp);
    to = min(end, from + each);
}

// The sum of what the warps in front of this one counted (`room`, kWarps entries, filled before a barrier), and of all.
__device__ __forceinline__ int32_t warps_before(const int32_t* room, int32_t& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int32_t of_warp = room[lane];
    static_assert(kWarps == 32, "a lane for each warp");
    total = warp_sum(of_warp);
    return __shfl_sync(0xffffffffu, warp_before(of_warp, lane), warp);
}

constexpr int kEach = 4;  // loads that a thread has on their way

template <bool GRID>
__global__ void __launch_bounds__(kThreads, 1) fork_kernel(const BookArgs a) {
    __shared__ int32_t freed_of[kWarps], needy_of[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t step = gridDim.x * kThreads, me = blockIdx.x * kThreads + tid;
    const int32_t warps = gridDim.x * kWarps, my_warp = blockIdx.x * kWarps + warp;
    constexpr int32_t kNobody = 0x7fffffff, kWide = 32 * kEach;  // columns of a row that a warp has at a time
    const int32_t segments = (a.max_pages + kWide - 1) / kWide;
    after_previous();
    let_next_start();
    const uint32_t call = a.barrier[2];
    if (call == 0) {  // the first call, or 2^32 later: higher numbers would count for more
        for (int32_t p = me; p < a.max_requests; p += step) a.first[p] = 0;
        if (!all_sync<GRID>(a)) return;
    }
    int32_t head, count;
    pool_of(a, head, count);
    for (int64_t i0 = me; i0 < a.n_pages; i0 += static_cast<int64_t>(kEach) * step) {
        int32_t v[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) v[u] = i0 + u * static_cast<int64_t>(step) < a.n_pages ? a.shares[i0 + u * static_cast<int64_t>(step)] : 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (i0 + u * static_cast<int64_t>(step) < a.n_pages) a.shares_after[i0 + u * static_cast<int64_t>(step)] = v[u];
    }
    auto parent_of = [&](int32_t r) {
        const int32_t p = a.parents[r];
        return p >= 0 && p < a.n_before ? p : -1;
    };
    for (int32_t r = me; r < a.n_after; r += step) {
        const int32_t p = parent_of(r);
        if (p >= 0) atomicMax(a.first + p, static_cast<unsigned long long>(call) << 32 | static_cast<uint32_t>(kNobody - r));
    }
    const bool met = all_sync<GRID>(a);
    if (me == 0 || !met) atomicAdd(a.barrier + 2, 1u);  // every CTA knows this call's number: the next one has another
    if (!met) return;
    // the first row that continues row p, kNobody if there is none: what earlier calls left does not count
    auto first_of = [&](int32_t p) {
        const unsigned long long v = a.first[p];
        return static_cast<uint32_t>(v >> 32) == call ? kNobody - static_cast<int32_t>(static_cast<uint32_t>(v)) : kNobody;
    };
    // rows that nobody continues let go of their pages
    for (int64_t w = my_warp; w < static_cast<int64_t>(a.n_before) * segments; w += warps) {
        const int32_t r = static_cast<int32_t>(w / segments), c0 = static_cast<int32_t>(w - static_cast<int64_t>(r) * segments) * kWide + lane;
        if (first_of(r) != kNobody) continue;
        const int32_t held = row_held(a, row_len(a, r));
        int32_t x[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) x[u] = c0 + u * 32 < held ? a.table[r * a.table_stride + c0 + u * 32] : 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            if (c0 + u * 32 >= held) continue;
            if (x[u] >= 0 && x[u] < a.n_pages) atomicSub(a.shares_after + x[u], 1);
            else atomicExch(a.status, MF_DEVICE_BAD_PAGE);
        }
    }
    // rows that need a page: marked, and counted
    int32_t page0, page1, row0, row1;
    {
        int32_t begin, end;
        share_of<32>(a.n_after, begin, end);
        warp_share<32>(begin, end, row0, row1);
        share_of<32>(a.n_pages, begin, end);
        warp_share<32>(begin, end, page0, page1);
    }
    {
        int32_t needy = 0;
        for (int32_t r = row0 + lane; r < row1; r += 32) {
            const int32_t p = parent_of(r);
            bool is = p >= 0 && first_of(p) != r;
            if (is) {
                const uint32_t len = row_len(a, p);
                is = len / a.page * a.page.d != len;
            }
            a.rank[r] = is ? 0 : -1;
            needy += is;
        }
        needy = warp_sum(needy);
        if (lane == 0) needy_of[warp] = needy;
    }
    if (!all_sync<GRID>(a)) return;
    // pages set free
    {
        int32_t freed = 0;
#pragma unroll 4
        for (int32_t i = page0 + lane; i < page1; i += 32) freed += a.shares_after[i] < 0;
        freed = warp_sum(freed);
        if (lane == 0) freed_of[warp] = freed;
    }
    __syncthreads();
    int32_t my_freed, my_needy;
    {
        int32_t all_freed, all_needy;
        my_freed = warps_before(freed_of, all_freed);
        my_needy = warps_before(needy_of, all_needy);
        if (tid == 0) a.of_cta[blockIdx.x] = make_int2(all_freed, all_needy);
    }
    if (!all_sync<GRID>(a)) return;
    int2 before, all;
    ctas_before(a, before, all);
    const int32_t freed = all.x;
    const int64_t there = static_cast<int64_t>(freed) + count;  // pages that can be given
    const int32_t taken = all.y < there ? all.y : static_cast<int32_t>(there);
    // free_after: the list of free pages without those that are taken; entry x of the whole list
    auto put_free = [&](int64_t x, int32_t page) {
        if (x >= taken && x - taken < a.n_pages) a.free_after[x - taken] = page;
    };
#pragma unroll 2
    for (int32_t i0 = page0, base = before.x + my_freed; i0 < page1; i0 += 32) {
        const int32_t i = i0 + lane;
        const bool is = i < page1 && a.shares_after[i] < 0;
        const uint32_t some = __ballot_sync(0xffffffffu, is);
        if (is) {
            const int32_t x = base + __popc(some & ((1u << lane) - 1u));
            a.shares_after[i] = 0;
            a.list[x] = i;
            put_free(x, i);
        }
        base += __popc(some);
    }
    for (int32_t r0 = row0, base = before.y + my_needy; r0 < row1; r0 += 32) {
        const int32_t r = r0 + lane;
        const bool is = r < row1 && a.rank[r] >= 0;
        const uint32_t some = __ballot_sync(0xffffffffu, is);
        if (is) a.rank[r] = base + __popc(some & ((1u << lane) - 1u));
        base += __popc(some);
    }
    for (int64_t i0 = me; i0 < count; i0 += static_cast<int64_t>(kEach) * step) {
        int32_t v[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) v[u] = i0 + u * static_cast<int64_t>(step) < count ? a.free_pages[head + i0 + u * static_cast<int64_t>(step)] : 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (i0 + u * static_cast<int64_t>(step) < count) put_free(freed + i0 + u * static_cast<int64_t>(step), v[u]);
    }
    if (me == 0) {
        const int64_t left = there - taken;
        if (left > a.n_pages) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
        a.pool_after[0] = 0;
        a.pool_after[1] = static_cast<int32_t>(left < a.n_pages ? left : a.n_pages);
        a.pool_after[2] = taken;
        a.pool_after[3] = all.y - taken;
    }
    if (!all_sync<GRID>(a)) return;
    // the rows
    for (int64_t w = my_warp; w < static_cast<int64_t>(a.n_after) * segments; w += warps) {
        const int32_t r = static_cast<int32_t>(w / segments), segment = static_cast<int32_t>(w - static_cast<int64_t>(r) * segments);
        const int32_t p = parent_of(r), x = a.rank[r];
        const bool lives = p >= 0 && x < taken;
        const uint32_t len = lives ? row_len(a, p) : 0;
        const int32_t held = row_held(a, len), full = len / a.page, c0 = segment * kWide + lane;
        int32_t number[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) number[u] = c0 + u * 32 < held ? a.table[p * a.table_stride + c0 + u * 32] : -1;
        const bool further = lives && first_of(p) != r;
        const int32_t mine = lives && x >= 0 ? (x < freed ? a.list[x] : a.free_pages[head + (x - freed)]) : -1;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            const int32_t c = c0 + u * 32;
            if (c < held && further) {
                if (c < full) {
                    if (number[u] >= 0 && number[u] < a.n_pages) atomicAdd(a.shares_after + number[u], 1);
                    else atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                } else {
                    if (static_cast<uint32_t>(number[u]) >= static_cast<uint32_t>(a.n_pages) ||
                        static_cast<uint32_t>(mine) >= static_cast<uint32_t>(a.n_pages))
                        atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                    a.moves[x] = mf_page_move{number[u], mine, static_cast<int32_t>(len - full * a.page.d), 0};
                    number[u] = mine;
                }
            }
            if (c < a.max_pages) a.table_after[r * a.table_stride + c] = number[u];
        }
        if (lane == 0 && segment == 0) a.lens_after[r] = static_cast<int32_t>(len);
    }
}

template <bool GRID>
__global__ void __launch_bounds__(kThreads, 1) compact_kernel(const BookArgs a) {
    __shared__ int32_t free_of[kWarps], below_of[kWarps];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t step = gridDim.x * kThreads, me = blockIdx.x * kThreads + tid;
    const int32_t warps = gridDim.x * kWarps, my_warp = blockIdx.x * kWarps + warp;
    after_previous();
    let_next_start();
    int32_t head, count;
    pool_of(a, head, count);
    const int32_t words = (a.n_pages + 31) / 32;
    // bits are zero, but after a call that gave up
    if (a.barrier[3] == 0) {
        for (int32_t i = me; i < words; i += step) a.bits[i] = 0;
        if (!all_sync<GRID>(a)) return;
    }
    for (int64_t i0 = me; i0 < count; i0 += static_cast<int64_t>(kEach) * step) {
        int32_t x[kEach];
        bool in[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            in[u] = i0 + u * static_cast<int64_t>(step) < count;
            x[u] = in[u] ? a.free_pages[head + i0 + u * static_cast<int64_t>(step)] : 0;
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            if (!in[u]) continue;
            if (x[u] >= 0 && x[u] < a.n_pages) atomicOr(a.bits + x[u] / 32, 1u << (x[u] & 31));
            else atomicExch(a.status, MF_DEVICE_BAD_PAGE);
        }
    }
    if (!all_sync<GRID>(a)) return;
    if (me == 0) a.barrier[3] = 0;
    int32_t begin, end, word0, word1;
    share_of<1>(words, begin, end);
    warp_share<1>(begin, end, word0, word1);
    {
        int32_t mine = 0;
#pragma unroll 4
        for (int32_t i = word0 + lane; i < word1; i += 32) mine += __popc(a.bits[i]);
        mine = warp_sum(mine);
        if (lane == 0) free_of[warp] = mine;
    }
    __syncthreads();
    int32_t of_all, my_free = warps_before(free_of, of_all);
    if (tid == 0) a.of_cta[blockIdx.x] = make_int2(of_all, 0);
    if (!all_sync<GRID>(a)) return;
    int2 before, all;
    ctas_before(a, before, all);
    const int32_t n_free = all.x, used = a.n_pages - n_free;
    if (me == 0 && n_free != count) atomicExch(a.status, MF_DEVICE_BAD_PAGE);  // a page twice, or one outside the cache
    const int32_t limit = min(max(a.limit, used), a.n_pages);
    // free pages below the limit, and the pages in use from it on: those move.  The CTA at whose words the limit lies counts
    // again what of them is below; the others count alike.
    int32_t below;
    {
        const int64_t each = (static_cast<int64_t>(words) + gridDim.x - 1) / gridDim.x;
        const int32_t last = limit / 32, at = static_cast<int32_t>(last / each);
        int32_t mine = 0;
        for (int32_t i = static_cast<int32_t>(at * each) + tid; i <= last && i < words; i += kThreads)
            mine += __popc(i < last ? a.bits[i] : a.bits[i] & ((1u << (limit & 31)) - 1u));
        for (int c = tid; c < at; c += kThreads) mine += a.of_cta[c].x;
        mine = warp_sum(mine);
        if (lane == 0) below_of[warp] = mine;
        __syncthreads();
        warps_before(below_of, below);
    }
    const int32_t moving = (a.n_pages - limit) - (n_free - below);
    int32_t free_before0 = before.x + my_free;
    for (int32_t w0 = word0; w0 < word1; w0 += 32) {
        const uint32_t held = w0 + lane < word1 ? a.bits[w0 + lane] : 0u;
        const int32_t here = min(32, word1 - w0);
        for (int k0 = 0; k0 < here; k0 += kEach) {
            int32_t shares[kEach];
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const int32_t i = (w0 + k0 + u) * 32 + lane;
                shares[u] = k0 + u < here && i < a.n_pages && i < limit ? a.shares[i] : 0;
            }
#pragma unroll
            for (int u = 0; u < kEach; ++u) {
                const uint32_t word = __shfl_sync(0xffffffffu, held, min(k0 + u, 31));
                const int32_t i = (w0 + k0 + u) * 32 + lane, free_before = free_before0 + __popc(word & ((1u << lane) - 1u));
                if (k0 + u >= here) continue;
                free_before0 += __popc(word);
                if (i >= a.n_pages) continue;
                const bool is_free = word >> lane & 1u;
                if (i >= limit) {
                    a.free_after[below - moving + (i - limit)] = i;
                    a.shares_after[i] = 0;
                    if (is_free) a.numbers[i] = i;
                    else a.list2[(i - limit) - (free_before - below)] = i;
                } else {
                    a.numbers[i] = i;
                    if (!is_free) {
                        a.shares_after[i] = shares[u];
                    } else if (free_before < moving) {
                        a.list[free_before] = i;
                    } else {
                        a.free_after[free_before - moving] = i;
                        a.shares_after[i] = 0;
                    }
                }
            }
        }
    }
    if (me == 0) {
        a.pool_after[0] = 0;
        a.pool_after[1] = n_free;
        a.pool_after[2] = moving;
        a.pool_after[3] = 0;
    }
    if (!all_sync<GRID>(a)) return;
    for (int32_t i = me; i < words; i += step) a.bits[i] = 0;
    for (int32_t j = me; j < moving; j += step) {
        const int32_t src = a.list2[j], dst = a.list[j];
        a.numbers[src] = dst;
        a.shares_after[dst] = a.shares[src];
        a.moves[j] = mf_page_move{src, dst, static_cast<int32_t>(a.page.d), 0};
    }
    if (!all_sync<GRID>(a)) return;
    if (me == 0) a.barrier[3] = 1;
    constexpr int32_t kWide = 32 * kEach;
    const int32_t segments = (a.max_pages + kWide - 1) / kWide;
    for (int64_t w = my_warp; w < static_cast<int64_t>(a.n_before) * segments; w += warps) {
        const int32_t r = static_cast<int32_t>(w / segments), c0 = static_cast<int32_t>(w - static_cast<int64_t>(r) * segments) * kWide + lane;
        const int32_t held = row_held(a, row_len(a, r));
        int32_t number[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) number[u] = c0 + u * 32 < held ? a.table[r * a.table_stride + c0 + u * 32] : -1;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            if (c0 + u * 32 >= held) continue;
            if (number[u] >= 0 && number[u] < a.n_pages) number[u] = a.numbers[number[u]];
            else atomicExch(a.status, MF_DEVICE_BAD_PAGE);
        }
#pragma unroll
        for (int u = 0; u < kEach; ++u)
            if (c0 + u * 32 < a.max_pages) a.table_after[r * a.table_stride + c0 + u * 32] = number[u];
    }
}

// ------------------------------------------------------------------ copies

constexpr int kCopyThreads = 256;
constexpr int kCopyCaches = 128;  // of a launch
constexpr int kInFlight = 4;      // pieces that a thread has on the way

// A page's first tokens as rows of pieces: `inner` pieces follow one another (times the tokens, where those do, too), `rows`
// of them (again times the tokens, where they are rows) are row_stride apart, and groups of rows group_stride apart.
struct CopyArgs {
    const mf_page_move* moves;
    const int32_t* count;
    int32_t* status;
    int64_t page_stride, token_stride, head_stride;  // bytes
    int32_t n_moves, n_caches, n_pages, page_size, heads, slices;
    int32_t row;    // pieces of a head's row
    int32_t order;  // 0: a head's tokens follow one another; 1: a token's heads do; 2: neither
    char* caches[kCopyCaches];
};

// PIECE: a type of 1 to 16 bytes to which every row's begin and length are aligned.
template <class PIECE>
__global__ void __launch_bounds__(kCopyThreads) copy_kernel(const __grid_constant__ CopyArgs a) {
    after_previous();
    let_next_start();
    const int32_t n_moves = a.count ? max(0, min(a.n_moves, *a.count)) : a.n_moves;
    const int64_t units = static_cast<int64_t>(n_moves) * a.n_caches * a.slices;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int32_t slice = static_cast<int32_t>(u % a.slices);
        const int64_t of = u / a.slices;
        const int32_t c = static_cast<int32_t>(of / n_moves), m = static_cast<int32_t>(of - static_cast<int64_t>(c) * n_moves);
        const mf_page_move move = a.moves[m];
        const bool ok = static_cast<uint32_t>(move.src) < static_cast<uint32_t>(a.n_pages) &&
                        static_cast<uint32_t>(move.dst) < static_cast<uint32_t>(a.n_pages);
        if (!ok) {
            if (threadIdx.x == 0) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
            continue;
        }
        const int32_t tokens = max(0, min(move.tokens, a.page_size));
        const char* src = a.caches[c] + move.src * a.page_stride;
        char* dst = a.caches[c] + move.dst * a.page_stride;
        // pieces that follow one another, and how far apart their beginnings are
        const uint32_t inner = a.order == 0 ? static_cast<uint32_t>(tokens) * a.row : a.order == 1 ? static_cast<uint32_t>(a.heads) * a.row : a.row;
        const int64_t apart = a.order == 0 ? a.head_stride : a.token_stride;
        const uint32_t pieces = static_cast<uint32_t>(tokens) * a.heads * a.row;
        const uint32_t begin = static_cast<uint32_t>(static_cast<uint64_t>(pieces) * slice / a.slices);
        const uint32_t end = static_cast<uint32_t>(static_cast<uint64_t>(pieces) * (slice + 1) / a.slices);
        auto place = [&](uint32_t i) -> int64_t {
            const uint32_t o = i / inner, x = i - o * inner;
            if (a.order < 2) return o * apart + static_cast<int64_t>(x) * static_cast<int64_t>(sizeof(PIECE));
            const uint32_t t = o / a.heads;
            return t * a.token_stride + (o - t * a.heads) * a.head_stride + static_cast<int64_t>(x) * static_cast<int64_t>(sizeof(PIECE));
        };
        for (uint32_t i0 = begin + threadIdx.x; i0 < end; i0 += kInFlight * kCopyThreads) {
            PIECE v[kInFlight];
            int64_t at[kInFlight];
#pragma unroll
            for (int x = 0; x < kInFlight; ++x) {
                const uint32_t i = i0 + x * kCopyThreads;
                if (i >= end) continue;
                at[x] = place(i);
                v[x] = *reinterpret_cast<const PIECE*>(src + at[x]);
            }
#pragma unroll
            for (int x = 0; x < kInFlight; ++x)
                if (i0 + x * kCopyThreads < end) *reinterpret_cast<PIECE*>(dst + at[x]) = v[x];
        }
    }
}

}  // namespace
}  // namespace mf

using namespace mf;

struct mf_page_book_s {
    mf_page_book_config config;
    BookArgs args;
    void* workspace;
    int device, ctas;
};

namespace {

// What a row of the table counts as: a warp takes up to 128 entries of it at a time, and as long for fewer (4 rows of a page
// continued by 1271, counted as they are, left one CTA with all of it: 38 us).
int64_t row_entries(int32_t max_pages) { return (static_cast<int64_t>(max_pages) + 127) / 128 * 128; }

// One launch: a cluster where the entries to read and write are few, else a grid of all SMs.
template <class Kernel>
int launch_book(mf_page_book h, Kernel cluster_kernel, Kernel grid_kernel, const BookArgs& a, int64_t entries, cudaStream_t s,
                const char* name) {
    // a CTA for each 4 thousand entries; past kClusterShare for each of a cluster the grid's slower barriers pay
    int64_t ctas = (entries + 4095) / 4096;
    if (entries <= kClusterShare * kCluster) {
        int n = 1;
        while (n < kCluster && n < ctas) n *= 2;
        cudaLaunchAttribute attr[2]{};
        attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[0].val.programmaticStreamSerializationAllowed = 1;
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = n;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cudaLaunchConfig_t config{};
        config.gridDim = dim3(n);
        config.blockDim = dim3(kThreads);
        config.stream = s;
        config.attrs = attr;
        config.numAttrs = 2;
        const cudaError_t err = cudaLaunchKernelEx(&config, cluster_kernel, a);
        return err == cudaSuccess ? MF_OK : cuda_fail(err, name);
    }
    if (ctas > h->ctas) ctas = h->ctas;
    BookArgs copy = a;
    void* params[] = {&copy};
    const cudaError_t err = cudaLaunchCooperativeKernel(reinterpret_cast<const void*>(grid_kernel), dim3(static_cast<unsigned>(ctas)),
                                                        dim3(kThreads), params, 0, s);
    return err == cudaSuccess ? MF_OK : cuda_fail(err, name);
}

}  // namespace

extern "C" int mf_page_book_create(const mf_page_book_config* config, mf_page_book* handle) {
    MF_ENTER();
    if (!config || !handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_create: NULL argument");
    *handle = nullptr;
    const mf_page_book_config& c = *config;
    if (c.page_size <= 0 || c.max_pages <= 0)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_book_create: page size %d, %d pages per request: both must be positive",
                    c.page_size, c.max_pages);
    if (c.table_stride < c.max_pages)
        return fail(MF_ERR_SHAPE_MISMATCH, "mf_page_book_create: table stride %lld is below the row's %d entries",
                    (long long)c.table_stride, c.max_pages);
    // loops over pages and rows step past their ends by a grid
    constexpr int32_t most = 0x7fffffff - kMostCtas * kThreads;
    if (c.n_pages <= 0 || c.n_pages > most || c.max_requests <= 0 || c.max_requests > most)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_book_create: %d pages, %d requests (1 to %d)", c.n_pages, c.max_requests, most);
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t firsts = up(static_cast<size_t>(c.max_requests) * 8), rows = up(static_cast<size_t>(c.max_requests) * 4), pages = up(static_cast<size_t>(c.n_pages) * 4);
    const size_t bits = up((static_cast<size_t>(c.n_pages) + 31) / 32 * 4), counted = up(kMostCtas * sizeof(int2));
    const size_t cleared = 256 + firsts, bytes = cleared + counted + rows + 2 * pages + bits;
    mf_page_book_s* h = new (std::nothrow) mf_page_book_s{};
    if (!h) return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_page_book_create: out of host memory");
    cudaError_t err = cudaMalloc(&h->workspace, bytes);
    if (err != cudaSuccess) {
        cudaGetLastError();
        delete h;
        if (err == cudaErrorMemoryAllocation)
            return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_page_book_create: %zu bytes: out of device memory", bytes);
        return cuda_fail(err, "mf_page_book_create: cudaMalloc");
    }
    err = cudaMemset(h->workspace, 0, cleared);
    if (err == cudaSuccess) err = cudaStreamSynchronize(nullptr);  // streams that do not wait for the default one may run it
    BookArgs& a = h->args;
    a.status = err == cudaSuccess ? sticky_status_ptr() : nullptr;
    if (!a.status) {
        cudaFree(h->workspace);
        delete h;
        return err != cudaSuccess ? cuda_fail(err, "mf_page_book_create: cudaMemset")
                                  : fail(MF_ERR_CUDA, "mf_page_book_create: sticky status word unavailable");
    }
    char* w = static_cast<char*>(h->workspace);
    h->config = c;
    h->device = state().device;
    h->ctas = state().sm_count < kMostCtas ? state().sm_count : kMostCtas;
    a.table_stride = c.table_stride;
    a.n_pages = c.n_pages;
    a.max_pages = c.max_pages;
    a.max_requests = c.max_requests;
    a.page = divisor(c.page_size);
    a.barrier = reinterpret_cast<uint32_t*>(w);
    a.first = reinterpret_cast<unsigned long long*>(w += 256);
    a.of_cta = reinterpret_cast<int2*>(w += firsts);
    a.rank = reinterpret_cast<int32_t*>(w += counted);
    a.list = reinterpret_cast<int32_t*>(w += rows);
    a.list2 = reinterpret_cast<int32_t*>(w += pages);
    a.bits = reinterpret_cast<uint32_t*>(w += pages);
    *handle = h;
    return MF_OK;
}

extern "C" int mf_page_book_fork(mf_page_book handle, const int32_t* table, const int32_t* lens, int32_t n_before,
                                 const int32_t* parents, int32_t n_after, const int32_t* shares, const int32_t* free_pages,
                                 const int32_t* pool, int32_t* table_after, int32_t* lens_after, int32_t* shares_after,
                                 int32_t* free_after, int32_t* pool_after, mf_page_move* moves, mf_stream stream) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_fork: handle is NULL");
    if (handle->device != state().device)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_fork: the handle belongs to device %d", handle->device);
    const int32_t most = handle->config.max_requests;
    if (n_before < 0 || n_before > most || n_after < 0 || n_after > most)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_book_fork: %d rows before, %d after (0 to %d)", n_before, n_after, most);
    if (!shares || !free_pages || !pool || !shares_after || !free_after || !pool_after || (n_before > 0 && (!table || !lens)) ||
        (n_after > 0 && (!parents || !table_after || !lens_after || !moves)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_fork: NULL buffer");
    if (shares_after == shares || free_after == free_pages || pool_after == pool || (table && table_after == table) ||
        (lens && lens_after == lens))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_fork: outputs may not be the inputs");
    if (!aligned16(moves)) return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_page_book_fork: moves must be 16-byte aligned");
    BookArgs a = handle->args;
    a.table = table;
    a.lens = lens;
    a.parents = parents;
    a.shares = shares;
    a.free_pages = free_pages;
    a.pool = pool;
    a.table_after = table_after;
    a.lens_after = lens_after;
    a.shares_after = shares_after;
    a.free_after = free_after;
    a.pool_after = pool_after;
    a.moves = moves;
    a.n_before = n_before;
    a.n_after = n_after;
    const int64_t entries = (static_cast<int64_t>(n_before) + n_after) * row_entries(handle->config.max_pages) + 3ll * handle->config.n_pages;
    return launch_book(handle, fork_kernel<false>, fork_kernel<true>, a, entries, static_cast<cudaStream_t>(stream),
                       "mf_page_book_fork");
}

extern "C" int mf_page_book_compact(mf_page_book handle, const int32_t* table, const int32_t* lens, int32_t n_requests,
                                    const int32_t* shares, const int32_t* free_pages, const int32_t* pool, int32_t limit,
                                    int32_t* table_after, int32_t* shares_after, int32_t* free_after, int32_t* pool_after,
                                    int32_t* numbers, mf_page_move* moves, mf_stream stream) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_compact: handle is NULL");
    if (handle->device != state().device)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_compact: the handle belongs to device %d", handle->device);
    if (n_requests < 0 || n_requests > handle->config.max_requests)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_book_compact: %d requests (0 to %d)", n_requests, handle->config.max_requests);
    if (limit < 0) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_compact: limit %d", limit);
    if (!shares || !free_pages || !pool || !shares_after || !free_after || !pool_after || !numbers || !moves ||
        (n_requests > 0 && (!table || !lens || !table_after)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_compact: NULL buffer");
    if (shares_after == shares || free_after == free_pages || pool_after == pool || (table && table_after == table))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_book_compact: outputs may not be the inputs");
    if (!aligned16(moves)) return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_page_book_compact: moves must be 16-byte aligned");
    BookArgs a = handle->args;
    a.table = table;
    a.lens = lens;
    a.shares = shares;
    a.free_pages = free_pages;
    a.pool = pool;
    a.table_after = table_after;
    a.shares_after = shares_after;
    a.free_after = free_after;
    a.pool_after = pool_after;
    a.numbers = numbers;
    a.moves = moves;
    a.n_before = n_requests;
    a.limit = limit;
    const int64_t entries = 2ll * n_requests * row_entries(handle->config.max_pages) + 4ll * handle->config.n_pages;
    return launch_book(handle, compact_kernel<false>, compact_kernel<true>, a, entries, static_cast<cudaStream_t>(stream),
                       "mf_page_book_compact");
}

extern "C" int mf_page_book_destroy(mf_page_book handle) {
    if (!handle) return MF_OK;
    const cudaError_t err = free_workspace(handle->device, handle->workspace);
    delete handle;
    if (err != cudaSuccess) return cuda_fail(err, "mf_page_book_destroy");
    return MF_OK;
}

extern "C" int mf_page_copy(const mf_cache_layout* layout, void* const* caches, int32_t n_caches, const mf_page_move* moves,
                            int32_t n_moves, const int32_t* count, mf_stream stream) {
    MF_ENTER();
    if (!layout || n_caches < 0 || n_moves < 0 || (n_caches > 0 && !caches))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_copy: NULL argument, or %d caches, %d moves", n_caches, n_moves);
    const mf_cache_layout& k = *layout;
    const int size = element_size(k.dtype);
    if (size == 0) return fail(MF_ERR_DTYPE_UNSUPPORTED, "mf_page_copy: dtype %d has no whole number of bytes", k.dtype);
    if (k.kv_heads <= 0 || k.head_dim <= 0 || k.page_size <= 0 || k.n_pages < 0 || k.n_pages > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_copy: %lld pages of %d tokens of %d heads of %d", (long long)k.n_pages,
                    k.page_size, k.kv_heads, k.head_dim);
    if (static_cast<double>(k.page_size) * k.kv_heads * k.head_dim * size >= 2147483648.0)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_copy: a page of 2 GB or more");
    constexpr int64_t far = int64_t(1) << 40;
    if (k.page_stride < 0 || k.token_stride < 0 || k.head_stride < 0 || k.page_stride > far || k.token_stride > far || k.head_stride > far)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_page_copy: strides must lie between 0 and 2^40");
    if (n_caches == 0 || n_moves == 0 || k.n_pages == 0) return MF_OK;
    if (!moves) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_copy: moves is NULL");
    if (!aligned16(moves)) return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_page_copy: moves must be 16-byte aligned");
    // the largest piece to which every row's begin and length are aligned; rows that follow one another are one
    const int64_t row = static_cast<int64_t>(k.head_dim) * size;
    uint64_t all = static_cast<uint64_t>(row) | static_cast<uint64_t>(k.page_stride * size) | static_cast<uint64_t>(k.token_stride * size) |
                   static_cast<uint64_t>(k.head_stride * size);
    for (int32_t c = 0; c < n_caches; ++c) {
        if (!caches[c]) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_copy: cache %d is NULL", c);
        all |= reinterpret_cast<uintptr_t>(caches[c]);
    }
    int piece = 16;
    while (all % piece) piece /= 2;
    if (piece < size) return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_page_copy: caches are not aligned to their dtype");
    CopyArgs a{};
    a.moves = moves;
    a.count = count;
    a.status = sticky_status_ptr();
    if (!a.status) return fail(MF_ERR_CUDA, "mf_page_copy: sticky status word unavailable");
    a.page_stride = k.page_stride * size;
    a.token_stride = k.token_stride * size;
    a.head_stride = k.head_stride * size;
    a.n_moves = n_moves;
    a.n_pages = static_cast<int32_t>(k.n_pages);
    a.page_size = k.page_size;
    a.heads = k.kv_heads;
    a.row = static_cast<int32_t>(row / piece);
    a.order = k.token_stride == k.head_dim ? 0 : k.head_stride == k.head_dim ? 1 : 2;
    const int sms = state().sm_count;
    for (int32_t c0 = 0; c0 < n_caches; c0 += kCopyCaches) {
        a.n_caches = n_caches - c0 < kCopyCaches ? n_caches - c0 : kCopyCaches;
        for (int32_t c = 0; c < a.n_caches; ++c) a.caches[c] = static_cast<char*>(caches[c0 + c]);
        // few pages are cut into slices of at least a round of pieces, so that every SM has work
        const int64_t pages = static_cast<int64_t>(n_moves) * a.n_caches, want = 8ll * sms;
        const int64_t rounds = (static_cast<int64_t>(a.row) * a.heads * a.page_size + kInFlight * kCopyThreads - 1) / (kInFlight * kCopyThreads);
        int64_t slices = (want + pages - 1) / pages;
        slices = slices < rounds ? slices : rounds;
        a.slices = static_cast<int32_t>(slices > 1 ? slices : 1);
        const int64_t units = pages * a.slices;
        const dim3 grid(static_cast<unsigned>(units < want ? units : want));
        auto kernel = piece == 16 ? copy_kernel<uint4> : piece == 8 ? copy_kernel<uint2> : piece == 4 ? copy_kernel<uint32_t>
                      : piece == 2 ? copy_kernel<uint16_t> : copy_kernel<uint8_t>;
        const cudaError_t err = launch_overlapped(kernel, grid, kCopyThreads, 0, static_cast<cudaStream_t>(stream), a);
        if (err != cudaSuccess) return cuda_fail(err, "mf_page_copy");
    }
    return MF_OK;
}
