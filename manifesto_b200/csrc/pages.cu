// pages.cu -- mf_page_assign: page tables, slots and positions of a step's
// new tokens, from the requests' lengths.
//
// Two exclusive prefix sums over the requests (new tokens, new pages) place
// everything: token i of the step belongs to the request whose token prefix
// holds i, and the j-th new page of a request is free page prefix + j.  A new
// page starts at exactly one new token (position % page_size == 0), so the
// thread of that token writes the table entry: no second pass over the pages.
//
// One launch, no CTA waits on another: every CTA scans all the requests
// itself (4096 of them are 32 KB, read from L2) in tiles of 2048, and handles
// every gridDim-th run of 512 tokens and of 512 requests, three runs at a time
// so that their loads travel together.  Bound: latency, the launch and one
// chain of dependent steps (lengths, scan, search, page number): 4.4 us for 8
// requests, 8.0 us for 1500 requests with 219 thousand new tokens, whose 3.6 MB
// take 0.6 us.  One CTA per SM: two and three were slower (11.6 and 13.7 us),
// since each repeats the scan.
#include "mf_divisor.cuh"
#include "mf_launch.cuh"
#include "mf_runtime.h"

namespace mf {
namespace {

constexpr int kAssignThreads = 512;
constexpr int kAssignItems = 4;                                // requests per thread and tile
constexpr int kAssignTile = kAssignThreads * kAssignItems;
constexpr int kAssignRuns = 3;                                 // runs of tokens in flight
constexpr uint32_t kNone = 0xffffffffu;

struct AssignArgs {
    const int32_t* lens;
    const int32_t* fresh;
    const int32_t* free_pages;
    const int32_t* pool;
    int32_t* table;
    int64_t* slots;
    int32_t* positions;
    int32_t* owner;
    int32_t* starts;
    int32_t* lens_after;
    int32_t* pool_after;
    int64_t tokens;
    int64_t table_stride;
    int32_t n_requests;
    int32_t max_pages;
    Divisor page;
    bool wide;  // lens and new_tokens are 16-byte aligned
};

struct Sums {
    int64_t tokens, pages;
};

__device__ __forceinline__ Sums warp_inclusive(Sums v, int lane) {
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t t = __shfl_up_sync(0xffffffffu, v.tokens, d);
        const int64_t p = __shfl_up_sync(0xffffffffu, v.pages, d);
        if (lane >= d) {
            v.tokens += t;
            v.pages += p;
        }
    }
    return v;
}

__device__ __forceinline__ int32_t clamp_i32(int64_t v) {
    return static_cast<int32_t>(v > 0x7fffffffll ? 0x7fffffffll : v);
}

// Pages of n tokens (n below 2^32, the one past 2^31 - 1 never asked for).
__device__ __forceinline__ uint32_t pages_of(uint32_t n, const Divisor& page) {
    const uint32_t q = n / page;
    return q + (q * page.d != n);
}

// A request's need of pages; `room`: whether its table row reaches that far.
__device__ __forceinline__ uint32_t pages_needed(uint32_t len, uint32_t fresh, const Divisor& page, uint32_t max_pages,
                                                 bool& room) {
    const uint32_t sum = len + fresh;  // both below 2^31: it fits
    room = sum <= 0x7fffffffu;
    if (!room) return 0;
    const uint32_t after = pages_of(sum, page);
    room = after <= max_pages;
    return room ? after - pages_of(len, page) : 0;
}

// Whether a request fits that needs `need` pages behind `before` others, its
// tokens numbered from `start` on (in 31 bits).
__device__ __forceinline__ bool fits_in(bool room, int64_t need, int64_t before, int64_t count, int64_t start, uint32_t fresh) {
    return room && (need == 0 || before + need <= count) && start + fresh <= 0x7fffffffll;
}

__global__ void __launch_bounds__(kAssignThreads) page_assign_kernel(const AssignArgs a) {
    __shared__ int32_t s_tok[kAssignTile];        // token prefix of the tile's requests, inside the tile
    __shared__ int32_t s_page[kAssignTile];       // page prefix, over all requests
    __shared__ uint32_t s_len[kAssignTile], s_new[kAssignTile];
    __shared__ Sums s_warp[kAssignThreads / 32];
    __shared__ long long s_taken;
    __shared__ int s_refused;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    after_previous();
    let_next_start();
    const Divisor page = a.page;
    const uint32_t max_pages = static_cast<uint32_t>(a.max_pages);
    const int32_t head = a.pool[0] < 0 ? 0 : a.pool[0];
    const int64_t count = a.pool[0] < 0 || a.pool[1] < 0 ? 0 : a.pool[1];
    if (tid == 0) {
        s_taken = 0;
        s_refused = 0;
    }
    int64_t tok_base = 0, page_base = 0;
    long long taken = 0;
    int refused = 0;
    for (int32_t r0 = 0; r0 < a.n_requests; r0 += kAssignTile) {
        uint32_t len[kAssignItems], fresh[kAssignItems];
        Sums mine{0, 0}, at[kAssignItems];
        bool room[kAssignItems];
        int64_t need[kAssignItems];
        const int32_t mine_at = r0 + tid * kAssignItems;
        int4 l4 = make_int4(0, 0, 0, 0), f4 = l4;
        static_assert(kAssignItems == 4, "");
        if (a.wide && mine_at + kAssignItems <= a.n_requests) {
            l4 = *reinterpret_cast<const int4*>(a.lens + mine_at);
            f4 = *reinterpret_cast<const int4*>(a.fresh + mine_at);
        } else {
            if (mine_at < a.n_requests) l4.x = a.lens[mine_at], f4.x = a.fresh[mine_at];
            if (mine_at + 1 < a.n_requests) l4.y = a.lens[mine_at + 1], f4.y = a.fresh[mine_at + 1];
            if (mine_at + 2 < a.n_requests) l4.z = a.lens[mine_at + 2], f4.z = a.fresh[mine_at + 2];
            if (mine_at + 3 < a.n_requests) l4.w = a.lens[mine_at + 3], f4.w = a.fresh[mine_at + 3];
        }
        len[0] = max(l4.x, 0), len[1] = max(l4.y, 0), len[2] = max(l4.z, 0), len[3] = max(l4.w, 0);
        fresh[0] = max(f4.x, 0), fresh[1] = max(f4.y, 0), fresh[2] = max(f4.z, 0), fresh[3] = max(f4.w, 0);
#pragma unroll
        for (int i = 0; i < kAssignItems; ++i) {
            need[i] = pages_needed(len[i], fresh[i], page, max_pages, room[i]);
            at[i] = mine;
            mine.tokens += fresh[i];
            mine.pages += need[i];
        }
        const Sums inc = warp_inclusive(mine, lane);
        __syncthreads();  // the tile before is done with the shared arrays
        if (lane == 31) s_warp[warp] = inc;
        __syncthreads();
        // the warps' sums: every warp scans them itself
        static_assert(kAssignThreads / 32 <= 32, "");
        const Sums of_warp = lane < kAssignThreads / 32 ? s_warp[lane] : Sums{0, 0};
        const Sums upto = warp_inclusive(of_warp, lane);
        const Sums all{__shfl_sync(0xffffffffu, upto.tokens, 31), __shfl_sync(0xffffffffu, upto.pages, 31)};
        const Sums before{__shfl_sync(0xffffffffu, upto.tokens - of_warp.tokens, warp) + inc.tokens - mine.tokens,
                          __shfl_sync(0xffffffffu, upto.pages - of_warp.pages, warp) + inc.pages - mine.pages};
#pragma unroll
        for (int i = 0; i < kAssignItems; ++i) {
            const int32_t k = tid * kAssignItems + i, r = r0 + k;
            const int64_t tok = before.tokens + at[i].tokens, pg = page_base + before.pages + at[i].pages;
            // what is past 31 bits is past what fits
            s_tok[k] = clamp_i32(tok);
            s_page[k] = clamp_i32(pg);
            s_len[k] = len[i];
            s_new[k] = fresh[i];
            if (r >= a.n_requests) continue;
            const bool fits = fits_in(room[i], need[i], pg, count, tok_base + tok, fresh[i]);
            refused += !fits;
            if (fits && need[i] > 0) taken = max(taken, static_cast<long long>(pg + need[i]));
            if ((r / kAssignThreads) % gridDim.x == blockIdx.x) {
                a.starts[r] = clamp_i32(tok_base + tok);
                a.lens_after[r] = static_cast<int32_t>(fits ? len[i] + fresh[i] : len[i]);
            }
        }
        __syncthreads();

        const int32_t in_tile = min(kAssignTile, a.n_requests - r0);
        // this CTA's runs of 512 tokens that meet the tile's
        const int64_t end = tok_base + all.tokens, reach = end < 0x7fffffffll ? end : 0x7fffffffll;
        int64_t run = tok_base / kAssignThreads;
        run += (static_cast<int64_t>(blockIdx.x) - run % gridDim.x + gridDim.x) % gridDim.x;
        // a few runs at a time, so that their loads of page numbers travel together
        for (; run * kAssignThreads < reach; run += static_cast<int64_t>(kAssignRuns) * gridDim.x) {
            uint32_t at[kAssignRuns], pos[kAssignRuns];  // request of the tile (kNone: no token here), position
            int32_t number[kAssignRuns];                 // page (-1: none)
            bool first_of_page[kAssignRuns];
#pragma unroll
            for (int b = 0; b < kAssignRuns; ++b) {
                const int64_t i = (run + static_cast<int64_t>(b) * gridDim.x) * kAssignThreads + tid;
                at[b] = kNone;
                if (i < tok_base || i >= reach) continue;
                const int32_t in_tokens = static_cast<int32_t>(i - tok_base);
                int lo = 0, hi = in_tile;  // the last request whose prefix is at or below the token
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s_tok[mid] <= in_tokens) lo = mid;
                    else hi = mid;
                }
                const uint32_t l = s_len[lo], f = s_new[lo];
                bool has_room;
                const int64_t n = pages_needed(l, f, page, max_pages, has_room);
                at[b] = lo;
                pos[b] = l + static_cast<uint32_t>(in_tokens - s_tok[lo]);
                number[b] = -1;
                first_of_page[b] = false;
                if (fits_in(has_room, n, s_page[lo], count, tok_base + s_tok[lo], f)) {
                    const uint32_t col = pos[b] / page, held = pages_of(l, page);
                    if (col >= held) {
                        number[b] = a.free_pages[static_cast<int64_t>(head) + s_page[lo] + (col - held)];
                        first_of_page[b] = col * page.d == pos[b];
                    } else {
                        number[b] = a.table[static_cast<int64_t>(r0 + lo) * a.table_stride + col];
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < kAssignRuns; ++b) {
                if (at[b] == kNone) continue;
                const int64_t i = (run + static_cast<int64_t>(b) * gridDim.x) * kAssignThreads + tid;
                const int32_t r = r0 + static_cast<int32_t>(at[b]);
                const uint32_t col = pos[b] / page;
                if (first_of_page[b]) a.table[static_cast<int64_t>(r) * a.table_stride + col] = number[b];
                if (i < a.tokens) {
                    a.slots[i] = number[b] < 0 ? -1 : static_cast<int64_t>(number[b]) * page.d + (pos[b] - col * page.d);
                    a.positions[i] = clamp_i32(pos[b]);
                    a.owner[i] = r;
                }
            }
        }
        tok_base = end;
        page_base += all.pages;
    }
    // entries past the total: no token
    for (int64_t i = tok_base + static_cast<int64_t>(blockIdx.x) * kAssignThreads + tid; i < a.tokens;
         i += static_cast<int64_t>(gridDim.x) * kAssignThreads) {
        a.slots[i] = -1;
        a.positions[i] = 0;
        a.owner[i] = -1;
    }
    if (blockIdx.x != 0) return;
    __syncthreads();
    if (taken) atomicMax(&s_taken, taken);
    if (refused) atomicAdd(&s_refused, refused);
    __syncthreads();
    if (tid == 0) {
        a.starts[a.n_requests] = clamp_i32(tok_base);
        a.pool_after[0] = clamp_i32(head + s_taken);
        a.pool_after[1] = clamp_i32(count - s_taken);
        a.pool_after[2] = clamp_i32(tok_base);
        a.pool_after[3] = s_refused;
    }
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" int mf_page_assign(const mf_page_config* config, const int32_t* lens, const int32_t* new_tokens,
                              int32_t n_requests, int32_t* table, const int32_t* free_pages, const int32_t* pool,
                              int64_t tokens, int64_t* slots, int32_t* positions, int32_t* owner, int32_t* starts,
                              int32_t* lens_after, int32_t* pool_after, mf_stream stream) {
    MF_ENTER();
    if (!config) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: config is NULL");
    if (config->page_size <= 0 || config->max_pages <= 0)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_assign: page size %d, %d pages per request: both must be positive",
                    config->page_size, config->max_pages);
    if (config->table_stride < config->max_pages)
        return fail(MF_ERR_SHAPE_MISMATCH, "mf_page_assign: table stride %lld is below the row's %d entries",
                    (long long)config->table_stride, config->max_pages);
    if (n_requests < 0 || n_requests > kMaxRequests || tokens < 0 || tokens > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_assign: %d requests (0 to 2^31 - 2^16), %lld tokens (0 to 2^31 - 1)", n_requests,
                    (long long)tokens);
    if (!pool || !starts || !pool_after) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL buffer");
    if (n_requests > 0 && (!lens || !new_tokens || !table || !free_pages || !lens_after))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL buffer");
    if (tokens > 0 && (!slots || !positions || !owner))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL token buffer");
    if (lens_after == lens || lens_after == new_tokens || pool_after == pool)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: outputs may not be the inputs (lens_after, pool_after)");
    AssignArgs a{lens, new_tokens, free_pages, pool, table, slots, positions, owner, starts, lens_after, pool_after,
                 tokens, config->table_stride, n_requests, config->max_pages, divisor(config->page_size),
                 aligned16(lens) && aligned16(new_tokens)};
    const int64_t work = tokens > n_requests ? tokens : n_requests;
    const int64_t grid = stream_grid(work, kAssignThreads, 1);
    const cudaError_t err = launch_overlapped(page_assign_kernel, dim3(static_cast<unsigned>(grid)), kAssignThreads, 0,
                                              static_cast<cudaStream_t>(stream), a);
    if (err != cudaSuccess) return cuda_fail(err, "mf_page_assign");
    return MF_OK;
}
