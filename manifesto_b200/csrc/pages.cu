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
// every gridDim-th run of 512 tokens and of 512 requests.  Bound: the launch
// and one chain of dependent loads for a decoding step; the 16 bytes written
// per token for a long prompt.
#include "mf_runtime.h"

namespace mf {
namespace {

constexpr int kAssignThreads = 512;
constexpr int kAssignItems = 4;                                // requests per thread and tile
constexpr int kAssignTile = kAssignThreads * kAssignItems;

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
    int32_t page;
    int32_t max_pages;
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

// A request's need of pages; `room`: whether its table row reaches that far.
__device__ __forceinline__ int64_t pages_needed(uint32_t len, uint32_t fresh, uint32_t page, uint32_t max_pages,
                                                bool& room) {
    const uint32_t held = len / page + (len % page != 0);
    const uint32_t sum = len + fresh;  // both below 2^31: it fits
    const uint32_t after = sum / page + (sum % page != 0);
    room = after <= max_pages && sum <= 0x7fffffffu;
    return room ? after - held : 0;
}

__global__ void __launch_bounds__(kAssignThreads) page_assign_kernel(const AssignArgs a) {
    __shared__ int64_t s_tok[kAssignTile + 1];   // token prefix of the tile's requests
    __shared__ int64_t s_page[kAssignTile];      // page prefix, over all requests
    __shared__ Sums s_warp[kAssignThreads / 32];
    __shared__ long long s_taken;
    __shared__ int s_refused;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t page = static_cast<uint32_t>(a.page), max_pages = static_cast<uint32_t>(a.max_pages);
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
#pragma unroll
        for (int i = 0; i < kAssignItems; ++i) {
            const int32_t r = r0 + tid * kAssignItems + i;
            const bool in = r < a.n_requests;
            const int32_t l = in ? a.lens[r] : 0, f = in ? a.fresh[r] : 0;
            len[i] = l < 0 ? 0u : static_cast<uint32_t>(l);
            fresh[i] = f < 0 ? 0u : static_cast<uint32_t>(f);
        }
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
        Sums all{0, 0}, before{0, 0};
#pragma unroll
        for (int w = 0; w < kAssignThreads / 32; ++w) {
            if (w == warp) before = all;
            all.tokens += s_warp[w].tokens;
            all.pages += s_warp[w].pages;
        }
        before.tokens += inc.tokens - mine.tokens;
        before.pages += inc.pages - mine.pages;
#pragma unroll
        for (int i = 0; i < kAssignItems; ++i) {
            const int32_t k = tid * kAssignItems + i, r = r0 + k;
            const int64_t tok = before.tokens + at[i].tokens, pg = page_base + before.pages + at[i].pages;
            s_tok[k] = tok;
            s_page[k] = pg;
            if (r >= a.n_requests) continue;
            const bool fits = room[i] && (need[i] == 0 || pg + need[i] <= count);
            refused += !fits;
            if (fits && need[i] > 0) taken = max(taken, static_cast<long long>(pg + need[i]));
            if ((r / kAssignThreads) % gridDim.x == blockIdx.x) {
                a.starts[r] = clamp_i32(tok_base + tok);
                a.lens_after[r] = static_cast<int32_t>(fits ? len[i] + fresh[i] : len[i]);
            }
        }
        if (tid == 0) s_tok[kAssignTile] = all.tokens;
        __syncthreads();

        const int32_t in_tile = min(kAssignTile, a.n_requests - r0);
        // this CTA's runs of 512 tokens that meet the tile's
        const int64_t end = tok_base + all.tokens;
        int64_t run = tok_base / kAssignThreads;
        run += (static_cast<int64_t>(blockIdx.x) - run % gridDim.x + gridDim.x) % gridDim.x;
        for (; run * kAssignThreads < end; run += gridDim.x) {
            const int64_t i = run * kAssignThreads + tid;
            if (i < tok_base || i >= end) continue;
            int lo = 0, hi = in_tile;  // the last request whose prefix is at or below the token
            while (hi - lo > 1) {
                const int mid = (lo + hi) >> 1;
                if (s_tok[mid] <= i - tok_base) lo = mid;
                else hi = mid;
            }
            const int32_t r = r0 + lo;
            const uint32_t l = static_cast<uint32_t>(max(a.lens[r], 0)), f = static_cast<uint32_t>(max(a.fresh[r], 0));
            bool has_room;
            const int64_t n = pages_needed(l, f, page, max_pages, has_room);
            const bool fits = has_room && (n == 0 || s_page[lo] + n <= count);
            const uint32_t pos = l + static_cast<uint32_t>(i - tok_base - s_tok[lo]);
            int64_t slot = -1;
            if (fits) {
                const uint32_t col = pos / page, off = pos % page, held = l / page + (l % page != 0);
                int32_t* entry = a.table + static_cast<int64_t>(r) * a.table_stride + col;
                int32_t number;
                if (col >= held) {
                    number = a.free_pages[head + s_page[lo] + (col - held)];
                    if (off == 0) *entry = number;
                } else {
                    number = *entry;
                }
                slot = static_cast<int64_t>(number) * page + off;
            }
            if (i < a.tokens) {
                a.slots[i] = slot;
                a.positions[i] = clamp_i32(pos);
                a.owner[i] = r;
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
    if (n_requests < 0 || tokens < 0 || tokens > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_page_assign: %d requests, %lld tokens", n_requests, (long long)tokens);
    if (!pool || !starts || !pool_after) return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL buffer");
    if (n_requests > 0 && (!lens || !new_tokens || !table || !free_pages || !lens_after))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL buffer");
    if (tokens > 0 && (!slots || !positions || !owner))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: NULL token buffer");
    if (lens_after == lens || lens_after == new_tokens || pool_after == pool)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_page_assign: outputs may not be the inputs (lens_after, pool_after)");
    AssignArgs a{lens, new_tokens, free_pages, pool, table, slots, positions, owner, starts, lens_after, pool_after,
                 tokens, config->table_stride, n_requests, config->page_size, config->max_pages};
    const int64_t work = tokens > n_requests ? tokens : n_requests;
    const int64_t grid = stream_grid(work, kAssignThreads, 1);
    page_assign_kernel<<<static_cast<unsigned>(grid), kAssignThreads, 0, static_cast<cudaStream_t>(stream)>>>(a);
    MF_LAUNCH_CHECK("mf_page_assign");
    return MF_OK;
}
