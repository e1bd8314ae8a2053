// prefix_attn.cu -- mf_prefix_attn_*: attention of one new token per request
// where groups of requests share the pages of their first tokens.
//
// A request's softmax over its tokens is that over the shared ones and that over
// its own, joined by their maxima and sums.  Three launches: the shared tokens of
// all groups (here), every request's own tokens (paged_attn.cu's kernel, from
// own_first on), and the join of both (here).
//
// The shared tokens are the products S = Q K^T and O = P V with up to 256 rows (a
// group's requests x the query heads of one key-value head), on tcgen05.mma with
// the accumulators in tensor memory.  One CTA per SM, in roles:
//   * four producer warps copy keys and values, tile by tile, into a ring in
//     shared memory (16-byte cp.async in the 128-byte swizzle that the products
//     read; FP8 codes become f16 on the way, exactly), rows found through the
//     page table, masked ones zero-filled;
//   * one thread issues the products: S into tensor memory, P (from tensor
//     memory) times V into the accumulator O in tensor memory;
//   * two groups of four softmax warps, a thread for each row, turn S into P in
//     place: running maximum and sum in float32, P as two 16-bit terms (high and
//     low: what the two leave out of a weight is 2^-16 of it in BF16, 2^-22 in
//     f16), O rescaled only when a maximum has grown by more than 2^8 (2^15).
// The groups alternate, so that one's softmax runs beside the other's products: of
// more than 128 rows each has 128 and sees every tile, else both have the same
// rows and every second tile.  The tiles of all (group, block of rows, key-value
// head) items in a row are cut evenly for the CTAs; every CTA leaves the part of
// its run, and the last launch joins a row's parts in the order of the tokens.
#include <new>

#include "mf_async.cuh"
#include "mf_attn.cuh"
#include "mf_divisor.cuh"
#include "mf_internal.h"
#include "mf_launch.cuh"
#include "mf_runtime.h"

namespace mf {
namespace {

// What the join needs of a request's group: the place of its first tile, tiles of an item (0: nothing is shared), its first
// request and its requests.
struct Shared {
    int32_t base, tiles, start, members;
};

struct PrefixArgs {
    const int32_t* lens;
    const int32_t* table;
    const int32_t* starts;
    const int32_t* shared;
    int32_t n_requests, n_groups;
    int32_t max_pages, page, window, kv_heads;
    const char* k;
    const char* v;
    int64_t page_bytes, row_bytes, head_bytes, table_stride;
    uint32_t n_pages;
    Divisor by_page;
    Divisor group;        // query heads of a key-value head
    int32_t head_dim;
    const char* q;
    int64_t q_req, q_head;
    int32_t q_heads, q_f16, q_wide;  // q_wide: rows of 16-byte pieces
    float scale, softcap;
    const float* slopes;
    const float* k_scale;
    const float* v_scale;
    // workspace
    int32_t* own_first;   // [requests]
    Shared* info;         // [requests]
    int2* cut;            // tiles of all items, CTAs that they are cut for
    float* part;          // [2][requests][q_heads][head_dim]: an item's first CTA, its two halves
    float2* part_ml;      // [2][requests][q_heads]
    float* cta_part;      // [CTAs][2][128][head_dim]: a CTA that begins inside an item
    float2* cta_ml;       // [CTAs][2][128]
    float* own;           // [requests][q_heads][head_dim]: the requests' own tokens
    float* own_lse;       // [requests][q_heads]
    char* out;
    int64_t out_req, out_head;
    float* lse;
    int32_t* status;
};

// ------------------------------------------------------------------ tcgen05

__device__ __forceinline__ void fence_proxy() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// The products issued so far by this thread arrive at `bar` when they are done.
__device__ __forceinline__ void tc_commit(uint64_t* bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// d (+)= a b, a and b in shared memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
                 "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
                 : "memory");
}
// The same with a in tensor memory.
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
                 "r"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
                 : "memory");
}
#define MF_R8(x, i) "=r"(x[i]), "=r"(x[i + 1]), "=r"(x[i + 2]), "=r"(x[i + 3]), "=r"(x[i + 4]), "=r"(x[i + 5]), "=r"(x[i + 6]), "=r"(x[i + 7])
#define MF_I8(x, i) "r"(x[i]), "r"(x[i + 1]), "r"(x[i + 2]), "r"(x[i + 3]), "r"(x[i + 4]), "r"(x[i + 5]), "r"(x[i + 6]), "r"(x[i + 7])
// 32 columns of this thread's row (lane of tensor memory).
__device__ __forceinline__ void tm_load(uint32_t (&r)[32], uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : MF_R8(r, 0), MF_R8(r, 8), MF_R8(r, 16), MF_R8(r, 24)
        : "r"(at)
        : "memory");
}
__device__ __forceinline__ void tm_store(uint32_t at, const uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,"
        "%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(at),
        MF_I8(r, 0), MF_I8(r, 8), MF_I8(r, 16), MF_I8(r, 24)
        : "memory");
}
// A shared-memory operand in the 128-byte swizzle: where it begins, and the bytes between groups of 8 rows (`stride`) and, of an
// operand whose rows run along the product's sum, between panels of 64 columns (`lead`).
__device__ __forceinline__ uint64_t operand(uint32_t at, uint32_t lead, uint32_t stride) {
    return static_cast<uint64_t>((at & 0x3ffffu) >> 4) | static_cast<uint64_t>(lead >> 4) << 16 | static_cast<uint64_t>(stride >> 4) << 32 |
           1ull << 46 | 2ull << 61;
}
// The product's shape and types: 128 x n, float32 sums; b_rows: B is stored with its rows along the sum.
__device__ __forceinline__ uint32_t product(bool bf16, int n, bool b_rows) {
    const uint32_t t = bf16 ? 1u : 0u;
    return 1u << 4 | t << 7 | t << 10 | (b_rows ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}

constexpr int kProducers = 128;
constexpr int kMasks = 8;  // tiles whose masks are kept: more than the ring holds

// MODE: dtype of the cache; DP: head_dim padded to 64, 128 or 256.
template <int MODE, int DP>
struct Prefix {
    static constexpr bool kFp8 = MODE == MF_DT_F8E4M3 || MODE == MF_DT_F8E5M2;
    static constexpr bool kBf16 = MODE == MF_DT_BF16;
    // Weights are exp2(s - m) with m a maximum less kBelow, replaced when a score exceeds it by kAbove: f16 ends at 2^16 and at
    // 2^-24, and so small weights beside a dominant one keep their bits (as in paged_attn.cu).
    static constexpr float kBelow = kBf16 ? 0.0f : 12.0f;
    static constexpr float kAbove = kBf16 ? 8.0f : 15.0f;
    static constexpr int kDim = DP;
    static constexpr int T = DP == 256 ? 64 : 128;       // tokens of a tile
    static constexpr int kStreams = DP == 256 ? 1 : 2;   // softmax groups
    static constexpr int kPanels = DP / 64;              // of 64 elements (128 bytes) of a row
    static constexpr int kUnit = T * DP * 2;             // bytes of a tile's keys, or values
    static constexpr int kQ = 128 * DP * 2;              // of 128 rows of queries
    static constexpr int kStages = DP == 64 ? 10 : 5;    // units of the ring
    static constexpr int kRows = 128 * kStreams;         // of a block
    static constexpr int kSoftmax = 128 * kStreams;      // threads
    static constexpr int kThreads = kSoftmax + kProducers + 32;
    static constexpr int kO = 2 * T;                     // columns of tensor memory: S of even and odd steps, then O
    struct Shared {
        uint64_t full[kStages], empty[kStages];
        uint64_t s_full[2], p_full[2], o_done[2], q_full[2], drained;
        uint32_t tmem;
        int32_t abandoned;
        int32_t group, into;        // where this CTA's run begins
        uint32_t mask[kMasks][4];   // tokens of a tile that are there
        int64_t row[2][T];          // where a tile's rows are, from the head's begin; -1: masked
    };
    static constexpr int kBytes = kStages * kUnit + kStreams * kQ + static_cast<int>(sizeof(Shared));
};

// Shared tokens of a group, and its requests; nothing is shared by a request alone.
struct Group {
    int32_t start, members, shared;
    bool bad;
};
__device__ __forceinline__ Group group_of(const PrefixArgs& a, int32_t g) {
    Group x;
    const int32_t s = a.starts[g], e = a.starts[g + 1];
    x.bad = s < 0 || e < s || e > a.n_requests;
    x.start = s;
    x.members = x.bad ? 0 : e - s;
    const int64_t reach = static_cast<int64_t>(a.max_pages) * a.page;
    x.shared = x.members < 2 ? 0 : max(a.shared[g], 0);
    if (x.shared > reach) x.shared = static_cast<int32_t>(reach);
    return x;
}
template <class K>
__device__ __forceinline__ int32_t tiles_of(const Group& x) {
    return static_cast<int32_t>((static_cast<uint32_t>(x.shared) + K::T - 1) / K::T);
}
template <class K>
__device__ __forceinline__ int64_t items_of(const PrefixArgs& a, const Group& x) {
    return (static_cast<int64_t>(x.members) * a.group.d + K::kRows - 1) / K::kRows * a.kv_heads;
}

// A run of tiles of one item.  Every role walks the same runs.
template <class K>
struct Run {
    Group of;
    int32_t g, tiles, items, item, t, left;
    // of the item at hand
    int32_t n, kv, block, rows;  // tiles of the run in it; its key-value head, block of rows, rows
    __device__ __forceinline__ Run(const PrefixArgs& a, int32_t group, int32_t into, int32_t run) : g(group), left(run) {
        of = group_of(a, g);
        tiles = tiles_of<K>(of);
        items = static_cast<int32_t>(items_of<K>(a, of));
        item = into / tiles;
        t = into - item * tiles;
        set(a);
    }
    __device__ __forceinline__ void set(const PrefixArgs& a) {
        const int32_t blocks = items / a.kv_heads;
        kv = item / blocks;
        block = item - kv * blocks;
        const int64_t after = static_cast<int64_t>(of.members) * a.group.d - static_cast<int64_t>(block) * K::kRows;
        rows = after < K::kRows ? static_cast<int32_t>(after) : K::kRows;
        n = min(tiles - t, left);
    }
    // whether each softmax group has rows of its own; else they share the rows and take turns at the tiles
    __device__ __forceinline__ bool dual() const { return K::kStreams == 2 && rows > 128; }
    __device__ __forceinline__ int32_t steps() const { return dual() ? 2 * n : n; }
    __device__ __forceinline__ bool next(const PrefixArgs& a) {
        left -= n;
        if (left <= 0) return false;
        t = 0;
        if (++item == items) {
            item = 0;
            do {
                of = group_of(a, ++g);
                tiles = tiles_of<K>(of);
            } while (tiles == 0 && g + 1 < a.n_groups);
            items = static_cast<int32_t>(items_of<K>(a, of));
        }
        set(a);
        return true;
    }
};

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Wait for a phase.  Once a wait of the CTA has run out none lasts any more: every role then goes through its remaining steps
// without waiting (all of its accesses stay in bounds), so that barriers and arrivals still match, and the status says so.
constexpr uint64_t kWaitNs = 2000000000;
__device__ __forceinline__ void wait(int32_t* abandoned, uint64_t* bar, uint32_t parity) {
    if (mbar_try_wait(bar, parity)) return;
    const uint64_t until = global_ns() + kWaitNs;
    while (!mbar_try_wait(bar, parity)) {
        if (*reinterpret_cast<volatile int32_t*>(abandoned)) return;
        if (global_ns() > until) {
            *reinterpret_cast<volatile int32_t*>(abandoned) = 1;
            return;
        }
    }
}

// Byte of piece `c` (16 bytes) of row `row` of a tile of `rows` rows: panels of 128 bytes, their pieces exchanged.
__device__ __forceinline__ uint32_t place(int rows, int row, int c) {
    return static_cast<uint32_t>((c >> 3) * (rows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// ------------------------------------------------------------------ roles

template <class K, int MODE>
__device__ __forceinline__ void produce(const PrefixArgs& a, typename K::Shared& sh, uint32_t ring, Run<K> run) {
    const int tid = threadIdx.x - K::kSoftmax, lane = tid & 31, warp = tid >> 5;
    constexpr int kBytesOf = K::kFp8 ? 1 : 2;
    const int pieces = (a.head_dim * kBytesOf + 15) / 16;  // 16-byte pieces of a row in memory
    constexpr int kMostPieces = K::kPanels * 8 / (K::kFp8 ? 2 : 1);
    const int piece = tid % kMostPieces, row0 = tid / kMostPieces;
    constexpr int kStep = kProducers / kMostPieces, kCopies = K::T / kStep;
    const bool mine = piece < pieces;
    const int64_t kv_gap = a.v - a.k;
    uint32_t unit = 0, told = 0;  // units begun, units of which the consumer knows
    int32_t tile = 0;             // tiles so far
    auto tell = [&]() {           // this warp's part of unit `told` is there
        fence_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[told % K::kStages]);
        ++told;
    };
    bool more = true;
    while (more) {
        const int64_t at_row = static_cast<int64_t>(run.of.start) * a.table_stride;
        const char* head = a.k + run.kv * a.head_bytes;
        int32_t number = 0;
        auto look_up = [&](int32_t t) {
            const uint32_t tok = static_cast<uint32_t>(t) * K::T + tid;
            if (tid < K::T && tok < static_cast<uint32_t>(run.of.shared)) number = a.table[at_row + tok / a.by_page];
        };
        look_up(run.t);
        for (int32_t i = 0; i < run.n; ++i, ++tile) {
            const int buf = tile & 1;
            if (tid < K::T) {
                const uint32_t tok = static_cast<uint32_t>(run.t + i) * K::T + tid;
                const bool in = tok < static_cast<uint32_t>(run.of.shared), ok = in && static_cast<uint32_t>(number) < a.n_pages;
                if (in && !ok) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                sh.row[buf][tid] = ok ? static_cast<int64_t>(number) * a.page_bytes + (tok - tok / a.by_page * a.page) * a.row_bytes : -1;
                const uint32_t word = __ballot_sync(0xffffffffu, ok);
                if (lane == 0) sh.mask[tile % kMasks][warp] = word;
            }
            asm volatile("bar.sync 1, %0;" ::"n"(kProducers) : "memory");
            if (i + 1 < run.n) look_up(run.t + i + 1);
#pragma unroll 1
            for (int of = 0; of < 2; ++of) {
                const uint32_t stage = unit % K::kStages, parity = (unit / K::kStages & 1u) ^ 1u;
                const uint32_t to = ring + stage * K::kUnit;
                const char* base = head + (of ? kv_gap : 0) + piece * 16;
                if constexpr (!K::kFp8) {
                    if (!__all_sync(0xffffffffu, mbar_try_wait(&sh.empty[stage], parity))) {
                        // no room: what is on the way may be what the consumer waits for
                        cp_async_wait<0>();
                        while (told < unit) tell();
                        wait(&sh.abandoned, &sh.empty[stage], parity);
                        __syncwarp();
                    }
                    if (mine) {
#pragma unroll 4
                        for (int x = 0; x < kCopies; ++x) {
                            const int r = row0 + x * kStep;
                            const int64_t off = sh.row[buf][r];
                            cp_async16(to + place(K::T, r, piece), off >= 0 ? base + off : a.k, off >= 0 ? 16u : 0u);
                        }
                    }
                    cp_async_commit();
                    ++unit;
                    if (unit - told > K::kStages - 2) {
                        cp_async_wait<K::kStages - 2>();
                        tell();
                    }
                } else {
                    uint4 code[kCopies];
                    if (mine) {
#pragma unroll
                        for (int x = 0; x < kCopies; ++x) {
                            const int64_t off = sh.row[buf][row0 + x * kStep];
                            code[x] = off >= 0 ? *reinterpret_cast<const uint4*>(base + off) : make_uint4(0, 0, 0, 0);
                        }
                    }
                    wait(&sh.abandoned, &sh.empty[stage], parity);
                    __syncwarp();
                    if (mine) {
#pragma unroll
                        for (int x = 0; x < kCopies; ++x) {
                            const int r = row0 + x * kStep;
                            uint4 lo, hi;
                            fp8x4_to_f16<MODE>(code[x].x, lo.x, lo.y);
                            fp8x4_to_f16<MODE>(code[x].y, lo.z, lo.w);
                            fp8x4_to_f16<MODE>(code[x].z, hi.x, hi.y);
                            fp8x4_to_f16<MODE>(code[x].w, hi.z, hi.w);
                            const uint32_t at0 = to + place(K::T, r, 2 * piece), at1 = to + place(K::T, r, 2 * piece + 1);
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at0), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
                            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at1), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
                        }
                    }
                    ++unit;
                    tell();
                }
            }
        }
        more = run.next(a);
    }
    if constexpr (!K::kFp8) {
        cp_async_wait<0>();
        while (told < unit) tell();
    }
}

// One thread issues every product.  Step x of an item: group x & 1 at tile x / 2 (dual) or x.
template <class K>
__device__ __forceinline__ void multiply(const PrefixArgs& a, typename K::Shared& sh, uint32_t ring, uint32_t queries, uint32_t tmem,
                                         Run<K> run) {
    const uint32_t of_s = product(K::kBf16, K::T, false);
    const int wide = (a.head_dim + 15) / 16;  // products of 16 along head_dim, and columns of O in 16s
    const uint32_t of_o = product(K::kBf16, wide * 16, true);
    uint32_t unit = 0;                               // first unit of the item at hand
    uint32_t s_steps[2] = {0, 0}, o_steps[2] = {0, 0}, q_items[2] = {0, 0};
    bool more = true;
    while (more) {
        const bool dual = run.dual();
        const int32_t steps = run.steps();
        auto tile_of = [&](int32_t x) { return dual ? x >> 1 : x; };
        auto scores = [&](int32_t x) {
            const int b = x & 1, s = K::kStreams == 2 ? b : 0;
            if (x < K::kStreams) {  // the group's queries of this item
                wait(&sh.abandoned, &sh.q_full[s], q_items[s] & 1u);
                ++q_items[s];
            }
            // its weights of the step before, in S's place, have been used
            if (o_steps[b] > 0) wait(&sh.abandoned, &sh.o_done[b], (o_steps[b] - 1) & 1u);
            const uint32_t u = unit + 2 * tile_of(x), stage = u % K::kStages;
            wait(&sh.abandoned, &sh.full[stage], u / K::kStages & 1u);
            tc_fence_after();
            const uint32_t keys = ring + stage * K::kUnit, q = queries + s * K::kQ;
            for (int c = 0; c < wide; ++c)
                mma_ss(tmem + b * K::T, operand(q + (c >> 2) * (128 * 128) + (c & 3) * 32, 16, 1024),
                       operand(keys + (c >> 2) * (K::T * 128) + (c & 3) * 32, 16, 1024), of_s, c > 0);
            tc_commit(&sh.s_full[b]);
            ++s_steps[b];
            if (!dual || b == 1) tc_commit(&sh.empty[stage]);
        };
        for (int32_t x = 0; x < 2 && x < steps; ++x)
            scores(x);
        for (int32_t x = 0; x < steps; ++x) {
            const int b = x & 1, s = K::kStreams == 2 ? b : 0;
            wait(&sh.abandoned, &sh.p_full[b], (s_steps[b] - 1) & 1u);
            const uint32_t u = unit + 2 * tile_of(x) + 1, stage = u % K::kStages;
            wait(&sh.abandoned, &sh.full[stage], u / K::kStages & 1u);
            tc_fence_after();
            const uint32_t values = ring + stage * K::kUnit, o = tmem + K::kO + s * K::kDim;
            const bool first = x < K::kStreams;  // of the group's steps in this item
#pragma unroll 1
            for (int c = 0; c < K::T / 16; ++c) {
                const uint64_t rows = operand(values + c * 2048, K::T * 128, 1024);
                // 32 tokens' weights: 16 columns of high terms, 16 of low ones
                const uint32_t p = tmem + b * K::T + (c >> 1) * 32 + (c & 1) * 8;
                mma_ts(o, p, rows, of_o, !first || c > 0);
                mma_ts(o, p + 16, rows, of_o, true);
            }
            tc_commit(&sh.o_done[b]);
            ++o_steps[b];
            if (!dual || b == 1) tc_commit(&sh.empty[stage]);
            if (x + 2 < steps) scores(x + 2);
        }
        unit += 2 * run.n;
        more = run.next(a);
    }
}

template <class K>
__device__ __forceinline__ void soften(const PrefixArgs& a, typename K::Shared& sh, unsigned char* queries, uint32_t tmem, Run<K> run) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3, stream = K::kStreams == 2 ? threadIdx.x >> 7 : 0;
    const int my_row = threadIdx.x & 127;
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    unsigned char* my_q = queries + stream * K::kQ;
    const uint32_t o_at = lanes + K::kO + stream * K::kDim;
    uint32_t s_steps[2] = {0, 0}, o_steps[2] = {0, 0};
    int32_t tile0 = 0;
    const float cap = a.softcap * kLog2e;
    bool more = true;
    while (more) {
        const bool dual = run.dual();
        const int32_t steps = run.steps();
        const int32_t rows = dual ? min(128, run.rows - 128 * stream) : run.rows;
        const bool busy = warp * 32 < rows;  // this warp has rows
        const bool valid = my_row < rows;
        // this row: request and query head
        const uint32_t nth = static_cast<uint32_t>(run.block * K::kRows + (dual ? 128 * stream : 0) + (valid ? my_row : 0));
        const int32_t member = nth / a.group, r = run.of.start + member, h = run.kv * a.group.d + (nth - member * a.group.d);
        float scale = a.scale * (a.k_scale ? a.k_scale[run.kv] : 1.0f);
        float m = -INFINITY, less = 0.0f, high = -INFINITY, l = 0.0f;
        if (stream < steps) {
            // the queries into shared memory
            const char* q = a.q + 2 * (r * a.q_req + h * a.q_head);
            const int pieces = a.head_dim / 8;
            auto piece = [&](int c) {
                if (a.q_wide) return *reinterpret_cast<const uint4*>(q + 16 * c);
                const uint32_t* w = reinterpret_cast<const uint32_t*>(q + 16 * c);
                return make_uint4(w[0], w[1], w[2], w[3]);
            };
            float fit = 1.0f;
            if constexpr (K::kFp8) {
                // f16 queries, scaled by a power of two to a largest magnitude in [1, 2)
                float top = 0.0f;
                if (valid)
                    for (int c = 0; c < pieces; ++c) {
                        const uint4 v = piece(c);
                        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(w[x], f0, f1);
                            else unpack2<true>(w[x], f0, f1);
                            top = fmaxf(top, fmaxf(fabsf(f0), fabsf(f1)));
                        }
                    }
                const uint32_t field = __float_as_uint(top) >> 23;  // biased exponent
                if (field >= 1 && field <= 254) {
                    const uint32_t e = min(field, 253u);
                    fit = __uint_as_float((254u - e) << 23);
                    scale *= __uint_as_float(e << 23);
                }
            }
            for (int c = 0; c < K::kPanels * 8; ++c) {
                uint4 v = make_uint4(0, 0, 0, 0);
                if (valid && c < pieces) {
                    v = piece(c);
                    if constexpr (K::kFp8) {
                        uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(w[x], f0, f1);
                            else unpack2<true>(w[x], f0, f1);
                            w[x] = pack2<false>(f0 * fit, f1 * fit);
                        }
                        v = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
                *reinterpret_cast<uint4*>(my_q + place(128, my_row, c)) = v;
            }
            fence_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[stream]);
        }
        scale = a.softcap > 0.0f ? __fdiv_rn(scale, a.softcap) * (2.0f * kLog2e) : scale * kLog2e;
        const int32_t len = valid ? a.lens[r] : 0;
        const uint32_t end = max(min(len, run.of.shared), 0), begin = a.window > 0 && len > a.window ? len - a.window : 0;
        const float slope = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
        for (int32_t x = K::kStreams == 2 ? stream : 0; x < steps; x += K::kStreams) {
            const int b = x & 1;
            const int32_t tile = dual ? x >> 1 : x;
            wait(&sh.abandoned, &sh.s_full[b], s_steps[b] & 1u);
            __syncwarp();
            ++s_steps[b];
            const uint32_t s_at = lanes + b * K::T;
            tc_fence_after();
            if (busy) {
                const uint32_t* words = sh.mask[(tile0 + tile) % kMasks];
                const uint32_t first = static_cast<uint32_t>(run.t + tile) * K::T;
                bool whole = first >= begin && first + K::T <= end;
#pragma unroll
                for (int c = 0; c < K::T / 32; ++c) whole &= words[c] == 0xffffffffu;
                const bool plain = __all_sync(0xffffffffu, (whole || !valid) && scale >= 0.0f) && a.softcap == 0.0f && a.slopes == nullptr;
                float top = -INFINITY;
                uint32_t v[32];
                if (plain) {
#pragma unroll
                    for (int c = 0; c < K::T / 32; ++c) {
                        tm_load(v, s_at + c * 32);
                        tc_wait_ld();
                        float t0 = -INFINITY, t1 = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            t0 = fmaxf(t0, __uint_as_float(v[i]));
                            t1 = fmaxf(t1, __uint_as_float(v[i + 1]));
                        }
                        top = fmaxf(top, fmaxf(t0, t1));
                    }
                    top *= scale;
                } else {
                    // scores as they count, put back in the place of the products
#pragma unroll 1
                    for (int c = 0; c < K::T / 32; ++c) {
                        tm_load(v, s_at + c * 32);
                        tc_wait_ld();
                        const uint32_t word = words[c];
                        const uint32_t tok = first + c * 32;
#pragma unroll
                        for (int i = 0; i < 32; ++i) {
                            float p = __uint_as_float(v[i]) * scale;
                            if (a.softcap > 0.0f) p = fabsf(p) < kSmallCapped ? cap_small(p, a.softcap) : cap_large(p, cap);
                            if (a.slopes) p = __fmaf_rn(slope, static_cast<float>(static_cast<int32_t>(tok + i) - (len - 1)), p);
                            const bool seen = (word >> i & 1u) && tok + i >= begin && tok + i < end;
                            p = seen ? p : -INFINITY;
                            v[i] = __float_as_uint(p);
                            top = fmaxf(top, p);
                        }
                        tm_store(s_at + c * 32, v);
                    }
                    tc_wait_st();
                }
                const float by = plain ? scale : 1.0f;
                if (__any_sync(0xffffffffu, valid && top > high)) {
                    float less_before = m;
                    if (top > high) {
                        m = fmaxf(top - K::kBelow, m);
                        high = __fadd_rd(m, K::kAbove);  // down: 2^16 would be past f16
                        less = m == -INFINITY ? 0.0f : m;
                    }
                    const float f = rescale(less_before, m);
                    l *= f;
                    if (x >= K::kStreams) {
                        // O of the steps before is complete
                        const int pb = K::kStreams == 2 ? b : (x - 1) & 1;
                        wait(&sh.abandoned, &sh.o_done[pb], (o_steps[pb] - 1) & 1u);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll 1
                        for (int c = 0; c < K::kDim; c += 32) {
                            if (c >= a.head_dim) break;
                            tm_load(v, o_at + c);
                            tc_wait_ld();
#pragma unroll
                            for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * f);
                            tm_store(o_at + c, v);
                        }
                        tc_wait_st();
                    }
                }
                float sum = 0.0f;
#pragma unroll 1
                for (int c = 0; c < K::T / 32; ++c) {
                    tm_load(v, s_at + c * 32);
                    tc_wait_ld();
                    float s0 = 0.0f, s1 = 0.0f;
                    uint32_t w[32];
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float p0 = exp2_fast(__fmaf_rn(__uint_as_float(v[2 * i]), by, -less));
                        const float p1 = exp2_fast(__fmaf_rn(__uint_as_float(v[2 * i + 1]), by, -less));
                        s0 += p0;
                        s1 += p1;
                        w[i] = pack2<K::kBf16>(p0, p1);
                        float h0, h1;
                        unpack2<K::kBf16>(w[i], h0, h1);
                        w[16 + i] = pack2<K::kBf16>(p0 - h0, p1 - h1);
                    }
                    sum += s0 + s1;
                    tm_store(s_at + c * 32, w);
                }
                l += sum;
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[b]);
            ++o_steps[b];
        }
        // this CTA's part of the row
        const bool first = run.t == 0;
        if (steps > stream) {
            const int32_t last = steps - 1 - ((steps - 1 - stream) % K::kStreams);
            const int b = last & 1;
            wait(&sh.abandoned, &sh.o_done[b], (o_steps[b] - 1) & 1u);
            __syncwarp();
            tc_fence_after();
        }
        const bool has = steps > stream;
        if (valid && (first || has || !dual)) {
            const int half = dual ? 0 : stream;
            const int64_t row = (static_cast<int64_t>(r) + static_cast<int64_t>(half) * a.n_requests) * a.q_heads + h;
            const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + stream) * 128 + my_row;
            if (first) a.part_ml[row] = make_float2(m, has ? l : 0.0f);
            else a.cta_ml[slot] = make_float2(m, has ? l : 0.0f);
        }
        if (busy && has) {
            const int half = dual ? 0 : stream;
            const int64_t row = (static_cast<int64_t>(r) + static_cast<int64_t>(half) * a.n_requests) * a.q_heads + h;
            const int64_t slot = (static_cast<int64_t>(blockIdx.x) * 2 + stream) * 128 + my_row;
            float* to = first ? a.part + row * a.head_dim : a.cta_part + slot * a.head_dim;
#pragma unroll 1
            for (int c = 0; c < a.head_dim; c += 32) {
                uint32_t v[32];
                tm_load(v, o_at + c);
                tc_wait_ld();
                if (valid) {
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        if (c + i < a.head_dim) *reinterpret_cast<uint4*>(to + c + i) = make_uint4(v[i], v[i + 1], v[i + 2], v[i + 3]);
                }
            }
            tc_fence_before();
        }
        tile0 += run.n;
        more = run.next(a);
    }
}

template <int MODE, int DP>
__global__ void __launch_bounds__(Prefix<MODE, DP>::kThreads, 1) prefix_kernel(const PrefixArgs a) {
    using K = Prefix<MODE, DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* queries = smem + K::kStages * K::kUnit;
    auto& sh = *reinterpret_cast<typename K::Shared*>(queries + K::kStreams * K::kQ);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int kWarps = K::kThreads / 32, kIssuer = kWarps - 1;
    after_previous();
    let_next_start();
    if (tid == 0) {
        for (int i = 0; i < K::kStages; ++i) {
            mbar_init(&sh.full[i], kProducers / 32);
            mbar_init(&sh.empty[i], 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.p_full[i], 4);
            mbar_init(&sh.o_done[i], 1);
            mbar_init(&sh.q_full[i], 4);
        }
        mbar_init(&sh.drained, 1);
        fence_barrier_init();
        sh.abandoned = 0;
    }
    // the tiles of thread i's `per` consecutive groups, in a row
    int64_t* sums = reinterpret_cast<int64_t*>(smem);  // [threads + 1], before the ring is used
    const int32_t per = (a.n_groups + K::kThreads - 1) / K::kThreads;
    int64_t mine = 0;
    bool bad = false;
    for (int32_t i = 0; i < per; ++i) {
        const int32_t g = tid * per + i;
        if (g >= a.n_groups) break;
        const Group x = group_of(a, g);
        bad |= x.bad;
        mine += items_of<K>(a, x) * tiles_of<K>(x);
    }
    bad = __syncthreads_or(bad);
    sums[tid] = mine;
    __syncthreads();
    if (warp == 0) {
        int64_t front = 0;
        for (int t0 = 0; t0 < K::kThreads; t0 += 32) {
            int64_t upto = sums[t0 + lane];
            const int64_t own = upto;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
                if (lane >= d) upto += x;
            }
            sums[t0 + lane] = front + upto - own;
            front += __shfl_sync(0xffffffffu, upto, 31);
        }
        if (lane == 0) sums[K::kThreads] = front;
    }
    __syncthreads();
    int64_t total64 = sums[K::kThreads];
    if (bad || total64 > 0x7fffffff) {
        // nothing is shared then: every request reads all of its tokens
        if (tid == 0) atomicExch(a.status, MF_DEVICE_TOO_LARGE);
        bad = true;
        total64 = 0;
    }
    const int32_t total = static_cast<int32_t>(total64), ctas = min(total, static_cast<int32_t>(gridDim.x));
    // what the other launches need to know
    if (blockIdx.x == 0 && tid == 0) *a.cut = make_int2(total, ctas);
    const int32_t begin = bad || a.n_groups == 0 ? a.n_requests : a.starts[0], end = bad || a.n_groups == 0 ? a.n_requests : a.starts[a.n_groups];
    for (int32_t r = blockIdx.x * K::kThreads + tid; r < a.n_requests; r += gridDim.x * K::kThreads)
        if (r < begin || r >= end) {
            a.own_first[r] = 0;
            a.info[r] = Shared{0, 0, 0, 0};
        }
    if (!bad)
        for (int32_t g = blockIdx.x; g < a.n_groups; g += gridDim.x) {
            const Group x = group_of(a, g);
            int64_t base = sums[g / max(per, 1)];
            for (int32_t b = g / per * per; b < g; ++b) {
                const Group y = group_of(a, b);
                base += items_of<K>(a, y) * tiles_of<K>(y);
            }
            for (int32_t i = tid; i < x.members; i += K::kThreads) {
                a.own_first[x.start + i] = x.shared;
                a.info[x.start + i] = Shared{static_cast<int32_t>(base), tiles_of<K>(x), x.start, x.members};
            }
        }
    if (static_cast<int32_t>(blockIdx.x) >= ctas) return;
    const Cut cut(total, ctas);
    const int32_t x0 = cut.start(blockIdx.x), run_of = cut.start(blockIdx.x + 1) - x0;
    const bool here = sums[tid] <= x0 && x0 < sums[tid] + mine;
    if (here) {
        int32_t into = x0 - static_cast<int32_t>(sums[tid]);
        for (int32_t g = tid * per;; ++g) {
            const Group x = group_of(a, g);
            const int64_t of = items_of<K>(a, x) * tiles_of<K>(x);
            if (into < of) {
                sh.group = g;
                sh.into = into;
                break;
            }
            into -= static_cast<int32_t>(of);
        }
    }
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem, ring = smem_u32(smem);
    // what is past the head in a row is never copied: zeros
    if (a.head_dim < DP) {
        for (int i = tid; i < K::kStages * K::kUnit / 16; i += K::kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy();
    }
    const Run<K> run(a, sh.group, sh.into, run_of);
    __syncthreads();
    if (tid < K::kSoftmax) soften<K>(a, sh, queries, tmem, run);
    else if (tid < K::kSoftmax + kProducers) produce<K, MODE>(a, sh, ring, run);
    else if (lane == 0) {
        multiply<K>(a, sh, ring, smem_u32(queries), tmem, run);
        // the products read shared and tensor memory until here
        tc_commit(&sh.drained);
        const uint64_t until = global_ns() + kWaitNs;
        while (!mbar_try_wait(&sh.drained, 0) && global_ns() < until) {
        }
    }
    if (warp > K::kSoftmax / 32 - 1 && warp < kIssuer) cp_async_wait<0>();
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.abandoned) atomicExch(a.status, MF_DEVICE_TIMEOUT);
    if (warp == kIssuer) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ------------------------------------------------------------------ the join

constexpr int kJoinThreads = 256;

// A warp for each query head of a request.  ROWS: of a block; DUAL: whether blocks of more than 128 rows are two; BELOW: what a
// weight of a maximum is, a power of two.
template <int ROWS, bool F16>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const PrefixArgs a) {
    constexpr float kBelow = F16 ? 12.0f : 0.0f, kMost = F16 ? 4096.0f : 1.0f;
    const int lane = threadIdx.x & 31;
    after_previous();
    let_next_start();
    const int64_t n = static_cast<int64_t>(a.n_requests) * a.q_heads;
    const int2 all = *a.cut;
    for (int64_t w = (static_cast<int64_t>(blockIdx.x) * kJoinThreads + threadIdx.x) >> 5; w < n; w += static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32)) {
        const int32_t r = static_cast<int32_t>(w / a.q_heads), h = static_cast<int32_t>(w - static_cast<int64_t>(r) * a.q_heads);
        const Shared x = a.info[r];
        // its own tokens as a part whose largest weight is kMost, too
        const float own = a.own_lse[w];
        float top = own * kLog2e - kBelow;
        int32_t parts = 0, first = 0, slot = 0;
        bool dual = false;
        if (x.tiles > 0) {
            const int32_t kv = h / a.group.d;
            const int64_t nth = static_cast<int64_t>(r - x.start) * a.group.d + (h - kv * a.group.d), rows = static_cast<int64_t>(x.members) * a.group.d;
            const int32_t blocks = static_cast<int32_t>((rows + ROWS - 1) / ROWS), block = static_cast<int32_t>(nth / ROWS);
            const int32_t row = static_cast<int32_t>(nth - static_cast<int64_t>(block) * ROWS);
            dual = ROWS == 256 && rows - static_cast<int64_t>(block) * ROWS > 128;
            const Cut cut(all.x, all.y);
            const int32_t begin = x.base + (kv * blocks + block) * x.tiles;
            first = cut.part_of(begin);
            parts = cut.part_of(begin + x.tiles - 1) - first + 1;
            slot = row;  // of the 2 x 128 of a CTA: the second half of a dual block, too
        }
        const int halves = dual || ROWS == 128 ? 1 : 2;
        auto ml_of = [&](int32_t p, int half) {
            return p == 0 ? a.part_ml[(static_cast<int64_t>(half) * a.n_requests + r) * a.q_heads + h]
                          : a.cta_ml[static_cast<int64_t>(first + p) * 256 + half * 128 + slot];
        };
        for (int32_t p = 0; p < parts; ++p)
            for (int half = 0; half < halves; ++half) {
                const float2 ml = ml_of(p, half);
                if (ml.y != 0.0f) top = fmaxf(top, ml.x);
            }
        // a NaN anywhere shows in the sum
        const float vs = a.v_scale ? a.v_scale[h / a.group.d] : 1.0f;
        const float own_w = own == -INFINITY ? 0.0f : kMost * exp2_fast(own * kLog2e - kBelow - top);
        float sum = own_w;
        float acc[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            acc[i] = d < a.head_dim && own_w != 0.0f ? a.own[w * a.head_dim + d] * own_w : 0.0f;
        }
        for (int32_t p = 0; p < parts; ++p)
            for (int half = 0; half < halves; ++half) {
                const float2 ml = ml_of(p, half);
                if (ml.y == 0.0f) continue;
                const float by = rescale(ml.x, top);
                sum = __fmaf_rn(ml.y, by, sum);
                const float* from = p == 0 ? a.part + ((static_cast<int64_t>(half) * a.n_requests + r) * a.q_heads + h) * a.head_dim
                                           : a.cta_part + (static_cast<int64_t>(first + p) * 256 + half * 128 + slot) * a.head_dim;
                const float weight = by * vs;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const int d = lane + 32 * i;
                    if (d < a.head_dim) acc[i] = __fmaf_rn(from[d], weight, acc[i]);
                }
            }
        const float inv = sum == 0.0f ? 0.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int d = lane + 32 * i;
            if (d >= a.head_dim) break;
            const uint32_t two = a.q_f16 ? pack2<false>(acc[i] * inv, 0.0f) : pack2<true>(acc[i] * inv, 0.0f);
            *reinterpret_cast<uint16_t*>(a.out + 2 * (r * a.out_req + h * a.out_head + d)) = static_cast<uint16_t>(two);
        }
        if (lane == 0 && a.lse) a.lse[w] = sum == 0.0f ? -INFINITY : (top + kBelow + log2f(sum * (1.0f / kMost))) * kLn2;
    }
}

// ------------------------------------------------------------------ host

struct Kernel {
    void (*fn)(PrefixArgs);
    void (*join)(PrefixArgs);
    int threads, shared;
};
template <int MODE, int DP>
Kernel kernel_of() {
    using K = Prefix<MODE, DP>;
    static_assert(K::kBytes <= 232448, "shared memory of one CTA");
    return Kernel{prefix_kernel<MODE, DP>, join_kernel<K::kRows, !K::kBf16>, K::kThreads, K::kBytes};
}
template <int MODE>
Kernel pick_dim(int head_dim) {
    return head_dim <= 64 ? kernel_of<MODE, 64>() : head_dim <= 128 ? kernel_of<MODE, 128>() : kernel_of<MODE, 256>();
}
Kernel pick(int dtype, int head_dim) {
    switch (dtype) {
    case MF_DT_BF16: return pick_dim<MF_DT_BF16>(head_dim);
    case MF_DT_F16: return pick_dim<MF_DT_F16>(head_dim);
    case MF_DT_F8E4M3: return pick_dim<MF_DT_F8E4M3>(head_dim);
    default: return pick_dim<MF_DT_F8E5M2>(head_dim);
    }
}

}  // namespace
}  // namespace mf

using namespace mf;

struct mf_prefix_attn_s {
    mf_paged_attn own;  // the requests' own tokens
    Kernel kernel;
    PrefixArgs args;
    void* workspace;
    int device, ctas;
    int32_t max_requests;
};

extern "C" int mf_prefix_attn_create(const mf_paged_attn_config* config, int32_t max_requests, mf_prefix_attn* handle) {
    MF_ENTER();
    if (!config || !handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_create: NULL argument");
    *handle = nullptr;
    if (max_requests <= 0 || max_requests > kMaxRequests)
        return fail(MF_ERR_SHAPE_INVALID, "mf_prefix_attn_create: %d requests (1 to 2^31 - 2^16)", max_requests);
    mf_paged_attn own = nullptr;
    int rc = mf_paged_attn_create(config, &own);  // checks the description
    if (rc == MF_OK) rc = paged_attn_enable_parts(own);
    if (rc != MF_OK) {
        mf_paged_attn_destroy(own);
        return rc;
    }
    const mf_paged_attn_config& c = *config;
    const mf_cache_layout& k = c.cache;
    const Kernel kernel = pick(k.dtype, k.head_dim);
    cudaError_t err = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, kernel.shared);
    const int ctas = state().sm_count;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t heads = static_cast<size_t>(max_requests) * c.q_heads;
    const size_t firsts = up(static_cast<size_t>(max_requests) * 4), infos = up(static_cast<size_t>(max_requests) * sizeof(Shared));
    const size_t parts = up(2 * heads * k.head_dim * 4), part_mls = up(2 * heads * 8);
    const size_t cta_parts = up(static_cast<size_t>(ctas) * 256 * k.head_dim * 4), cta_mls = up(static_cast<size_t>(ctas) * 256 * 8);
    const size_t owns = up(heads * k.head_dim * 4), lses = up(heads * 4);
    const size_t bytes = 256 + firsts + infos + parts + part_mls + cta_parts + cta_mls + owns + lses;
    mf_prefix_attn_s* h = err == cudaSuccess ? new (std::nothrow) mf_prefix_attn_s{} : nullptr;
    if (!h) {
        mf_paged_attn_destroy(own);
        return err != cudaSuccess ? cuda_fail(err, "mf_prefix_attn_create: cudaFuncSetAttribute")
                                  : fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_prefix_attn_create: out of host memory");
    }
    err = cudaMalloc(&h->workspace, bytes);
    PrefixArgs& a = h->args;
    a.status = err == cudaSuccess ? sticky_status_ptr() : nullptr;
    if (!a.status) {
        cudaGetLastError();
        if (err == cudaSuccess) cudaFree(h->workspace);
        delete h;
        mf_paged_attn_destroy(own);
        if (err == cudaErrorMemoryAllocation)
            return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_prefix_attn_create: %zu bytes: out of device memory", bytes);
        return err != cudaSuccess ? cuda_fail(err, "mf_prefix_attn_create: cudaMalloc")
                                  : fail(MF_ERR_CUDA, "mf_prefix_attn_create: sticky status word unavailable");
    }
    const int code = is_fp8(k.dtype) ? 1 : 2;
    char* w = static_cast<char*>(h->workspace);
    h->own = own;
    h->kernel = kernel;
    h->device = state().device;
    h->ctas = ctas;
    h->max_requests = max_requests;
    a.max_pages = c.max_pages;
    a.page = k.page_size;
    a.window = c.window;
    a.kv_heads = k.kv_heads;
    a.page_bytes = k.page_stride * code;
    a.row_bytes = k.token_stride * code;
    a.head_bytes = k.head_stride * code;
    a.table_stride = c.table_stride;
    a.n_pages = static_cast<uint32_t>(k.n_pages < 0x7fffffff ? k.n_pages : 0x7fffffff);
    a.by_page = divisor(k.page_size);
    a.group = divisor(c.q_heads / k.kv_heads);
    a.head_dim = k.head_dim;
    a.q_req = c.q_token_stride;
    a.q_head = c.q_head_stride;
    a.q_heads = c.q_heads;
    a.q_f16 = c.q_dtype == MF_DT_F16;
    a.scale = c.scale;
    a.softcap = c.softcap;
    a.slopes = c.slopes;
    a.k_scale = is_fp8(k.dtype) ? c.k_scale_inv : nullptr;
    a.v_scale = is_fp8(k.dtype) ? c.v_scale_inv : nullptr;
    a.out_req = c.out_token_stride;
    a.out_head = c.out_head_stride;
    a.cut = reinterpret_cast<int2*>(w);
    a.own_first = reinterpret_cast<int32_t*>(w += 256);
    a.info = reinterpret_cast<Shared*>(w += firsts);
    a.part = reinterpret_cast<float*>(w += infos);
    a.part_ml = reinterpret_cast<float2*>(w += parts);
    a.cta_part = reinterpret_cast<float*>(w += part_mls);
    a.cta_ml = reinterpret_cast<float2*>(w += cta_parts);
    a.own = reinterpret_cast<float*>(w += cta_mls);
    a.own_lse = reinterpret_cast<float*>(w += owns);
    *handle = h;
    return MF_OK;
}

extern "C" int mf_prefix_attn_run(mf_prefix_attn handle, const void* q, const void* k_cache, const void* v_cache,
                                  const int32_t* table, const int32_t* lens, int32_t n_requests, const int32_t* starts,
                                  const int32_t* shared, int32_t n_groups, void* out, float* lse, mf_stream stream) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_run: handle is NULL");
    if (handle->device != state().device)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_run: the handle belongs to device %d", handle->device);
    if (n_requests < 0 || n_requests > handle->max_requests)
        return fail(MF_ERR_SHAPE_INVALID, "mf_prefix_attn_run: %d requests (0 to %d)", n_requests, handle->max_requests);
    if (n_groups < 0 || n_groups > kMaxRequests)
        return fail(MF_ERR_SHAPE_INVALID, "mf_prefix_attn_run: %d groups (0 to 2^31 - 2^16)", n_groups);
    if (n_requests == 0) return MF_OK;
    if (!q || !k_cache || !v_cache || !table || !lens || !out || (n_groups > 0 && (!starts || !shared)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_run: NULL buffer");
    if (!aligned16(k_cache) || !aligned16(v_cache))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_prefix_attn_run: cache buffers must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(q) % 4 || reinterpret_cast<uintptr_t>(out) % 8)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_prefix_attn_run: q must be 4-byte and out 8-byte aligned");
    PrefixArgs a = handle->args;
    a.q = static_cast<const char*>(q);
    a.q_wide = aligned16(q) && a.q_req % 8 == 0 && a.q_head % 8 == 0;
    a.k = static_cast<const char*>(k_cache);
    a.v = static_cast<const char*>(v_cache);
    a.table = table;
    a.lens = lens;
    a.n_requests = n_requests;
    a.starts = starts;
    a.shared = shared;
    a.n_groups = n_groups;
    a.out = static_cast<char*>(out);
    a.lse = lse;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t err = launch_overlapped(handle->kernel.fn, dim3(static_cast<unsigned>(handle->ctas)), handle->kernel.threads,
                                        handle->kernel.shared, s, a);
    if (err != cudaSuccess) return cuda_fail(err, "mf_prefix_attn_run");
    const int rc = paged_attn_run_parts(handle->own, q, k_cache, v_cache, table, lens, n_requests, a.own_first, a.own, a.own_lse, s);
    if (rc != MF_OK) return rc;
    const int64_t grid = stream_grid(static_cast<int64_t>(n_requests) * a.q_heads * 32, kJoinThreads, 8);
    err = launch_overlapped(handle->kernel.join, dim3(static_cast<unsigned>(grid)), kJoinThreads, 0, s, a);
    if (err != cudaSuccess) return cuda_fail(err, "mf_prefix_attn_run");
    return MF_OK;
}

extern "C" int mf_prefix_attn_destroy(mf_prefix_attn handle) {
    if (!handle) return MF_OK;
    const cudaError_t err = free_workspace(handle->device, handle->workspace);
    const int rc = mf_paged_attn_destroy(handle->own);
    delete handle;
    if (err != cudaSuccess) return cuda_fail(err, "mf_prefix_attn_destroy");
    return rc;
}
