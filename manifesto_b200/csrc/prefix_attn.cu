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
//   * one warp finds the rows of the tiles to come through the page table;
//   * four producer warps copy keys and values, tile by tile, into a ring in
//     shared memory (16-byte cp.async in the 128-byte swizzle that the products
//     read; FP8 codes wait in a ring of their own and become f16 there, exactly),
//     masked rows zero-filled;
//   * one warp issues the products: S into tensor memory, P (from tensor memory)
//     times V into the accumulator O in tensor memory;
//   * two groups of four softmax warps, a thread for each row, turn S into P in
//     place: running maximum and sum in float32, P as two 16-bit terms (high and
//     low: what the two leave out of a weight is 2^-16 of it in BF16, 2^-22 in
//     f16), O rescaled only when a
//     maximum has grown by more than 2^8 (f16: 2^15);
//   * one warp writes down for the other launches what each request shares.
// The groups alternate, so that one's softmax runs beside the other's products: of
// more than 128 rows each has 128 and sees every tile, else both have the same
// rows and every second tile.  Up to 64 rows stand in tensor memory two or four
// times over, and a tile's tokens are shared out among the warps that hold them
// (24 prompts of 8 beams over E4M3, 32 rows: 404 -> 326 us at that time, when
// FP8 caches had one term of the weights; now 150, 148 with one).  The
// tiles of all (group, block of rows, key-value head) items in a row are cut evenly
// for the CTAs, an item counting four tiles more than it has (without them items of
// two tiles filled a CTA's whole share: 240 -> 146 us, with the parts' layout); every CTA leaves the part of
// its run, and the last launch joins a row's parts in the order of the tokens.
//
// A masked token's weight is 0, and 0 times a value that is not finite is NaN in the
// row's sums, though the row does not see it (a shorter request, a token in front of
// a window).  So a row that ends with such a number marks its request for the call,
// and the second launch reads all of that request's tokens, masked ones not at all.
//
// Measured (B200): 250 requests behind 8192 shared tokens, 32/8 heads of 128, BF16: 170 us for the whole call,
// this kernel 72 from cold caches (the products at the measured rate of the tensor cores: 20 us,
// 31 with the low terms), tensor pipe 38% of the time busy.  Bound by latency: a
// step's chain is some 5 thousand clocks (scores 0.5, softmax 2.4 to 3, values 1.0,
// the rest hand-overs; read in an instrumented copy, which is slower itself), two
// such chains run at a time, and the issuer waits for a step's products before it
// lets the next scores into their place.  24 prompts of 8 beams, prefixes ragged to
// 6000 tokens, E4M3: 149 us, 107 from cold caches (23 to read the codes), tensor pipe 32%.  Copies of an
// earlier form that skipped work: of 168 us, no softmax 154, no parts written 158, no
// copies 161; of 141 us over E4M3, then with one term of the weights, no copies 121, no
// softmax 125, no parts written 130, no conversions 147.
#include <new>

#include "mf_async.cuh"
#include "mf_attn.cuh"
#include "mf_divisor.cuh"
#include "mf_internal.h"
#include "mf_launch.cuh"
#include "mf_runtime.h"

namespace mf {
namespace {

// What the join needs of a request's group: the place of its first item, tiles of an item (0: nothing is shared), its first
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
    int32_t reach;  // tokens that a row of the table holds, 2^31 - 1 at most
    int32_t page, window, kv_heads;
    const char* k;
    const char* v;
    int64_t head_bytes, table_stride;
    uint32_t page_units, row_units, unit;  // a page, a row of it in units of `unit` bytes, a power of two
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
    int32_t always;       // share whatever can be shared
    float token_ps;       // of reading a token again, see kItemPs
    uint32_t wait_ns;     // that a wait may last
    // workspace
    int32_t* own_first;   // [requests]
    int32_t* kept;        // [requests], by a group's first: the tokens that it shares; every CTA writes the same, for itself
    Shared* info;         // [requests]
    int2* cut;            // places of all items, CTAs that they are cut for
    uint32_t* call;       // the number of the call, for the launches behind the first; of the last call that came to its end
    uint32_t* alone;      // [requests]: the number of the call that found a number that is not finite, see soften
    float* part;          // [2][requests][q_heads][head_dim]: an item's first CTA, its two halves
    float2* part_ml;      // [2][requests][q_heads]
    float* cta_part;      // [CTAs][2][128][head_dim]: a CTA that begins inside an item
    float2* cta_ml;       // [CTAs][2][128]
    float* own;           // [requests][q_heads][head_dim]: the requests' own tokens
    float2* own_ml;       // [requests][q_heads]: their maximum and sum, as part_ml's
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
__device__ __forceinline__ void tm_load16(uint32_t (&r)[16], uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : MF_R8(r, 0), MF_R8(r, 8)
                 : "r"(at)
                 : "memory");
}
__device__ __forceinline__ void tm_store16(uint32_t at, const uint32_t (&r)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(at), MF_I8(r, 0),
                 MF_I8(r, 8)
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

// Four groups of four warps: softmax, softmax, producers, and single ones (the products' issuer, the pages', the notes').  The
// registers of the launch (128 each) go where a row of scores is held: 128 x (192 + 192 + 64 + 64) = 512 x 128.
constexpr int kThreads = 512;
constexpr int kProducers = 128, kFirstProducer = 256, kIssuer = 12, kPager = 13, kNoter = 14;
constexpr int kSoftmaxRegs = 192, kProducerRegs = 64, kOtherRegs = 64;
constexpr int kPlaces = 4;  // tiles whose rows are known in advance
constexpr int kMasks = 16;  // tiles whose masks are kept: more than the ring and the places hold

// How long the waits of a CTA may last, and whether one has run out.
struct Waits {
    uint32_t ns;
    int32_t abandoned;
};

// Shared tokens of a group, and its requests; nothing is shared by a request alone, nor where it does not pay.
struct Group {
    int32_t start, members, shared;
    bool bad;
};
// Whether a group's tokens are shared, and whether any are.  The requests of a group follow one another, so that its tokens come
// out of L2 for all but one of them: reading them again, as far as each of the others sees them (its length, its window), costs
// 8 + 0.32 ps an element of a head a token and key-value head with all SMs at work (of FP8 codes 0.64 of that), an item of shared
// tokens 90 ns, a tile, seen or not, 3 (8 with more than 128 rows; four times as much where a window takes the way of masked
// tiles), and the first of them all 28 us.  The prices are fitted to 1176 cases with cold caches, both ways timed: 7 shapes of heads
// of 64 to 256, BF16 and E4M3, 1 to 100 groups of 2 to 250 requests with 48 to 8192 tokens, windows, idle requests.  Calls by the
// rule take a tenth and 6 us more than the better way in 79 of them (1.4 times at most).  32/8 heads of 128, BF16, us with sharing and
// without: 100 groups of 2 that share 48 tokens 84 and 39, 30 of 16 with 48 83 and 54, with 800 106 and 180; one of 4 with 896 32
// and 20; one of 250 with 8192 135 and 643, with a window of 128 136 and 40, with 2 of the 250 not idle 87 and 29.
constexpr float kItemPs = 90e3f, kTilePs = 3e3f, kWideTilePs = 8e3f, kWindowed = 4.0f, kFirstPs = 28e6f;
constexpr uint32_t kMasked = 0xffffffffu;

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
    static constexpr int kStages = (DP == 64 ? 2 : 1) * (kFp8 ? 4 : 5);  // units of the ring
    static constexpr int kRaw = !kFp8 ? 0 : DP == 64 ? 4 : 2;  // units of FP8 codes on their way
    static constexpr int kRing = kStages * kUnit + kRaw * (kUnit / 2);
    static constexpr int kRows = 128 * kStreams;         // of a block
    static constexpr int kO = 2 * T;                     // columns of tensor memory: S of even and odd steps, then O
    struct Shared {
        uint64_t full[kStages], empty[kStages];
        uint64_t s_full[2], p_full[2], o_done[2], q_full[2], drained;
        uint64_t rows_known[kPlaces], rows_used[kPlaces];
        uint32_t tmem;
        Waits waits;
        Group of;                   // where this CTA's run begins
        int32_t group, into;
        uint32_t mask[kMasks][4];   // tokens of a tile that are there
        uint32_t row[kPlaces][T];   // where a tile's rows are, from the head's begin, in units of `unit` bytes; kMasked: nowhere
    };
    static constexpr int kBytes = kRing + kStreams * kQ + static_cast<int>(sizeof(Shared));
};

// A group as the caller has it.
__device__ __forceinline__ Group asked_group(const PrefixArgs& a, int32_t g) {
    Group x;
    const int32_t s = a.starts[g], e = a.starts[g + 1];
    x.bad = s < 0 || e < s || e > a.n_requests;
    x.start = s;
    x.members = x.bad ? 0 : e - s;
    x.shared = x.members < 2 ? 0 : min(max(a.shared[g], 0), a.reach);
    return x;
}
// As it is shared, once that is decided.
__device__ __forceinline__ Group group_of(const PrefixArgs& a, int32_t g) {
    Group x;
    const int32_t s = a.starts[g], e = a.starts[g + 1];
    x.bad = false;
    x.start = s;
    x.members = e - s;
    x.shared = x.members < 2 ? 0 : a.kept[s];
    return x;
}
// What sharing saves if its requests would read `again` tokens more than once, in picoseconds of the whole GPU.
template <class K>
__device__ __forceinline__ float worth_of(const PrefixArgs& a, const Group& x, float again) {
    const float heads = static_cast<float>(a.kv_heads), rows = static_cast<float>(x.members) * static_cast<float>(a.group.d);
    const float tiles = ceilf(static_cast<float>(x.shared) * (1.0f / K::T)), items = ceilf(rows * (1.0f / K::kRows));
    const float tile = (rows > 128.0f ? kWideTilePs : kTilePs) * (a.window > 0 ? kWindowed : 1.0f);
    return heads * (again * a.token_ps - items * (kItemPs + tiles * tile));
}
// The shared tokens that the requests of a group see, and the most of them that one sees.
struct Seen {
    int64_t all;
    int32_t most;
};
// EACH requests from `first` on, `apart` from one another, of which those in front of `end` count.
template <int EACH>
__device__ __forceinline__ void look(const PrefixArgs& a, int32_t first, int32_t apart, int32_t end, int32_t shared, Seen& seen) {
    int32_t len[EACH];
#pragma unroll
    for (int u = 0; u < EACH; ++u) len[u] = end - first > u * apart ? min(a.lens[first + u * apart], a.reach) : 0;
#pragma unroll
    for (int u = 0; u < EACH; ++u) {
        const int32_t sees = max(min(len[u], shared) - (a.window > 0 && len[u] > a.window ? len[u] - a.window : 0), 0);
        seen.all += sees;
        seen.most = max(seen.most, sees);
    }
}
// What each lane's group is worth, 0 if it is not shared (whose x.shared is 0 then).  All lanes.
template <class K>
__device__ __forceinline__ float decide(const PrefixArgs& a, Group& x) {
    constexpr int32_t kOfLane = 64;  // requests that a lane looks at itself; a warp together at more
    constexpr int kEach = 8;
    const int lane = threadIdx.x & 31;
    const bool some = x.members > 1 && x.shared > 0;
    float worth = 0.0f;
    // not if it would not pay though every request saw all of it
    const bool may = some && !a.always && worth_of<K>(a, x, static_cast<float>(x.members - 1) * static_cast<float>(x.shared)) > 0.0f;
    Seen seen{0, 0};
    if (may && x.members <= kOfLane)
        for (int32_t i = 0; i < x.members; i += kEach) look<kEach>(a, x.start + i, 1, x.start + x.members, x.shared, seen);
    for (uint32_t large = __ballot_sync(0xffffffffu, may && x.members > kOfLane); large; large &= large - 1) {
        const int src = __ffs(large) - 1;
        const int32_t start = __shfl_sync(0xffffffffu, x.start, src), end = start + __shfl_sync(0xffffffffu, x.members, src);
        const int32_t shared = __shfl_sync(0xffffffffu, x.shared, src);
        Seen part{0, 0};
        for (int32_t i = start; i < end; i += 32 * kEach) look<kEach>(a, min(i + lane, end), 32, end, shared, part);
#pragma unroll
        for (int d = 16; d; d >>= 1) part.all += __shfl_xor_sync(0xffffffffu, part.all, d);
        part.most = __reduce_max_sync(0xffffffffu, part.most);
        if (lane == src) seen = part;
    }
    if (may) worth = fmaxf(worth_of<K>(a, x, static_cast<float>(seen.all - seen.most)), 0.0f);
    if (worth == 0.0f && !a.always) x.shared = 0;
    if (x.members > 1) a.kept[x.start] = x.shared;
    return worth;
}
template <class K>
__device__ __forceinline__ int32_t tiles_of(const Group& x) {
    return static_cast<int32_t>((static_cast<uint32_t>(x.shared) + K::T - 1) / K::T);
}
template <class K>
__device__ __forceinline__ int64_t items_of(const PrefixArgs& a, const Group& x) {
    return (static_cast<int64_t>(x.members) * a.group.d + K::kRows - 1) / K::kRows * a.kv_heads;
}

// What an item costs a CTA besides its tiles, in tiles: its queries into shared memory, an empty pipeline, and its part out of
// tensor memory.  An item is `tiles` + kItemCost places long where the row of all items is cut for the CTAs.
constexpr int kItemCost = 4;

template <class K>
__device__ __forceinline__ int32_t places_of(const Group& x) {
    const int32_t tiles = tiles_of<K>(x);
    return tiles > 0 ? tiles + kItemCost : 0;
}

// A run of tiles of one item.  Every role walks the same runs.
template <class K>
struct Run {
    Group of;
    int32_t g, tiles, items, item, at, left;  // at: the run's place in its item; left: places from there on
    // of the item at hand
    int32_t t, n, kv, block, rows;  // first tile of the run and how many; its key-value head, block of rows, rows
    __device__ __forceinline__ Run(const PrefixArgs& a, const Group& first, int32_t group, int32_t into, int32_t run)
        : of(first), g(group), left(run) {
        tiles = tiles_of<K>(of);
        items = static_cast<int32_t>(items_of<K>(a, of));
        item = into / (tiles + kItemCost);
        at = into - item * (tiles + kItemCost);
        n = 0;
        if (!set(a)) next(a);
    }
    // false: nothing but places that cost
    __device__ __forceinline__ bool set(const PrefixArgs& a) {
        const int32_t places = min(tiles + kItemCost - at, left);
        t = max(at - kItemCost, 0);
        n = max(at + places - kItemCost, 0) - t;
        const int32_t blocks = items / a.kv_heads;
        kv = item / blocks;
        block = item - kv * blocks;
        const int64_t after = static_cast<int64_t>(of.members) * a.group.d - static_cast<int64_t>(block) * K::kRows;
        rows = after < K::kRows ? static_cast<int32_t>(after) : K::kRows;
        at += places;
        left -= places;
        return n > 0;
    }
    // whether each softmax group has rows of its own; else they share the rows and take turns at the tiles
    __device__ __forceinline__ bool dual() const { return K::kStreams == 2 && rows > 128; }
    // among how many warps a row's tokens of a tile are shared out, where there are no rows for four
    __device__ __forceinline__ int32_t sharers() const { return rows <= 32 && K::T == 128 ? 4 : rows <= 64 ? 2 : 1; }
    // Units of the item's tiles (a tile's keys, or its values) in the order in which products want them.  Dual: keys and values of a
    // tile by turns.  Else scores run two steps ahead: K0 K1 V0 K2 V1 ... V(n-2) V(n-1).
    __device__ __forceinline__ uint32_t keys_at(int32_t tile) const { return dual() ? 2 * tile : tile == 0 ? 0 : 2 * tile - 1; }
    __device__ __forceinline__ uint32_t values_at(int32_t tile) const { return dual() || tile == n - 1 ? 2 * tile + 1 : 2 * tile + 2; }
    __device__ __forceinline__ int32_t tile_at(int32_t unit, bool& values) const {
        if (dual() || unit == 0 || unit == 2 * n - 1) {
            values = unit & 1;
            return unit >> 1;
        }
        values = !(unit & 1);
        return values ? unit / 2 - 1 : (unit + 1) / 2;
    }
    __device__ __forceinline__ int32_t steps() const { return dual() ? 2 * n : n; }
    // false: the run is over (and n is 0)
    __device__ __forceinline__ bool next(const PrefixArgs& a) {
        n = 0;
        while (left > 0) {
            if (at == tiles + kItemCost) {
                at = 0;
                if (++item == items) {
                    item = 0;
                    do {
                        of = group_of(a, ++g);
                        tiles = tiles_of<K>(of);
                    } while (tiles == 0 && g + 1 < a.n_groups);
                    items = static_cast<int32_t>(items_of<K>(a, of));
                }
            }
            if (set(a)) return true;
        }
        return false;
    }
};

__device__ __forceinline__ uint64_t global_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// Wait for a phase.  Once a wait of the CTA has run out none lasts any more: every role then goes through its remaining steps
// without waiting, so that barriers and arrivals still match, and the status says so.  All of its accesses stay in bounds: a
// place whose rows have not been found has kMasked in it, or the rows of an earlier tile, and everything else goes by indexes.
constexpr uint32_t kWaitNs = 2000000000;
__device__ __forceinline__ void wait(Waits* waits, uint64_t* bar, uint32_t parity) {
    volatile int32_t& abandoned = waits->abandoned;
    if (mbar_try_wait(bar, parity) || abandoned) return;
    const uint64_t until = global_ns() + waits->ns;
    while (!mbar_try_wait(bar, parity)) {
        if (abandoned) return;
        if (global_ns() > until) {
            abandoned = 1;
            return;
        }
    }
}

// Byte of piece `c` (16 bytes) of row `row` of a tile of `rows` rows: panels of 128 bytes, their pieces exchanged.
__device__ __forceinline__ uint32_t place(int rows, int row, int c) {
    return static_cast<uint32_t>((c >> 3) * (rows * 128) + row * 128 + (((c & 7) ^ (row & 7)) << 4));
}

// ------------------------------------------------------------------ roles

// Of a group's shared tokens those that some request sees, and the first of the requests that reach the last of them: its row
// of the table is read.  Others (idle, shorter) may name less.
struct Lead {
    int32_t row, from, to;
};
__device__ __forceinline__ Lead lead_of(const PrefixArgs& a, const Group& of) {
    constexpr int kEach = 4;  // loads that a lane has on their way
    const int lane = threadIdx.x & 31;
    int32_t most = 0, least = 0x7fffffff, who = 0;
    for (int32_t i0 = 0; i0 < of.members; i0 += 32 * kEach) {
        int32_t len[kEach];
#pragma unroll
        for (int u = 0; u < kEach; ++u) len[u] = of.members - i0 > u * 32 + lane ? min(a.lens[of.start + i0 + u * 32 + lane], a.reach) : 0;
#pragma unroll
        for (int u = 0; u < kEach; ++u) {
            if (len[u] > 0) least = min(least, len[u]);
            const int32_t sees = min(len[u], of.shared);
            if (sees > most) {
                most = sees;
                who = i0 + u * 32 + lane;
            }
        }
        if (a.window == 0 && __any_sync(0xffffffffu, most == of.shared)) break;
    }
    const int32_t to = __reduce_max_sync(0xffffffffu, most);
    who = __reduce_min_sync(0xffffffffu, most == to ? who : 0x7fffffff);
    least = __reduce_min_sync(0xffffffffu, least);
    return Lead{of.start + who, a.window > 0 && to > 0 && least > a.window ? least - a.window : 0, to};
}

// One warp finds the rows of the tiles to come in the page table.
template <class K>
__device__ __forceinline__ void find_rows(const PrefixArgs& a, typename K::Shared& sh, Run<K> run) {
    const int lane = threadIdx.x & 31;
    uint32_t tile = 0;
    bool more = run.n > 0;
    Lead lead{0, 0, 0};
    int32_t group = -1;
    while (more) {
        if (run.g != group) {
            group = run.g;
            lead = lead_of(a, run.of);
        }
        const int64_t at_row = static_cast<int64_t>(lead.row) * a.table_stride;
        for (int32_t i = 0; i < run.n; ++i, ++tile) {
            uint32_t off[K::T / 32];
            int32_t number[K::T / 32];
#pragma unroll
            for (int w = 0; w < K::T / 32; ++w) {
                const uint32_t tok = static_cast<uint32_t>(run.t + i) * K::T + w * 32 + lane, idx = tok / a.by_page;
                const bool in = tok >= static_cast<uint32_t>(lead.from) && tok < static_cast<uint32_t>(lead.to);
                off[w] = in ? (tok - idx * a.page) * a.row_units : kMasked;
                number[w] = in ? a.table[at_row + idx] : 0;
            }
            const uint32_t at = tile % kPlaces;
            wait(&sh.waits, &sh.rows_used[at], (tile / kPlaces & 1u) ^ 1u);
            __syncwarp();
#pragma unroll
            for (int w = 0; w < K::T / 32; ++w) {
                const bool in = off[w] != kMasked, ok = in && static_cast<uint32_t>(number[w]) < a.n_pages;
                if (in && !ok) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                sh.row[at][w * 32 + lane] = ok ? static_cast<uint32_t>(number[w]) * a.page_units + off[w] : kMasked;
                const uint32_t word = __ballot_sync(0xffffffffu, ok);
                if (lane == 0) sh.mask[tile % kMasks][w] = word;
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.rows_known[at]);
        }
        more = run.next(a);
    }
}

template <class K, int MODE>
__device__ __forceinline__ void produce(const PrefixArgs& a, typename K::Shared& sh, uint32_t ring, Run<K> run) {
    const int tid = threadIdx.x - kFirstProducer, lane = tid & 31;
    constexpr int kBytesOf = K::kFp8 ? 1 : 2;
    const int pieces = (a.head_dim * kBytesOf + 15) / 16;  // 16-byte pieces of a row in memory
    constexpr int kMostPieces = K::kPanels * 8 / (K::kFp8 ? 2 : 1);
    const int piece = tid % kMostPieces, row0 = tid / kMostPieces;
    // FP8: a warp copies whole rows (as few lines as it can), and converts them with four pieces of two rows for every eight lanes,
    // so that what they write falls on different banks; odd rows' halves are exchanged on the way, so that what they read does, too.
    constexpr bool kSwaps = kMostPieces >= 8;
    const int piece_of = kSwaps ? (lane & 3) | (lane >> 3 & (kMostPieces / 4 - 1)) << 2 : lane % kMostPieces;
    const int row_in = kSwaps ? (lane >> 2 & 1) | lane / (2 * kMostPieces) << 1 : lane / kMostPieces;
    const int row_of = tid / 32 * (32 / kMostPieces) + row_in;
    const int slot_to = (kSwaps ? tid ^ (row0 & 1) << 2 : tid) * 16;
    const int slot_from = (tid / 32 * 32 + (kSwaps ? (row_in * kMostPieces + piece_of) ^ (row_in & 1) << 2 : lane)) * 16;
    constexpr int kStep = kProducers / kMostPieces, kCopies = K::T / kStep, kAtOnce = kCopies < 8 ? kCopies : 8;
    const bool mine = piece < pieces;
    const int64_t kv_gap = a.v - a.k;
    uint32_t unit = 0, told = 0, tile = 0;  // units begun, units that the consumer has, tiles so far
    // Unit `told` is there: tell the consumer.  FP8: convert it first; every warp converts the pieces that it copied itself.
    auto tell = [&]() {
        if constexpr (K::kFp8) {
            const uint32_t stage = told % K::kStages, to = ring + stage * K::kUnit;
            const uint32_t from = ring + K::kStages * K::kUnit + told % K::kRaw * (K::kUnit / 2) + slot_from;
            wait(&sh.waits, &sh.empty[stage], (told / K::kStages & 1u) ^ 1u);
            __syncwarp();
            if (piece_of < pieces) {
                uint4 code[kCopies];
#pragma unroll
                for (int x = 0; x < kCopies; ++x)
                    asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];"
                                 : "=r"(code[x].x), "=r"(code[x].y), "=r"(code[x].z), "=r"(code[x].w) : "r"(from + x * (kProducers * 16)) : "memory");
#pragma unroll
                for (int x = 0; x < kCopies; ++x) {
                    const int r = row_of + x * kStep;
                    uint4 lo, hi;
                    fp8x4_to_f16<MODE>(code[x].x, lo.x, lo.y);
                    fp8x4_to_f16<MODE>(code[x].y, lo.z, lo.w);
                    fp8x4_to_f16<MODE>(code[x].z, hi.x, hi.y);
                    fp8x4_to_f16<MODE>(code[x].w, hi.z, hi.w);
                    const uint32_t at0 = to + place(K::T, r, 2 * piece_of), at1 = to + place(K::T, r, 2 * piece_of + 1);
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at0), "r"(lo.x), "r"(lo.y), "r"(lo.z), "r"(lo.w) : "memory");
                    asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at1), "r"(hi.x), "r"(hi.y), "r"(hi.z), "r"(hi.w) : "memory");
                }
            }
        }
        fence_proxy();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.full[told % K::kStages]);
        ++told;
    };
    constexpr uint32_t kAhead = K::kFp8 ? K::kRaw - 1 : K::kStages - 2;  // units on their way
    bool more = run.n > 0;
    while (more) {
        const char* keys = a.k + run.kv * a.head_bytes + piece * 16;
        for (int32_t j = 0; j < 2 * run.n; ++j) {
            bool of_v;
            const uint32_t at = tile + run.tile_at(j, of_v);
            if (!of_v) {
                wait(&sh.waits, &sh.rows_known[at % kPlaces], at / kPlaces & 1u);
                __syncwarp();
            }
            const uint32_t* rows = sh.row[at % kPlaces];
            const uint32_t stage = unit % K::kStages, parity = (unit / K::kStages & 1u) ^ 1u;
            const uint32_t to = K::kFp8 ? ring + K::kStages * K::kUnit + unit % K::kRaw * (K::kUnit / 2) + slot_to : ring + stage * K::kUnit;
            const char* base = keys + (of_v ? kv_gap : 0);
            if (!K::kFp8 && !__all_sync(0xffffffffu, mbar_try_wait(&sh.empty[stage], parity))) {
                // no room: what is on the way may be what the consumer waits for
                cp_async_wait<0>();
                while (told < unit) tell();
                wait(&sh.waits, &sh.empty[stage], parity);
                __syncwarp();
            }
            if (mine) {
#pragma unroll
                for (int x0 = 0; x0 < kCopies; x0 += kAtOnce) {
                    uint32_t off[kAtOnce];
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x) off[x] = rows[row0 + (x0 + x) * kStep];
#pragma unroll
                    for (int x = 0; x < kAtOnce; ++x)
                        cp_async16(to + (K::kFp8 ? (x0 + x) * (kProducers * 16) : place(K::T, row0 + (x0 + x) * kStep, piece)),
                                   base + static_cast<uint64_t>(off[x] == kMasked ? 0u : off[x]) * a.unit, off[x] == kMasked ? 0u : 16u);
                }
            }
            cp_async_commit();
            ++unit;
            if (unit - told > kAhead) {
                cp_async_wait<kAhead>();
                tell();
            }
            if (of_v) {
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.rows_used[at % kPlaces]);
            }
        }
        tile += run.n;
        more = run.next(a);
    }
    cp_async_wait<0>();
    while (told < unit) tell();
}

__device__ __forceinline__ bool elect_one() {
    uint32_t is;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
    return is != 0;
}

// One warp waits, and one of its threads issues every product.  Step x of an item: group x & 1 at tile x / 2 (dual) or x.
template <class K>
__device__ __forceinline__ void multiply(const PrefixArgs& a, typename K::Shared& sh, uint32_t ring, uint32_t queries, uint32_t tmem,
                                         Run<K> run) {
    const bool leader = elect_one();
    const uint32_t of_s = product(K::kBf16, K::T, false);
    const int wide = (a.head_dim + 15) / 16;  // products of 16 along head_dim, and columns of O in 16s
    const uint32_t of_o = product(K::kBf16, wide * 16, true);
    uint32_t unit = 0;                               // first unit of the item at hand
    uint32_t s_steps[2] = {0, 0}, o_steps[2] = {0, 0}, q_items[2] = {0, 0};
    bool more = run.n > 0;
    while (more) {
        const bool dual = run.dual();
        const int32_t steps = run.steps();
        auto tile_of = [&](int32_t x) { return dual ? x >> 1 : x; };
        auto scores = [&](int32_t x) {
            const int b = x & 1, s = K::kStreams == 2 ? b : 0;
            if (x < K::kStreams) {  // the group's queries of this item
                wait(&sh.waits, &sh.q_full[s], (b ? q_items[1] : q_items[0]) & 1u);
                if (b) ++q_items[1];
                else ++q_items[0];
            }
            // its weights of the step before, in S's place, have been used
            const uint32_t done = b ? o_steps[1] : o_steps[0];
            if (done > 0) wait(&sh.waits, &sh.o_done[b], (done - 1) & 1u);
            const uint32_t u = unit + run.keys_at(tile_of(x)), stage = u % K::kStages;
            wait(&sh.waits, &sh.full[stage], u / K::kStages & 1u);
            __syncwarp();
            tc_fence_after();
            if (leader) {
                const uint64_t q = operand(queries + s * K::kQ, 16, 1024), keys = operand(ring + stage * K::kUnit, 16, 1024);
                const uint32_t to = tmem + b * K::T;
#pragma unroll
                for (int c = 0; c < K::kDim / 16; ++c)
                    if (c < wide) mma_ss(to, q + (c >> 2) * (128 * 8) + (c & 3) * 2, keys + (c >> 2) * (K::T * 8) + (c & 3) * 2, of_s, c > 0);
                tc_commit(&sh.s_full[b]);
                if (!dual || b == 1) tc_commit(&sh.empty[stage]);
            }
            __syncwarp();
            if (b) ++s_steps[1];
            else ++s_steps[0];
        };
        for (int32_t x = 0; x < 2 && x < steps; ++x) scores(x);
#pragma unroll 1
        for (int32_t x = 0; x < steps; ++x) {
            const int b = x & 1, s = K::kStreams == 2 ? b : 0;
            const uint32_t u = unit + run.values_at(tile_of(x)), stage = u % K::kStages;
            wait(&sh.waits, &sh.full[stage], u / K::kStages & 1u);
            wait(&sh.waits, &sh.p_full[b], ((b ? s_steps[1] : s_steps[0]) - 1) & 1u);
            __syncwarp();
            tc_fence_after();
            if (leader) {
                const uint64_t values = operand(ring + stage * K::kUnit, K::T * 128, 1024);
                const uint32_t o = tmem + K::kO + s * K::kDim, p = tmem + b * K::T;
                const bool first = x < K::kStreams;  // of the group's steps in this item
                // 32 tokens' weights: 16 columns of high terms, 16 of low ones
#pragma unroll
                for (int c = 0; c < K::T / 16; ++c) {
                    mma_ts(o, p + (c >> 1) * 32 + (c & 1) * 8, values + c * 128, of_o, !first || c > 0);
                    mma_ts(o, p + (c >> 1) * 32 + (c & 1) * 8 + 16, values + c * 128, of_o, true);
                }
                tc_commit(&sh.o_done[b]);
                if (!dual || b == 1) tc_commit(&sh.empty[stage]);
            }
            __syncwarp();
            if (b) ++o_steps[1];
            else ++o_steps[0];
            if (x + 2 < steps) scores(x + 2);
        }
        unit += 2 * run.n;
        more = run.next(a);
    }
    // the products read shared and tensor memory until here: waited for whatever has run out
    if (leader) tc_commit(&sh.drained);
    const uint64_t until = global_ns() + kWaitNs;
    bool drained = mbar_try_wait(&sh.drained, 0);
    while (!drained && global_ns() < until) drained = mbar_try_wait(&sh.drained, 0);
    if (!drained) *reinterpret_cast<volatile int32_t*>(&sh.waits.abandoned) = 1;
}

// A row of a softmax group: what its scores are made of, the tokens that it sees, and its running maximum and sum.
struct Row {
    float scale, slope, cap;
    int32_t len;
    uint32_t begin, end;
    float m, less, high, l;  // less: m, or 0 while it is -inf; high: what raises m
    bool seen;               // whether the row sees any of the shared tokens
};

// f of 32 numbers, two at a time.
template <class F>
__device__ __forceinline__ void each_two(uint32_t (&v)[32], F&& f) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
        const float2 p = f(make_float2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
        v[i] = __float_as_uint(p.x);
        v[i + 1] = __float_as_uint(p.y);
    }
}

// 32 products as scores that count: capped, biased, masked.  `tok`: the first token; `word`: those that are there.
__device__ __forceinline__ void count_scores(const PrefixArgs& a, const Row& row, uint32_t (&v)[32], uint32_t tok, uint32_t word) {
    each_two(v, [&](float2 p) { return __fmul2_rn(p, make_float2(row.scale, row.scale)); });
    if (a.softcap > 0.0f) {
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < 32; ++i) most = fmaxf(most, fabsf(__uint_as_float(v[i])));
        if (__any_sync(0xffffffffu, most >= kSmallCapped)) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float p = __uint_as_float(v[i]);
                v[i] = __float_as_uint(fabsf(p) < kSmallCapped ? cap_small(p, a.softcap) : cap_large(p, row.cap));
            }
        } else {
            each_two(v, [&](float2 p) { return cap_small2(p, a.softcap); });
        }
    }
    if (a.slopes) {
        // distance to the newest token, <= 0
        const float away = static_cast<float>(static_cast<int32_t>(tok) - (row.len - 1));
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(__fmaf_rn(row.slope, away + static_cast<float>(i), __uint_as_float(v[i])));
    }
    if (tok < row.begin) word = row.begin - tok >= 32 ? 0u : word & (0xffffffffu << (row.begin - tok));
    if (row.end < tok + 32) word = row.end <= tok ? 0u : word & (0xffffffffu >> (32 - (row.end - tok)));
    if (__any_sync(0xffffffffu, word != 0xffffffffu)) {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = word >> i & 1u ? v[i] : 0xff800000u;
    }
}

__device__ __forceinline__ float largest(const uint32_t (&v)[32]) {
    float t[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int i = 0; i < 32; i += 8)
#pragma unroll
        for (int x = 0; x < 4; ++x) t[x] = fmaxf(t[x], fmaxf(__uint_as_float(v[i + 2 * x]), __uint_as_float(v[i + 2 * x + 1])));
    return fmaxf(fmaxf(t[0], t[1]), fmaxf(t[2], t[3]));
}

// A new maximum; `before`: whether O holds what earlier steps summed, which is then complete.
template <class K, class Before>
__device__ __forceinline__ void raise(const PrefixArgs& a, Row& row, float top, uint32_t o_at, Before&& before) {
    if (!__any_sync(0xffffffffu, row.seen && top > row.high)) return;
    const float m = row.m;
    if (top > row.high) {
        row.m = fmaxf(top - K::kBelow, m);
        row.high = __fadd_rd(row.m, K::kAbove);  // down: 2^16 would be past f16
        row.less = row.m == -INFINITY ? 0.0f : row.m;
    }
    const float f = rescale(m, row.m);
    row.l *= f;
    if (!before()) return;
#pragma unroll 1
    for (int c = 0; c < a.head_dim; c += 16) {
        uint32_t o[16];
        tm_load16(o, o_at + c);
        tc_wait_ld();
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
        tm_store16(o_at + c, o);
    }
}

// The weights of 32 scores, to where those were: their high terms in 16 columns and their low terms in the 16 behind; their sum.
template <class K>
__device__ __forceinline__ float2 weights(const uint32_t (&v)[32], float by, float less, uint32_t at) {
    const float2 by2 = make_float2(by, by), less2 = make_float2(-less, -less);
    float2 sum = make_float2(0.0f, 0.0f);
    uint32_t high[16], low[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        float2 p = __ffma2_rn(make_float2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1])), by2, less2);
        p = make_float2(exp2_fast(p.x), exp2_fast(p.y));
        sum = __fadd2_rn(sum, p);
        high[i] = pack2<K::kBf16>(p.x, p.y);
        float2 h;
        unpack2<K::kBf16>(high[i], h.x, h.y);
        const float2 rest = __fadd2_rn(p, make_float2(-h.x, -h.y));
        low[i] = pack2<K::kBf16>(rest.x, rest.y);
    }
    tm_store16(at, high);
    tm_store16(at + 16, low);
    return sum;
}

// The weights of a tile of tokens from `first` on, whose products are at `at`, in their place.
template <class K, class Before>
__device__ __forceinline__ void weigh(const PrefixArgs& a, Row& row, uint32_t at, uint32_t first, const uint32_t* words, uint32_t o_at,
                                      Before&& before) {
    constexpr int kChunks = K::T / 32;
    bool plain = first >= row.begin && first + K::T <= row.end;
#pragma unroll
    for (int c = 0; c < kChunks; ++c) plain &= words[c] == 0xffffffffu;
    plain = __all_sync(0xffffffffu, (plain || !row.seen) && row.scale >= 0.0f) && a.softcap == 0.0f && a.slopes == nullptr;
    uint32_t v[kChunks][32];
    if (!plain) {
#pragma unroll 1
        for (int c = 0; c < kChunks; ++c) {
            tm_load(v[0], at + c * 32);
            tc_wait_ld();
            count_scores(a, row, v[0], first + c * 32, words[c]);
            tm_store(at + c * 32, v[0]);
        }
        tc_wait_st();
    }
#pragma unroll
    for (int c = 0; c < kChunks; ++c) tm_load(v[c], at + c * 32);
    tc_wait_ld();
    const float by = plain ? row.scale : 1.0f;
    float top = largest(v[0]);
#pragma unroll
    for (int c = 1; c < kChunks; ++c) top = fmaxf(top, largest(v[c]));
    raise<K>(a, row, top * by, o_at, before);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
    for (int c = 0; c < kChunks; ++c) sum = __fadd2_rn(sum, weights<K>(v[c], by, row.less, at + c * 32));
    row.l += sum.x + sum.y;
}

// The same for `mine` of the tile's chunks of 32 tokens, from c0 on; the others, other warps' with the same rows, weigh nothing here.
template <class K, class Before>
__device__ __forceinline__ void weigh_share(const PrefixArgs& a, Row& row, uint32_t at, uint32_t first, const uint32_t* words, int c0, int mine,
                                            uint32_t o_at, Before&& before) {
    uint32_t v[32];
    float top = -INFINITY;
#pragma unroll 1
    for (int c = c0; c < c0 + mine; ++c) {
        tm_load(v, at + c * 32);
        tc_wait_ld();
        count_scores(a, row, v, first + c * 32, words[c]);
        top = fmaxf(top, largest(v));
        if (mine > 1) tm_store(at + c * 32, v);
    }
    if (mine > 1) tc_wait_st();
    raise<K>(a, row, top, o_at, before);
    float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll 1
    for (int c = c0; c < c0 + mine; ++c) {
        if (mine > 1) {
            tm_load(v, at + c * 32);
            tc_wait_ld();
        }
        sum = __fadd2_rn(sum, weights<K>(v, 1.0f, row.less, at + c * 32));
    }
    row.l += sum.x + sum.y;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = 0u;
#pragma unroll 1
    for (int c = 0; c < K::T / 32; ++c)
        if (c < c0 || c >= c0 + mine) tm_store(at + c * 32, v);
}

template <class K>
__device__ __forceinline__ void soften(const PrefixArgs& a, typename K::Shared& sh, unsigned char* queries, uint32_t tmem, Run<K> run) {
    const int lane = threadIdx.x & 31, warp = (threadIdx.x >> 5) & 3, stream = K::kStreams == 2 ? threadIdx.x >> 7 : 0;
    const int my_lane = threadIdx.x & 127;  // of tensor memory
    const uint32_t lanes = tmem + (static_cast<uint32_t>(warp * 32) << 16);
    unsigned char* my_q = queries + stream * K::kQ;
    const uint32_t o_at = lanes + K::kO + stream * K::kDim;
    uint32_t s_steps[2] = {0, 0}, o_steps[2] = {0, 0};
    uint32_t tile0 = 0;
    Row row;
    row.cap = a.softcap * kLog2e;
    bool more = run.n > 0;
    while (more) {
        const bool dual = run.dual();
        const int32_t steps = run.steps(), sharers = dual ? 1 : run.sharers(), apart = 4 / sharers;  // warps of different rows
        const int32_t rows = dual ? min(128, run.rows - 128 * stream) : run.rows;
        const int set = warp & (apart - 1), my_row = set * 32 + lane, my_share = warp / apart;
        const bool busy = set * 32 < rows;  // this warp has rows
        const bool valid = my_row < rows;
        // this row: request and query head
        const uint32_t nth = static_cast<uint32_t>(run.block * K::kRows + (dual ? 128 * stream : 0) + (valid ? my_row : 0));
        const int32_t member = nth / a.group, r = run.of.start + member, h = run.kv * a.group.d + (nth - member * a.group.d);
        row.scale = a.scale * (a.k_scale ? a.k_scale[run.kv] : 1.0f);
        row.m = row.high = -INFINITY;
        row.less = row.l = 0.0f;
        row.len = valid ? min(a.lens[r], a.reach) : 0;
        if (stream < steps) {
            // the queries into shared memory: a few rows at a time, the lanes of a row side by side
            constexpr int kLanes = K::kPanels * 8, kAtOnce = 32 / kLanes;  // 16-byte pieces of a row; rows of an instruction
            const int64_t q_of = r * a.q_req + h * a.q_head;  // of a row that is not: the first row's
            const int c = lane % kLanes;
            const bool has = c < a.head_dim / 8;
            constexpr int kBatch = 8;
#pragma unroll 1
            for (int i0 = 0; i0 < 32 / kAtOnce; i0 += kBatch) {
                uint32_t batch[kBatch][4];
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const char* q = a.q + 2 * (__shfl_sync(0xffffffffu, q_of, (i0 + i) * kAtOnce + lane / kLanes) + (has ? c * 8 : 0));
                    if (a.q_wide) {
                        const uint4 v = *reinterpret_cast<const uint4*>(q);
                        batch[i][0] = v.x, batch[i][1] = v.y, batch[i][2] = v.z, batch[i][3] = v.w;
                    } else {
#pragma unroll
                        for (int x = 0; x < 4; ++x) batch[i][x] = reinterpret_cast<const uint32_t*>(q)[x];
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i) {
                    const bool there = __shfl_sync(0xffffffffu, valid, (i0 + i) * kAtOnce + lane / kLanes) && has;
#pragma unroll
                    for (int x = 0; x < 4; ++x) batch[i][x] = there ? batch[i][x] : 0u;
                }
                if constexpr (K::kFp8) {
                    // f16 queries, scaled by a power of two to a largest magnitude in [1, 2)
                    float top[kBatch];
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        top[i] = 0.0f;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(batch[i][x], f0, f1);
                            else unpack2<true>(batch[i][x], f0, f1);
                            top[i] = fmaxf(top[i], fmaxf(fabsf(f0), fabsf(f1)));
                        }
                    }
#pragma unroll
                    for (int d = 1; d < kLanes; d <<= 1)
#pragma unroll
                        for (int i = 0; i < kBatch; ++i) top[i] = fmaxf(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
#pragma unroll
                    for (int i = 0; i < kBatch; ++i) {
                        const uint32_t field = __float_as_uint(top[i]) >> 23;  // biased exponent
                        const bool scales = field >= 1 && field <= 254;
                        const uint32_t e = min(field, 253u);
                        const float fit = scales ? __uint_as_float((254u - e) << 23) : 1.0f, back = scales ? __uint_as_float(e << 23) : 1.0f;
#pragma unroll
                        for (int x = 0; x < 4; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(batch[i][x], f0, f1);
                            else unpack2<true>(batch[i][x], f0, f1);
                            batch[i][x] = pack2<false>(f0 * fit, f1 * fit);
                        }
                        const float mine = __shfl_sync(0xffffffffu, back, lane % kAtOnce * kLanes);
                        if (lane / kAtOnce == i0 + i) row.scale *= mine;
                    }
                }
#pragma unroll
                for (int i = 0; i < kBatch; ++i)
                    *reinterpret_cast<uint4*>(my_q + place(128, warp * 32 + (i0 + i) * kAtOnce + lane / kLanes, c)) =
                        make_uint4(batch[i][0], batch[i][1], batch[i][2], batch[i][3]);
            }
            fence_proxy();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[stream]);
        }
        row.scale = a.softcap > 0.0f ? __fdiv_rn(row.scale, a.softcap) * (2.0f * kLog2e) : row.scale * kLog2e;
        row.end = max(min(row.len, run.of.shared), 0);
        row.begin = a.window > 0 && row.len > a.window ? row.len - a.window : 0;
        row.slope = a.slopes ? a.slopes[h] * kLog2e : 0.0f;
        row.seen = valid && row.begin < row.end;
#pragma unroll 1
        for (int32_t x = K::kStreams == 2 ? stream : 0; x < steps; x += K::kStreams) {
            const int b = x & 1;
            const int32_t tile = dual ? x >> 1 : x;
            wait(&sh.waits, &sh.s_full[b], (b ? s_steps[1] : s_steps[0]) & 1u);
            __syncwarp();
            if (b) ++s_steps[1];
            else ++s_steps[0];
            tc_fence_after();
            if (busy) {
                const uint32_t s_at = lanes + b * K::T;
                const uint32_t* words = sh.mask[(tile0 + tile) % kMasks];
                const uint32_t first = static_cast<uint32_t>(run.t + tile) * K::T;
                auto before = [&]() {
                    if (x < K::kStreams) return false;
                    const int pb = K::kStreams == 2 ? b : (x - 1) & 1;
                    wait(&sh.waits, &sh.o_done[pb], ((pb ? o_steps[1] : o_steps[0]) - 1) & 1u);
                    __syncwarp();
                    tc_fence_after();
                    return true;
                };
                const int each = K::T / 32 / sharers;
                if (sharers == 1) weigh<K>(a, row, s_at, first, words, o_at, before);
                else weigh_share<K>(a, row, s_at, first, words, my_share * each, each, o_at, before);
                tc_wait_st();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.p_full[b]);
            if (b) ++o_steps[1];
            else ++o_steps[0];
        }
        // This CTA's part of the rows, through the place of the queries, with which the products are done: rows side by side, and the
        // warps that share rows joined.
        const bool has = steps > stream, first = run.t == 0;
        const int64_t row0 = first ? (static_cast<int64_t>(dual ? 0 : stream) * a.n_requests + run.of.start) * a.q_heads +
                                         static_cast<int64_t>(run.kv) * run.of.members * a.group.d + run.block * K::kRows + (dual ? 128 * stream : 0)
                                   : (static_cast<int64_t>(blockIdx.x) * 2 + stream) * 128;
        float2* ml_to = (first ? a.part_ml : a.cta_ml) + row0 + my_row;
        float odd = 0.0f;  // NaN once a number is not finite
        if (!has) {
            if (valid && my_share == 0) *ml_to = make_float2(-INFINITY, 0.0f);
        } else {
            const int b = (steps - 1 - (steps - 1 - stream) % K::kStreams) & 1;
            wait(&sh.waits, &sh.o_done[b], ((b ? o_steps[1] : o_steps[0]) - 1) & 1u);
            __syncwarp();
            tc_fence_after();
            if (!row.seen) {  // what it has is of nothing
                row.m = -INFINITY;
                row.l = 0.0f;
            }
            float top = row.m, sum = row.l, weight = 1.0f;
            if (sharers > 1) {
                float2* ml = reinterpret_cast<float2*>(my_q);
                ml[my_lane] = make_float2(row.m, row.l);
                asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
                sum = 0.0f;
                for (int x = 0; x < sharers; ++x) top = fmaxf(top, ml[x * apart * 32 + my_row].x);
                for (int x = 0; x < sharers; ++x) {
                    const float2 of = ml[x * apart * 32 + my_row];
                    if (of.y != 0.0f) sum += of.y * rescale(of.x, top);
                }
                weight = rescale(row.m, top);
                asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
            }
            if (valid && my_share == 0) *ml_to = make_float2(top, sum);
            // of this warp's set of rows the share of this warp, four rows at a time: a lane's row and elements
            const int own = my_share * (32 / sharers) + (lane >> 3), piece = lane & 7;
            float* to = (first ? a.part : a.cta_part) + (row0 + set * 32 + own) * a.head_dim + piece * 4;
            float4* lines = reinterpret_cast<float4*>(my_q);  // [128][8], pieces exchanged
#pragma unroll 1
            for (int c = 0; c < a.head_dim; c += 32) {
                uint32_t v[32];
                tm_load(v, o_at + c);
                tc_wait_ld();
#pragma unroll
                for (int i = 0; i < 16; ++i) odd = __fmaf_rn(__uint_as_float(v[i]), 0.0f, odd);
                if (c + 16 < a.head_dim) {  // no product wrote what is behind
#pragma unroll
                    for (int i = 16; i < 32; ++i) odd = __fmaf_rn(__uint_as_float(v[i]), 0.0f, odd);
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float4 f = make_float4(__uint_as_float(v[4 * i]) * weight, __uint_as_float(v[4 * i + 1]) * weight,
                                                 __uint_as_float(v[4 * i + 2]) * weight, __uint_as_float(v[4 * i + 3]) * weight);
                    lines[my_lane * 8 + (i ^ (lane & 7))] = row.l == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : f;
                }
                if (sharers > 1) asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
                else __syncwarp();
                const bool in = c + piece * 4 < a.head_dim;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if (i * 4 >= 32 / sharers) break;
                    const int j = own + i * 4;
                    float4 f = lines[(set * 32 + j) * 8 + (piece ^ (j & 7))];
#pragma unroll
                    for (int x = 1; x < 4; ++x)
                        if (x < sharers) {
                            const float4 g = lines[((x * apart + set) * 32 + j) * 8 + (piece ^ (j & 7))];
                            f = make_float4(f.x + g.x, f.y + g.y, f.z + g.z, f.w + g.w);
                        }
                    if (in && set * 32 + j < rows) *reinterpret_cast<float4*>(to + i * 4 * a.head_dim + c) = f;
                }
                if (sharers > 1) asm volatile("bar.sync %0, 128;" ::"r"(2 + stream) : "memory");
                else __syncwarp();
            }
            // A weight of 0 times a value that is not finite is NaN, and the row may not even see that value's token: then its
            // request reads all of its tokens in the launch behind this one, where every row has its own.
            if (busy && row.l != 0.0f && __fmaf_rn(row.l, 0.0f, odd) != 0.0f) a.alone[r] = a.call[1] + 1;
            tc_fence_before();
        }
        tile0 += run.n;
        more = run.next(a);
    }
}

// One warp tells the other launches each request's first token of its own, and where its shared part's pieces will be.
template <class K>
__device__ __forceinline__ void take_notes(const PrefixArgs& a, bool none) {
    const int lane = threadIdx.x & 31;
    const int32_t begin = none || a.n_groups == 0 ? a.n_requests : a.starts[0], end = none || a.n_groups == 0 ? a.n_requests : a.starts[a.n_groups];
    for (int32_t r = blockIdx.x * 32 + lane; r < a.n_requests; r += gridDim.x * 32)
        if (r < begin || r >= end) {
            a.own_first[r] = 0;
            a.info[r] = Shared{0, 0, 0, 0};
        }
    if (none) return;
    int64_t front = 0;
    for (int32_t g0 = 0; g0 < a.n_groups; g0 += 32) {
        const int32_t g = g0 + lane;
        Group x{};
        if (g < a.n_groups) x = group_of(a, g);
        const int64_t of = items_of<K>(a, x) * places_of<K>(x);
        int64_t upto = of;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int64_t y = __shfl_up_sync(0xffffffffu, upto, d);
            if (lane >= d) upto += y;
        }
        const int32_t base = static_cast<int32_t>(front + upto - of);
        front += __shfl_sync(0xffffffffu, upto, 31);
        uint32_t mine = __ballot_sync(0xffffffffu, g < a.n_groups && g % gridDim.x == blockIdx.x);
        while (mine) {
            const int src = __ffs(mine) - 1;
            mine &= mine - 1;
            const Shared note{__shfl_sync(0xffffffffu, base, src), __shfl_sync(0xffffffffu, tiles_of<K>(x), src), __shfl_sync(0xffffffffu, x.start, src),
                              __shfl_sync(0xffffffffu, x.members, src)};
            const int32_t shared = __shfl_sync(0xffffffffu, x.shared, src);
            for (int32_t i = lane; i < note.members; i += 32) {
                a.own_first[note.start + i] = shared;
                a.info[note.start + i] = note;
            }
        }
    }
}

template <int MODE, int DP>
__global__ void __launch_bounds__(kThreads, 1) prefix_kernel(const PrefixArgs a) {
    using K = Prefix<MODE, DP>;
    extern __shared__ __align__(1024) unsigned char smem[];
    unsigned char* queries = smem + K::kRing;
    auto& sh = *reinterpret_cast<typename K::Shared*>(queries + K::kStreams * K::kQ);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
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
        for (int i = 0; i < kPlaces; ++i) {
            mbar_init(&sh.rows_known[i], 1);
            mbar_init(&sh.rows_used[i], kProducers / 32);
        }
        mbar_init(&sh.drained, 1);
        fence_barrier_init();
        sh.waits = Waits{a.wait_ns, a.wait_ns == 0};
    }
    // nothing is known of any tile's rows
    for (int i = tid; i < kPlaces * K::T; i += kThreads) sh.row[i / K::T][i % K::T] = kMasked;
    for (int i = tid; i < kMasks * 4; i += kThreads) sh.mask[i / 4][i % 4] = 0;
    if (warp == kIssuer) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&sh.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    after_previous();
    let_next_start();
    // the tiles of thread i's `per` consecutive groups, in a row
    int64_t* sums = reinterpret_cast<int64_t*>(queries);  // of the warps, before the queries come
    float* worths = reinterpret_cast<float*>(sums + kThreads / 32);
    const int32_t per = (a.n_groups + kThreads - 1) / kThreads;
    int64_t mine = 0;
    bool bad = false;
    Group last{};
    float worth = 0.0f;
    for (int32_t i = 0; i < per; ++i) {
        const int32_t g = tid * per + i;
        last = Group{};
        if (g < a.n_groups) last = asked_group(a, g);
        bad |= last.bad;
        worth += decide<K>(a, last);
        mine += items_of<K>(a, last) * places_of<K>(last);
    }
    int64_t upto = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t x = __shfl_up_sync(0xffffffffu, upto, d);
        if (lane >= d) upto += x;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) worth += __shfl_xor_sync(0xffffffffu, worth, d);
    if (lane == 31) {
        sums[warp] = upto;
        worths[warp] = worth;
    }
    // what is past the head in a row is never copied: zeros
    if (a.head_dim < DP) {
        for (int i = tid; i < K::kRing / 16; i += kThreads) reinterpret_cast<uint4*>(smem)[i] = make_uint4(0, 0, 0, 0);
        fence_proxy();
    }
    tc_fence_before();
    bad = __syncthreads_or(bad);
    tc_fence_after();
    const uint32_t tmem = sh.tmem, ring = smem_u32(smem);
    int64_t total64 = 0, front = 0;
    worth = 0.0f;
#pragma unroll
    for (int w = 0; w < kThreads / 32; ++w) {
        worth += worths[w];
        if (w == warp) front = total64;
        total64 += sums[w];
    }
    front += upto - mine;
    if (bad || total64 > 0x7fffffff) {
        // nothing is shared then: every request reads all of its tokens
        if (tid == 0) atomicExch(a.status, MF_DEVICE_TOO_LARGE);
        bad = true;
    }
    const bool none = bad || (!a.always && worth < kFirstPs);
    if (none) total64 = 0;
    const int32_t total = static_cast<int32_t>(total64), ctas = min(total, static_cast<int32_t>(gridDim.x));
    if (blockIdx.x == 0 && tid == 0) {
        *a.cut = make_int2(total, ctas);
        a.call[0] = a.call[1] + 1;
    }
    if (static_cast<int32_t>(blockIdx.x) < ctas) {
        const Cut cut(total, ctas);
        const int32_t x0 = cut.start(blockIdx.x), run_of = cut.start(blockIdx.x + 1) - x0;
        if (front <= x0 && x0 < front + mine) {
            int32_t into = x0 - static_cast<int32_t>(front), g = tid * per;
            if (per > 1) {
                for (;; ++g) {
                    last = group_of(a, g);
                    const int64_t of = items_of<K>(a, last) * places_of<K>(last);
                    if (into < of) break;
                    into -= static_cast<int32_t>(of);
                }
            }
            sh.of = last;
            sh.group = g;
            sh.into = into;
        }
        __syncthreads();
        const Run<K> run(a, sh.of, sh.group, sh.into, run_of);
        const int role = tid >> 7;
        if (role < K::kStreams) {
            asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
            soften<K>(a, sh, queries, tmem, run);
        } else if (role == kFirstProducer / 128) {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kProducerRegs));
            produce<K, MODE>(a, sh, ring, run);
        } else {
            asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
            if (warp == kIssuer) multiply<K>(a, sh, ring, smem_u32(queries), tmem, run);
            else if (warp == kPager) find_rows<K>(a, sh, run);
            else if (warp == kNoter) take_notes<K>(a, none);
        }
        __syncwarp();
    } else if (warp == kNoter) {
        take_notes<K>(a, none);
    }
    tc_fence_before();
    __syncthreads();
    if (tid == 0 && sh.waits.abandoned && static_cast<int32_t>(blockIdx.x) < ctas) atomicExch(a.status, MF_DEVICE_TIMEOUT);
    if (warp == kIssuer) {
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

// ------------------------------------------------------------------ the join

constexpr int kJoinThreads = 256;

// A warp for each query head of a request.  ROWS: of a block; F16: the weights of a maximum are 2^12.
template <int ROWS, bool F16>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const PrefixArgs a) {
    constexpr float kBelow = F16 ? 12.0f : 0.0f, kMost = F16 ? 4096.0f : 1.0f;
    const int lane = threadIdx.x & 31;
    after_previous();
    let_next_start();
    const int64_t n = static_cast<int64_t>(a.n_requests) * a.q_heads;
    const int2 all = *a.cut;
    const uint32_t call = a.call[0];
    if (blockIdx.x == 0 && threadIdx.x == 0) a.call[1] = call;  // the next call's number is another
    const int32_t dim = a.head_dim;
    for (int64_t w = (static_cast<int64_t>(blockIdx.x) * kJoinThreads + threadIdx.x) >> 5; w < n; w += static_cast<int64_t>(gridDim.x) * (kJoinThreads / 32)) {
        const int32_t r = static_cast<int32_t>(w / a.q_heads), h = static_cast<int32_t>(w - static_cast<int64_t>(r) * a.q_heads);
        const int32_t kv = h / a.group;
        const float vs = a.v_scale ? a.v_scale[kv] : 1.0f;
        const Shared x = a.info[r];
        // its own tokens: a part that is normalised already.  Joined by maximum and sum as the others are: in one logarithm the
        // weight of a part whose scores are large would lose bits (half a step of float32 at 20000 is 2^-10)
        const float2 own = a.own_ml[w];
        float4 acc[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = 4 * (lane + 32 * i);
            acc[i] = d < dim ? *reinterpret_cast<const float4*>(a.own + w * dim + d) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
        // the parts of its shared tokens, in order: an item's first CTA's, then the other CTAs', each of one half or two
        int32_t parts = 0, halves = 1;
        int64_t first_at = 0, first_apart = 0, at = 0;  // rows of part, cta_part
        if (x.tiles > 0 && a.alone[r] != call) {
            const int64_t nth = static_cast<int64_t>(r - x.start) * a.group.d + (h - kv * static_cast<int32_t>(a.group.d)), rows = static_cast<int64_t>(x.members) * a.group.d;
            const int32_t blocks = static_cast<int32_t>((rows + ROWS - 1) / ROWS), block = static_cast<int32_t>(nth / ROWS);
            halves = ROWS == 128 || rows - static_cast<int64_t>(block) * ROWS > 128 ? 1 : 2;
            const Cut cut(all.x, all.y);
            const int32_t begin = x.base + (kv * blocks + block) * (x.tiles + kItemCost) + kItemCost, cta = cut.part_of(begin);
            parts = (cut.part_of(begin + x.tiles - 1) - cta + 1) * halves;
            first_at = static_cast<int64_t>(x.start) * a.q_heads + kv * rows + nth;
            first_apart = n;
            at = static_cast<int64_t>(cta) * 256 + (nth - static_cast<int64_t>(block) * ROWS);
        }
        auto row_of = [&](int32_t p) {  // of part p: negative in part (one less than minus its row), else of cta_part
            const int32_t k = halves == 2 ? p >> 1 : p, half = halves == 2 ? p & 1 : 0;
            return k == 0 ? -(first_at + half * first_apart) - 1 : at + static_cast<int64_t>(k) * 256 + half * 128;
        };
        float top = own.x;
        float2 ml = make_float2(-INFINITY, 0.0f);
        int64_t row = 0;
        for (int32_t p0 = 0; p0 < parts; p0 += 32) {
            if (p0 + lane < parts) {
                row = row_of(p0 + lane);
                ml = row < 0 ? a.part_ml[-row - 1] : a.cta_ml[row];
                if (ml.y != 0.0f) top = fmaxf(top, ml.x);
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
        // alone it stays as it is
        const float own_l = own.y == 0.0f ? 0.0f : own.y * rescale(own.x, top), own_w = parts == 0 && own.y != 0.0f ? 1.0f : own_l;
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 2; ++i)
            acc[i] = own_w == 0.0f ? make_float4(0.0f, 0.0f, 0.0f, 0.0f) : make_float4(acc[i].x * own_w, acc[i].y * own_w, acc[i].z * own_w, acc[i].w * own_w);
        for (int32_t p0 = 0; p0 < parts; p0 += 32) {
            if (parts > 32 && p0 + lane < parts) {
                row = row_of(p0 + lane);
                ml = row < 0 ? a.part_ml[-row - 1] : a.cta_ml[row];
            }
            const bool in = p0 + lane < parts && ml.y != 0.0f;
            const float by = in ? rescale(ml.x, top) : 0.0f;
            sum += in ? ml.y * by : 0.0f;
            const int32_t here = min(32, parts - p0);
#pragma unroll 4
            for (int32_t p = 0; p < here; ++p) {
                const float weight = __shfl_sync(0xffffffffu, by, p) * vs;
                const int64_t of = __shfl_sync(0xffffffffu, row, p);
                const bool some = __shfl_sync(0xffffffffu, in, p);
                const float* from = of < 0 ? a.part + (-of - 1) * dim : a.cta_part + of * dim;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int d = 4 * (lane + 32 * i);
                    if (some && d < dim) {
                        const float4 f = *reinterpret_cast<const float4*>(from + d);
                        acc[i] = make_float4(__fmaf_rn(f.x, weight, acc[i].x), __fmaf_rn(f.y, weight, acc[i].y), __fmaf_rn(f.z, weight, acc[i].z),
                                             __fmaf_rn(f.w, weight, acc[i].w));
                    }
                }
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
        sum += own_l;
        const float inv = parts == 0 || sum == 0.0f ? 1.0f : __fdiv_rn(1.0f, sum);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int d = 4 * (lane + 32 * i);
            if (d >= dim) break;
            const float4 f = make_float4(acc[i].x * inv, acc[i].y * inv, acc[i].z * inv, acc[i].w * inv);
            const uint2 two = a.q_f16 ? make_uint2(pack2<false>(f.x, f.y), pack2<false>(f.z, f.w)) : make_uint2(pack2<true>(f.x, f.y), pack2<true>(f.z, f.w));
            *reinterpret_cast<uint2*>(a.out + 2 * (r * a.out_req + h * a.out_head + d)) = two;
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
    return Kernel{prefix_kernel<MODE, DP>, join_kernel<K::kRows, !K::kBf16>, kThreads, K::kBytes};
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
    // places of rows are kept in 32 bits, in the largest unit that strides allow
    const int code = is_fp8(k.dtype) ? 1 : 2;
    const int64_t page_bytes = k.page_stride * code, row_bytes = k.token_stride * code;
    uint32_t unit = 4;
    while (unit < 30 && ((page_bytes | row_bytes) >> unit & 1) == 0) ++unit;
    const int64_t n_pages = k.n_pages < 0x7fffffff ? k.n_pages : 0x7fffffff;
    if (static_cast<double>(n_pages) * page_bytes + static_cast<double>(k.page_size) * row_bytes >= 4294967295.0 * (1ll << unit)) {
        mf_paged_attn_destroy(own);
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_prefix_attn_create: %lld pages of %lld bytes: more than 2^32 - 1 units of %lld bytes",
                    (long long)n_pages, (long long)page_bytes, 1ll << unit);
    }
    const Kernel kernel = pick(k.dtype, k.head_dim);
    cudaError_t err = cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel.fn), cudaFuncAttributeMaxDynamicSharedMemorySize, kernel.shared);
    const int ctas = state().sm_count;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t heads = static_cast<size_t>(max_requests) * c.q_heads, alones = up(static_cast<size_t>(max_requests) * 4);
    const size_t firsts = up(static_cast<size_t>(max_requests) * 4), kepts = firsts, infos = up(static_cast<size_t>(max_requests) * sizeof(Shared));
    const size_t parts = up(2 * heads * k.head_dim * 4), part_mls = up(2 * heads * 8);
    const size_t cta_parts = up(static_cast<size_t>(ctas) * 256 * k.head_dim * 4), cta_mls = up(static_cast<size_t>(ctas) * 256 * 8);
    const size_t owns = up(heads * k.head_dim * 4), own_mls = up(heads * 8);
    const size_t cleared = 256 + alones, bytes = cleared + firsts + kepts + infos + parts + part_mls + cta_parts + cta_mls + owns + own_mls;
    mf_prefix_attn_s* h = err == cudaSuccess ? new (std::nothrow) mf_prefix_attn_s{} : nullptr;
    if (!h) {
        mf_paged_attn_destroy(own);
        return err != cudaSuccess ? cuda_fail(err, "mf_prefix_attn_create: cudaFuncSetAttribute")
                                  : fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_prefix_attn_create: out of host memory");
    }
    err = cudaMalloc(&h->workspace, bytes);
    if (err == cudaSuccess) err = cudaMemset(h->workspace, 0, cleared);
    if (err == cudaSuccess) err = cudaStreamSynchronize(nullptr);  // streams that do not wait for the default one may run it
    PrefixArgs& a = h->args;
    a.status = err == cudaSuccess ? sticky_status_ptr() : nullptr;
    if (!a.status) {
        cudaGetLastError();
        cudaFree(h->workspace);  // NULL: nothing
        delete h;
        mf_paged_attn_destroy(own);
        if (err == cudaErrorMemoryAllocation)
            return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_prefix_attn_create: %zu bytes: out of device memory", bytes);
        return err != cudaSuccess ? cuda_fail(err, "mf_prefix_attn_create: workspace")
                                  : fail(MF_ERR_CUDA, "mf_prefix_attn_create: sticky status word unavailable");
    }
    char* w = static_cast<char*>(h->workspace);
    h->own = own;
    h->kernel = kernel;
    h->device = state().device;
    h->ctas = ctas;
    h->max_requests = max_requests;
    const int64_t reach = static_cast<int64_t>(c.max_pages) * k.page_size;
    a.reach = reach < 0x7fffffff ? static_cast<int32_t>(reach) : 0x7fffffff;
    a.page = k.page_size;
    a.always = 0;
    a.wait_ns = kWaitNs;
    a.token_ps = (8.0f + 0.32f * k.head_dim) * (is_fp8(k.dtype) ? 0.64f : 1.0f) * ((c.q_heads / k.kv_heads + 15) / 16);
    a.window = c.window;
    a.kv_heads = k.kv_heads;
    a.unit = 1u << unit;
    a.page_units = static_cast<uint32_t>(page_bytes >> unit);
    a.row_units = static_cast<uint32_t>(row_bytes >> unit);
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
    a.call = reinterpret_cast<uint32_t*>(w + 64);
    a.alone = reinterpret_cast<uint32_t*>(w += 256);
    a.own_first = reinterpret_cast<int32_t*>(w += alones);
    a.kept = reinterpret_cast<int32_t*>(w += firsts);
    a.info = reinterpret_cast<Shared*>(w += kepts);
    a.part = reinterpret_cast<float*>(w += infos);
    a.part_ml = reinterpret_cast<float2*>(w += parts);
    a.cta_part = reinterpret_cast<float*>(w += part_mls);
    a.cta_ml = reinterpret_cast<float2*>(w += cta_parts);
    a.own = reinterpret_cast<float*>(w += cta_mls);
    a.own_ml = reinterpret_cast<float2*>(w += owns);
    *handle = h;
    return MF_OK;
}

extern "C" int mf_prefix_attn_share(mf_prefix_attn handle, int32_t always) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_share: handle is NULL");
    if (always != 0 && always != 1) return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_share: %d (0 or 1)", always);
    handle->args.always = always;
    return MF_OK;
}

extern "C" int mf_prefix_attn_limit(mf_prefix_attn handle, int64_t wait_ns) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_limit: handle is NULL");
    if (wait_ns < 0 || wait_ns > 0xffffffffll)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_prefix_attn_limit: %lld ns (0 to 2^32 - 1)", (long long)wait_ns);
    handle->args.wait_ns = static_cast<uint32_t>(wait_ns);
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
    const int rc = paged_attn_run_parts(handle->own, q, k_cache, v_cache, table, lens, n_requests, a.own_first, a.alone, a.call, a.own,
                                        a.own_ml, s);
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
