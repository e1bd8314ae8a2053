// paged_attn.cu -- attention of one new token per request over a paged
// key-value cache (mf_paged_attn_*).
//
// For request r and query head h over its tokens n:
//   s_n = scale * q.k_n  (capped, biased),  out = sum exp(s_n) v_n / sum exp(s_n).
// One pass over the cache with a running maximum m and sum l: a new maximum
// multiplies what is summed so far by exp(m_old - m_new).  Parts of a request
// summed apart join the same way, from their (m, l, unnormalised out).
//
// Bound: HBM.  Each key and value byte is used for the query heads of its
// key-value head only (4 operations per element and query head: 8 heads on
// BF16 are 32 operations for 2 bytes), far below what tensor cores need to
// be the limit, so the design is about keeping loads in flight:
//   * The work is cut into tiles of 16 or 32 tokens (8 KB of keys and values
//     where a row has up to 256 bytes) of one item: a request, a key-value head
//     and a block of its query heads.  The tiles of all items in a row are cut
//     evenly for the teams of the grid, whatever the lengths; a small batch's
//     items get CTAs of their own.
//   * A team is a warp, or two that share a ring where more than 8 query heads
//     share a key-value head.  It works alone: a ring of stages in shared
//     memory filled by 16-byte cp.async (rows of masked tokens are zero-filled,
//     not read), no CTA barrier inside the loop, page numbers read one tile
//     ahead.  Twelve warps per SM; copying warps that feed the others were
//     slower (108 us with four of them for the 92 below: a copy instruction of
//     512 bytes needs more issue slots than a few warps have), and so were
//     bulk copies a row at a time (67 clocks each per issuing warp).
//   * Products run on mma.m16n8k16 with tokens (then head_dim) on the long side
//     and query heads on the side of 8: S^T = K Q^T and O^T = V^T P^T.  The
//     weights move from the first product's result layout to the second's
//     operand layout by movmatrix, in registers.  The wide tensor-core form
//     (tcgen05) needs 64 or more rows of queries to be fed: there are 1 to 16;
//     the tensor pipe is 14% (BF16) to 23% (FP8) busy.
//   * exp(s - m) is rounded to two 16-bit terms (high and low).  Two BF16 terms
//     carry 16 bits of any weight, two f16 terms 22 bits of the large ones and,
//     since f16 ends at 2^-24, no more than 2^-25 absolutely: the f16 forms put
//     m below the maximum (see kBelow), so that this is 2^-37 of the largest
//     weight.  (One f16 term for FP8 caches missed the bound that two give.)
//   * FP8 codes become f16 in registers (exact); the queries are then f16 too,
//     scaled by a power of two per head so that none overflows.
// Where a run of tiles ends inside an item, the teams of a CTA join their
// parts in shared memory, CTAs through the workspace: the last of an item's
// CTAs to arrive (a ticket) joins them in the order of the tokens, so the
// result does not depend on who was last.
//
// Measured (B200, keys and values in the loop come at 7.4 TB/s, the copy rate
// of the roofline is 6.55): 64 requests of 2048 tokens, 32/8 heads of 128: BF16
// 92 us (82 at the copy rate), E4M3 54 us (41); 2 of 131071: 160 us (164); the
// same 64 with 16/8 heads of 256: 168 us (164).  What a call costs besides:
// about 3 us until the first tile is there and 4 to 6 us for the joins, mostly
// instruction fetches of code that runs once; more where parts are large and
// few CTAs join them (one request of 30011 tokens, 16/1 heads of 256: 27 us, 5
// at the copy rate).
#include <new>

#include "mf_attn.cuh"
#include "mf_divisor.cuh"
#include "mf_internal.h"
#include "mf_launch.cuh"
#include "mf_runtime.h"
#include "mf_vec.cuh"

namespace mf {
namespace {

constexpr int kBlock = 16;         // tokens of one product; a tile is one or two blocks

// Ordered by first use: the start of a run waits for a line of parameters only once or twice.
struct AttnArgs {
    const int32_t* lens;
    const int32_t* table;
    int32_t n_requests, items;  // items: kv_heads * blocks
    int32_t max_pages, page, window, blocks;  // blocks of query heads per key-value head
    const char* k;
    const char* v;
    int32_t page_bytes, row_bytes;
    int64_t head_bytes, table_stride;
    uint32_t n_pages;
    Divisor by_page;
    Divisor used_heads;   // query heads of an item that has all of its own
    int32_t head_dim;
    const char* q;
    int64_t q_req, q_head;
    int32_t q_heads, group, q_f16;
    float scale, softcap;
    const float* slopes;
    const float* k_scale;
    const float* v_scale;
    char* out;
    int64_t out_req, out_head;
    float* lse;
    float* team_part;     // [teams][heads * (DP + 2)]: parts that end inside a team's run
    float* cta_part;      // [CTAs][3][heads * (DP + 2)]: parts that leave the CTA, and joined groups of them
    int32_t* tickets;     // [2][CTAs], zero between runs
    int32_t* status;
    const int32_t* own_first;  // of a run of parts: each request's first token; 0 where `alone` has the number of the call
    const uint32_t* alone;
    const uint32_t* call;
};

// ------------------------------------------------------------------ pieces

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
// c = a b (FIRST) or c += a b, 16 x 16 by 16 x 8.
template <bool BF16, bool FIRST = false>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (FIRST && BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else if constexpr (FIRST)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else if constexpr (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Barrier of a team's warps.
template <int TM>
__device__ __forceinline__ void team_sync(int team) {
    if constexpr (TM == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(1 + team), "n"(32 * TM) : "memory");
}
// The same for codes 0, 2 and codes 1, 3.
template <int DT>
__device__ __forceinline__ void fp8x4_to_f16_strided(uint32_t four, uint32_t& even, uint32_t& odd) {
    if constexpr (DT == MF_DT_F8E4M3) {
        fp8x4_to_f16<DT>(__byte_perm(four, 0u, 0x3120u), even, odd);
    } else {
        even = __byte_perm(four, 0u, 0x2404u);
        odd = __byte_perm(four, 0u, 0x3414u);
    }
}
// A request's tokens: [first, len) are seen, in tiles from `base` on (a multiple
// of the block, so that a block never crosses a page of whole blocks).
struct Span {
    int32_t len, first, base;
};
template <bool PART>
__device__ __forceinline__ Span span_of(const AttnArgs& a, int32_t r) {
    const int64_t reach = static_cast<int64_t>(a.max_pages) * a.page;
    Span s;
    s.len = max(a.lens[r], 0);
    if (s.len > reach) s.len = static_cast<int32_t>(reach);
    s.first = a.window > 0 && s.len > a.window ? s.len - a.window : 0;
    if constexpr (PART) s.first = min(max(s.first, a.alone[r] == *a.call ? 0 : a.own_first[r]), s.len);
    s.base = PART && s.first == s.len ? s.len : s.first & ~(kBlock - 1);
    return s;
}
template <int T>
__device__ __forceinline__ int32_t tiles_of(const Span& s) {
    return static_cast<int32_t>((static_cast<uint32_t>(s.len - s.base) + (T - 1)) / T);
}

// A place in the row of all tiles: request, item of the request, tile of the item.
template <int T, bool PART>
struct Place {
    int32_t r, item, t, nt;   // nt: tiles of the request's items
    Span span;
    __device__ __forceinline__ void next(const AttnArgs& a, int32_t items) {
        if (++t < nt) return;
        t = 0;
        if (++item < items) return;
        item = 0;
        nt = 0;
        while (++r < a.n_requests) {
            span = span_of<PART>(a, r);
            nt = tiles_of<T>(span);
            if (nt > 0) return;
        }
    }
};

// What is known of one part of an item that a warp or CTA summed.
struct Part {
    int32_t start;   // first tile of the item in the row of all tiles; -1: no part
    int32_t r, item, nt;
    int32_t ta, tb;  // its tiles of the item
};

// An item of which this CTA has parts: the parts, where it belongs, and whether it is whole (slot -1) or other CTAs have
// parts of it, too.  Slot 0 is the end or middle of an item that began in an earlier CTA, slot 1 the start of one that ends
// in a later CTA.
struct Joined {
    uint32_t parts;
    int32_t r, kv, head0, heads, slot, start, nt;
};

constexpr int kFills = 3;  // ways to give each item CTAs of its own
constexpr int kJoin = 16;  // most parts that one step of a join between CTAs takes
// MODE: dtype of the cache; DP: head_dim padded to 64, 128 or 256; TM: warps of a team; W: warps; T: tokens of a
// tile; S: stages of a team's ring.  A team works on one item at a time, each of its warps for 8 query heads.
template <int MODE, int DP, int TM, int W, int T, int S>
struct Attn {
    static constexpr bool kFp8 = MODE == MF_DT_F8E4M3 || MODE == MF_DT_F8E5M2;
    static constexpr bool kBf16 = MODE == MF_DT_BF16;
    // Weights are exp2(s - m), m a maximum less kBelow.  It is only replaced when a score exceeds it by kAbove: until
    // then the weights grow up to 2^kAbove and what is summed is not rescaled.  BF16 terms and float32 sums hold any
    // weight: m is a maximum itself.  f16 terms end at 2^16 and at 2^-24: 2^15 at the top leaves the small ones of
    // a token that leads by 18 (2^-26) 11 bits, where a maximum as m left none.
    static constexpr float kBelow = kBf16 ? 0.0f : 12.0f;
    static constexpr float kAbove = kBf16 ? 8.0f : 15.0f;
    static constexpr float kMost = kBf16 ? 1.0f : 4096.0f;  // 2^kBelow
    static constexpr int kBytes = kFp8 ? 1 : 2;
    static constexpr int kRow = DP * kBytes;          // bytes of a token's row
    static constexpr int kChunks = kRow / 16;         // 16-byte pieces of it
    static constexpr int kStage = 2 * T * kRow;       // keys, then values
    static constexpr int kBlocks = T / kBlock;
    static constexpr uint32_t kAll = T == 32 ? 0xffffffffu : 0xffffu;  // every token of a tile
    static constexpr int kSteps = DP / 16;            // products of 16 along head_dim
    static constexpr int kTeams = W / TM;
    static constexpr int kHeads = 8 * TM;             // query heads of an item, at most
    static constexpr int kFour = DP / 4;
    static constexpr int kPart = kHeads * (DP + 2);   // floats of a part in the workspace: out, then m, l
    static constexpr int kThreads = 32 * W;
    static constexpr int kRing = kTeams * S * kStage;
    static constexpr int kLd = DP + 4;                // floats of a staged head's row (spread over the banks)
    static constexpr int kStaged = 2 * kTeams * kHeads * kLd * 4;
    static constexpr int kBuffer = kRing > kStaged ? kRing : kStaged;
    static_assert(2 * kTeams <= 32, "a lane for each part of a CTA");
    static_assert(TM == 1 || kTeams < 16, "a barrier for each team");
    static_assert(W >= 2 && (T == kBlock || T == 2 * kBlock), "");

    struct Shared {
        int64_t warp_sum[W];            // tiles of the requests of each warp's threads
        int32_t thread_sum[kThreads];   // and of each thread's
        int32_t thread_nt[kThreads];    // tiles of an item of each thread's last request
        uint32_t warp_ctas[kFills][W];  // the CTAs that the requests of each warp get where each item has its own
        Part part[2 * kTeams];          // first and last part of each team
        float m[2 * kTeams][kHeads], l[2 * kTeams][kHeads];  // of the parts; m becomes their weight
        Joined joined[2 * kTeams];
        float joined_m[2 * kTeams][kHeads], joined_l[2 * kTeams][kHeads];
        float weight[kJoin][kHeads], top[kHeads], sum[kHeads];
        uint32_t mask[kTeams][S];       // tokens of each stage that are there
        int32_t items;                  // joined items
        int32_t won[2];                 // whether this CTA joins its group of the item of its slot
        int32_t won_groups[2];          // and whether it joins that item's groups
        int32_t first[2], last[2], size[2];  // that item's CTAs, and how many join at a time
    };
    static constexpr int kSharedBytes = kBuffer + static_cast<int>(sizeof(Shared));
};

// Piece `c` of row `row` of a tile: the pieces of a row are exchanged so that
// eight rows of one column fall on different banks.  (Rows 16 bytes longer
// than they are do that too, and need no exclusive-or, but then the 32-byte
// sectors of a copy cross those of shared memory: 102 instead of 92 us for 64
// requests of 2048 tokens, 32/8 heads of 128.)
template <int CHUNKS>
__device__ __forceinline__ uint32_t swizzled(int row, int c) {
    if constexpr (CHUNKS >= 8) return static_cast<uint32_t>(row * CHUNKS + (c ^ (row & 7))) * 16u;
    else return static_cast<uint32_t>(row * CHUNKS + (c ^ ((row >> 1) & (CHUNKS - 1)))) * 16u;
}

// The same for an even piece c more, from the place of a row's piece 0 or 1 (stages start at multiples of 128).
template <int CHUNKS>
__device__ __forceinline__ uint32_t pieces_on(uint32_t at, int c) {
    if constexpr (CHUNKS >= 8) return (at ^ static_cast<uint32_t>((c & 7) * 16)) + static_cast<uint32_t>((c >> 3) * 128);
    else return at ^ static_cast<uint32_t>(c * 16);
}

// Write `f` (4 floats of head h, elements d..d+3, normalised) to the output; a run of parts has a float32 one.
template <bool PART>
__device__ __forceinline__ void store_out4(const AttnArgs& a, int32_t r, int32_t head, int d, float4 f) {
    if (d >= a.head_dim) return;
    if constexpr (PART) {
        *reinterpret_cast<float4*>(a.out + 4 * (r * a.out_req + head * a.out_head + d)) = f;
        return;
    }
    char* p = a.out + 2 * (r * a.out_req + head * a.out_head + d);
    const float v[4] = {f.x, f.y, f.z, f.w};
    uint32_t w[2];
    if (a.q_f16) encode4<MF_DT_F16>(v, w, 0);
    else encode4<MF_DT_BF16>(v, w, 0);
    *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
}

// l is at least K::kMost, the largest weight of a maximum: its logarithm is taken over that, which leaves it the low bits.  A run
// of parts leaves maximum and sum.
template <class K, bool PART>
__device__ __forceinline__ void store_lse(const AttnArgs& a, int32_t r, int32_t head, float m, float l) {
    if constexpr (PART) {
        reinterpret_cast<float2*>(a.lse)[static_cast<int64_t>(r) * a.q_heads + head] = make_float2(l == 0.0f ? -INFINITY : m, l);
        return;
    }
    if (!a.lse) return;
    a.lse[static_cast<int64_t>(r) * a.q_heads + head] =
        l == 0.0f ? -INFINITY : (m + K::kBelow + log2f(l * (1.0f / K::kMost))) * kLn2;
}

__device__ __forceinline__ float4 fma4(float4 f, float r, float4 acc) {
    return make_float4(__fmaf_rn(f.x, r, acc.x), __fmaf_rn(f.y, r, acc.y), __fmaf_rn(f.z, r, acc.z), __fmaf_rn(f.w, r, acc.w));
}
__device__ __forceinline__ float4 scale4(float4 f, float r) { return make_float4(f.x * r, f.y * r, f.z * r, f.w * r); }

// Query heads of an item: the first of them, how many, and their key-value head.
template <int HEADS>
struct Heads {
    int32_t kv, head0, count;
    __device__ __forceinline__ Heads(const AttnArgs& a, int32_t item) {
        kv = a.blocks == 1 ? item : item / a.blocks;
        head0 = kv * a.group + (item - kv * a.blocks) * HEADS;
        count = min(HEADS, (kv + 1) * a.group - head0);
    }
};

// One more arrival at a ticket that `count` CTAs share; true for the last one,
// which leaves the ticket at zero.  What every thread of the CTA wrote before
// the last barrier is visible to whoever arrives later (the release is
// cumulative over what the barrier ordered before it).
__device__ __forceinline__ bool arrive_last(int32_t* ticket, int32_t count) {
    int32_t old;
    asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(ticket) : "memory");
    if (old != count - 1) return false;
    *ticket = 0;
    return true;
}

// Joins parts 0 .. n-1 (n <= kJoin) at first + k * stride floats, but the first
// at at0 and the last at at_end: to the output if `to` is NULL, else to a part
// there.  All threads of the CTA; the parts pass through shared memory, as many
// at a time as it holds.
template <class K, int DP, bool PART>
__device__ __forceinline__ void join_parts(const AttnArgs& a, typename K::Shared& sh, unsigned char* smem, const float* first,
                                           int64_t stride, const float* at0, const float* at_end, int32_t n, const Joined& w,
                                           float* to) {
    constexpr int kFloats = K::kHeads * DP, kRound = K::kBuffer / (kFloats * 4);
    constexpr int kEach = (K::kHeads * K::kFour + K::kThreads - 1) / K::kThreads;
    static_assert(kRound >= 1, "");
    const int tid = threadIdx.x, lane = tid & 31, used = w.heads * K::kFour;
    const float* in = reinterpret_cast<const float*>(smem);
    const uint32_t buffer = static_cast<uint32_t>(__cvta_generic_to_shared(smem));
    auto part = [&](int k) { return k == 0 ? at0 : k == n - 1 ? at_end : first + k * stride; };
    float4 acc[kEach];
#pragma unroll
    for (int e = 0; e < kEach; ++e) acc[e] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int k0 = 0; k0 < n; k0 += kRound) {
        const int k1 = min(k0 + kRound, n);
#pragma unroll 1
        for (int k = k0; k < k1; ++k) {
            const float* from = part(k);
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = tid + e * K::kThreads;
                if (i < used) cp_async16(buffer + ((k - k0) * kFloats + i * 4) * 4, from + i * 4, 16u);
            }
        }
        cp_async_commit();
        if (k0 == 0) {
            // the weights meanwhile: a warp for each head, a lane for each part
#pragma unroll 1
            for (int h = tid >> 5; h < w.heads; h += K::kThreads / 32) {
                const float* of = part(lane < n ? lane : 0) + kFloats + h;
                const float m = lane < n ? __ldcg(of) : -INFINITY, l = lane < n ? __ldcg(of + K::kHeads) : 0.0f;
                float top = m;
#pragma unroll
                for (int d = 1; d < kJoin; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                top = __shfl_sync(0xffffffffu, top, 0);
                const float by = rescale(m, top);
                float sum = l * by;
#pragma unroll
                for (int d = 1; d < kJoin; d <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
                if (lane < kJoin) sh.weight[lane][h] = by;
                if (lane == 0) {
                    sh.top[h] = top;
                    sh.sum[h] = sum;
                }
            }
        }
        cp_async_wait<0>();
        __syncthreads();
#pragma unroll 1
        for (int k = k0; k < k1; ++k) {
#pragma unroll
            for (int e = 0; e < kEach; ++e) {
                const int i = tid + e * K::kThreads;
                if (i < used)
                    acc[e] = fma4(*reinterpret_cast<const float4*>(in + (k - k0) * kFloats + i * 4), sh.weight[k][i / K::kFour], acc[e]);
            }
        }
        __syncthreads();
    }
    const float vs = a.v_scale ? a.v_scale[w.kv] : 1.0f;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
        const int i = tid + e * K::kThreads, h = i / K::kFour, d = i % K::kFour * 4;
        if (i >= used) break;
        const float sum = sh.sum[h];
        if (to) {
            *reinterpret_cast<float4*>(to + i * 4) = acc[e];
            if (d == 0) {
                to[kFloats + h] = sh.top[h];
                to[kFloats + K::kHeads + h] = sum;
            }
        } else {
            store_out4<PART>(a, w.r, w.head0 + h, d, scale4(acc[e], sum == 0.0f ? 0.0f : __fdiv_rn(vs, sum)));
            if (d == 0) store_lse<K, PART>(a, w.r, w.head0 + h, sh.top[h], sum);
        }
    }
    __syncthreads();
}

// CTAs of an item of nt tiles where each item has its own, so that a team has up to kOwnTiles[fill] tiles.  A handful
// of tiles takes no longer than the join between two CTAs; the first limit whose CTAs are all there is taken, and a
// request alone gets all there are when it has more than one CTA's.  8 requests of 1000 tokens, 32/8 heads of 128:
// 16.1 us with the row of tiles cut evenly, 13.4 so; 8 of 2000: 22.2 and 20.8.
__device__ constexpr int kOwnTiles[kFills] = {3, 6, 12};
template <class K>
__device__ __forceinline__ int32_t ctas_of(const AttnArgs& a, int32_t nt, int fill) {
    if (nt == 0) return 0;
    const int32_t n = (nt - 1) / (K::kTeams * kOwnTiles[fill]) + 1;
    if (n == 1 || a.n_requests > 1) return n;
    return max(min(static_cast<int32_t>(gridDim.x) / a.items, (nt - 1) / K::kTeams + 1), 1);
}

// PART: the requests' tokens from own_first on alone, to a float32 out.
template <int MODE, int DP, int TM, int W, int T, int S, bool PART>
__global__ void __launch_bounds__(32 * W, 1) paged_attn_kernel(const AttnArgs a) {
    using K = Attn<MODE, DP, TM, W, T, S>;
    extern __shared__ __align__(128) unsigned char smem[];
    auto& sh = *reinterpret_cast<typename K::Shared*>(smem + K::kBuffer);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int team = warp / TM, member = warp % TM;
    const int g = lane >> 2, j = lane & 3;  // row and column pair of a product's fragment
    const int32_t items = a.items, used_heads = a.used_heads.d;

    after_previous();
    let_next_start();
    // the tiles of thread i's `per` consecutive requests
    const int32_t per = (a.n_requests + K::kThreads - 1) / K::kThreads;
    int64_t sum = 0;
    bool empty = false;
    int32_t nt_of = 0;
    for (int32_t i = 0; i < per; ++i) {
        const int32_t r = tid * per + i;
        if (r >= a.n_requests) break;
        const int32_t nt = tiles_of<T>(span_of<PART>(a, r));
        sum += static_cast<int64_t>(nt) * items;
        nt_of = nt;
        empty |= nt == 0 && r % gridDim.x == blockIdx.x;
    }
    sh.thread_sum[tid] = static_cast<int32_t>(sum);
    const bool few = static_cast<int64_t>(a.n_requests) * items <= gridDim.x;  // there may be CTAs for each item
    if (few) {
        sh.thread_nt[tid] = nt_of;
#pragma unroll 1
        for (int f = 0; f < kFills; ++f) {
            const int64_t mine = static_cast<int64_t>(ctas_of<K>(a, nt_of, f)) * items;
            const uint32_t all = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(mine < (1 << 20) ? mine : 1 << 20));
            if (lane == 0) sh.warp_ctas[f][warp] = all;
        }
    }
    {
        const int64_t low = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum & 0xffff));
        const int64_t high = __reduce_add_sync(0xffffffffu, static_cast<uint32_t>(sum >> 16 < (1 << 26) ? sum >> 16 : 1 << 26));
        if (lane == 0) sh.warp_sum[warp] = (high << 16) + low;
    }
    if (tid < 2 * K::kTeams) sh.part[tid].start = -1;
    if (__syncthreads_or(empty)) {
        // requests that see nothing
        for (int32_t r = blockIdx.x; r < a.n_requests; r += gridDim.x) {
            if (tiles_of<T>(span_of<PART>(a, r)) > 0) continue;
            for (int i = tid; i < a.q_heads * (a.head_dim / 4); i += K::kThreads)
                store_out4<PART>(a, r, i / (a.head_dim / 4), i % (a.head_dim / 4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
            for (int i = tid; i < a.q_heads; i += K::kThreads) store_lse<K, PART>(a, r, i, 0.0f, 0.0f);
        }
    }
    // Of W values of warps and the values of their threads, in a row: the thread that place `key` is at, and how far into it.
    auto locate = [&](int64_t of_warp, auto of_threads, int32_t key, int32_t& into) {
        int64_t in_front = of_warp;
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) {
            const int64_t x = __shfl_up_sync(0xffffffffu, in_front, d);
            if (lane >= d) in_front += x;
        }
        in_front -= of_warp;
        const int in_warp = 31 - __clz(__ballot_sync(0xffffffffu, lane < W && in_front <= key));
        const int32_t before = static_cast<int32_t>(__shfl_sync(0xffffffffu, in_front, in_warp));
        const int32_t of_thread = of_threads(32 * in_warp + lane);
        int32_t ahead = of_thread;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int32_t x = __shfl_up_sync(0xffffffffu, ahead, d);
            if (lane >= d) ahead += x;
        }
        ahead -= of_thread;
        const int in_lane = 31 - __clz(__ballot_sync(0xffffffffu, before + ahead <= key));
        into = key - before - __shfl_sync(0xffffffffu, ahead, in_lane);
        return 32 * in_warp + in_lane;
    };
    // Each item has CTAs of its own where those suffice; else the row of all tiles is cut evenly.
    const int64_t tiles_of_warp = lane < W ? sh.warp_sum[lane] : 0;
    int64_t total64 = tiles_of_warp;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) total64 += __shfl_xor_sync(0xffffffffu, total64, d);
    uint32_t ctas_of_warp = 0, all_ctas = 0xffffffffu;
    int fill = -1;
    while (few && all_ctas > gridDim.x && ++fill < kFills) {
        ctas_of_warp = lane < W ? sh.warp_ctas[fill][lane] : 0;
        all_ctas = __reduce_add_sync(0xffffffffu, ctas_of_warp);
    }
    if (total64 == 0) return;
    if (total64 > 0x7fffffff) {
        if (tid == 0) atomicExch(a.status, MF_DEVICE_TOO_LARGE);
        return;
    }
    const bool own = all_ctas <= gridDim.x;
    const int32_t total = static_cast<int32_t>(total64), want = (total - 1) / K::kTeams + 1;
    const int32_t ctas = own ? static_cast<int32_t>(all_ctas) : min(want, static_cast<int32_t>(gridDim.x));
    if (blockIdx.x >= ctas) return;
    const Cut by_cta(total, ctas);
    const int32_t id = blockIdx.x * K::kTeams + team;
    Place<T, PART> at{};
    int32_t x0, my_tiles, own_first = 0, own_last = 0;  // first tile in the row (of the item, if it has its own CTAs), tiles
    if (own) {
        int32_t into;
        at.r = locate(ctas_of_warp, [&](int t) { return ctas_of<K>(a, sh.thread_nt[t], fill) * items; }, blockIdx.x, into);
        at.span = span_of<PART>(a, at.r);
        at.nt = tiles_of<T>(at.span);
        const int32_t each = ctas_of<K>(a, at.nt, fill);
        at.item = into / each;
        const int32_t nth = into - at.item * each;
        const Cut of_item(at.nt, each);
        const int32_t from = of_item.start(nth);
        const Cut by_team(of_item.start(nth + 1) - from, K::kTeams);
        x0 = at.t = from + by_team.start(team);
        my_tiles = from + by_team.start(team + 1) - x0;
        own_first = blockIdx.x - nth;
        own_last = own_first + each - 1;
    } else {
        const int32_t cta_tile = by_cta.start(blockIdx.x);
        const Cut by_team(by_cta.start(blockIdx.x + 1) - cta_tile, K::kTeams);
        x0 = cta_tile + by_team.start(team);
        my_tiles = cta_tile + by_team.start(team + 1) - x0;
        if (my_tiles > 0) {
            int32_t into;
            at.r = locate(tiles_of_warp, [&](int t) { return sh.thread_sum[t]; }, x0, into);
            if (per > 1) {
                for (int32_t r0 = at.r * per;; r0 += 32) {
                    const int32_t mine = r0 + lane < a.n_requests ? tiles_of<T>(span_of<PART>(a, r0 + lane)) * items : 0;
                    int32_t upto = mine;
#pragma unroll 1
                    for (int d = 1; d < 32; d <<= 1) {
                        const int32_t x = __shfl_up_sync(0xffffffffu, upto, d);
                        if (lane >= d) upto += x;
                    }
                    const uint32_t past = __ballot_sync(0xffffffffu, upto > into);
                    if (past || r0 + 32 >= a.n_requests) {
                        const int src = past ? __ffs(past) - 1 : 0;
                        at.r = r0 + src;
                        into -= __shfl_sync(0xffffffffu, upto - mine, src);
                        break;
                    }
                    into -= __shfl_sync(0xffffffffu, upto, 31);
                }
            }
            at.span = span_of<PART>(a, at.r);
            at.nt = tiles_of<T>(at.span);
            at.item = into / at.nt;
            at.t = into - at.item * at.nt;
        }
    }

    uint32_t qf[K::kSteps][2];
    float o[K::kSteps][4];
    float m[2], l[2];
    if (my_tiles > 0) {
        unsigned char* my_ring = smem + team * (S * K::kStage);
        const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(my_ring));
        Place<T, PART> load = at;
        int32_t to_load = my_tiles;
        const bool whole = a.page % kBlock == 0;         // a block lies in one page
        const bool dense = a.row_bytes == DP * K::kBytes;  // rows follow one another
        constexpr int kRows = 32 / K::kChunks > 0 ? 32 / K::kChunks : 1;  // rows that one instruction copies
        constexpr int kCopies = kBlock * K::kChunks / 32 / TM;            // of a block, by one warp
        static_assert(kCopies > 0, "");
        const int piece_row = lane / K::kChunks + member * (kCopies * kRows), piece = lane % K::kChunks;
        const int64_t lane_bytes = static_cast<int64_t>(piece_row) * a.row_bytes + piece * 16;
        const bool piece_in = piece * (16 / K::kBytes) < a.head_dim;
        const int64_t kv_gap = a.v - a.k;
        const int32_t lane_tok = whole ? 0 : lane & (T - 1);
        // of the blocks of the tile at `load` (or, blocks not being whole, of this lane's row): their pages, the pages'
        // entries in the table and the blocks' places in the pages.  Tokens are unsigned: the last tile of a request of
        // nearly 2^31 tokens ends past them.
        const char* head_at = nullptr;
        const int32_t* entry[K::kBlocks];
        int32_t page_no[K::kBlocks];
        uint32_t page_off[K::kBlocks], tok0 = 0;
        auto look_up = [&](bool new_item) {
            if (new_item) {
                tok0 = load.span.base + load.t * T;
                head_at = a.k + (a.blocks == 1 ? load.item : load.item / a.blocks) * a.head_bytes + lane_bytes;
            } else {
                tok0 += T;
            }
#pragma unroll
            for (int b = 0; b < K::kBlocks; ++b) {
                const uint32_t tok = tok0 + lane_tok + (whole ? b * kBlock : 0);
                if (new_item || !whole) {
                    const int32_t idx = tok / a.by_page;
                    page_off[b] = tok - idx * a.page;
                    entry[b] = a.table + load.r * a.table_stride + idx;
                } else {
                    page_off[b] += T;
#pragma unroll
                    for (int x = 0; x < K::kBlocks; ++x)
                        if (page_off[b] >= a.by_page.d) {
                            page_off[b] -= a.page;
                            ++entry[b];
                        }
                }
                if (tok < static_cast<uint32_t>(load.span.len)) page_no[b] = *entry[b];
            }
        };
        uint32_t partial = 0;  // stages that lack some of their tokens: those have a mask
        auto issue = [&](int stage) {
            if (to_load > 0) {
                const uint32_t to = ring + stage * K::kStage, first = load.span.first, len = load.span.len;
                bool ok[K::kBlocks], all = whole && tok0 >= first && tok0 + T <= len;
                int64_t at_block[K::kBlocks];
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b) {
                    ok[b] = static_cast<uint32_t>(page_no[b]) < a.n_pages;
                    all &= ok[b];
                    at_block[b] = static_cast<int64_t>(page_no[b]) * a.page_bytes + page_off[b] * a.row_bytes;
                }
                if (all) {
                    partial &= ~(1u << stage);
#pragma unroll
                    for (int b = 0; b < K::kBlocks; ++b) {
                        const char* kp = head_at + at_block[b];
                        const char* vp = kp + kv_gap;
                        if (piece_in && dense) {
#pragma unroll
                            for (int i = 0; i < kCopies; ++i) {
                                const uint32_t dst = to + b * kBlock * K::kRow + swizzled<K::kChunks>(i * kRows + piece_row, piece);
                                cp_async16(dst, kp + i * (kRows * DP * K::kBytes), 16u);
                                cp_async16(dst + T * K::kRow, vp + i * (kRows * DP * K::kBytes), 16u);
                            }
                        } else if (piece_in) {
#pragma unroll
                            for (int i = 0; i < kCopies; ++i) {
                                const uint32_t dst = to + b * kBlock * K::kRow + swizzled<K::kChunks>(i * kRows + piece_row, piece);
                                cp_async16(dst, kp + i * kRows * a.row_bytes, 16u);
                                cp_async16(dst + T * K::kRow, vp + i * kRows * a.row_bytes, 16u);
                            }
                        }
                    }
                } else {
                    // the row of this lane: whether it is there, and where
                    const int mine = whole ? (lane & (T - 1)) / kBlock : 0;
                    const uint32_t tok = tok0 + (lane & (T - 1));
                    const bool seen = tok >= first && tok < len;
                    const bool mine_ok = mine == 0 ? ok[0] : ok[K::kBlocks - 1];
                    if (seen && !mine_ok) atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                    const uint32_t mask = __ballot_sync(0xffffffffu, seen && mine_ok) & K::kAll;
                    partial = (partial & ~(1u << stage)) | (mask != K::kAll ? 1u << stage : 0u);
                    if (lane == 0) sh.mask[team][stage] = mask;
                    const int64_t row = (mine == 0 ? at_block[0] : at_block[K::kBlocks - 1]) + (whole ? (lane & (kBlock - 1)) * a.row_bytes : 0);
                    const char* base = head_at - static_cast<int64_t>(piece_row) * a.row_bytes;
#pragma unroll 2
                    for (int i = 0; i < K::kBlocks * kCopies; ++i) {
                        const int at_row = i / kCopies * kBlock + i % kCopies * kRows, rw = at_row + piece_row;
                        const char* kp = base + __shfl_sync(0xffffffffu, row, rw);
                        const bool get = (mask >> rw) & 1u;
                        if (piece_in) {
                            const uint32_t dst = to + swizzled<K::kChunks>(rw, piece);
                            cp_async16(dst, get ? kp : a.k, get ? 16u : 0u);
                            cp_async16(dst + T * K::kRow, get ? kp + kv_gap : a.k, get ? 16u : 0u);
                        }
                    }
                }
                if (--to_load > 0) {
                    load.next(a, items);
                    look_up(load.t == 0);
                }
            }
            cp_async_commit();
        };
        look_up(true);
        if (a.head_dim < DP) {  // what is past the head is never copied: zeros
            for (int i = member * 32 + lane; i < S * K::kStage / 16; i += 32 * TM)
                reinterpret_cast<uint4*>(my_ring)[i] = make_uint4(0, 0, 0, 0);
            team_sync<TM>(team);
        }
        // the queries of the item at `p`, as they are
        auto load_queries = [&](const Place<T, PART>& p) {
            const Heads<K::kHeads> hd(a, p.item);
            const int h = member * 8 + g;
            const char* q = a.q + 2 * (p.r * a.q_req + (hd.head0 + h) * a.q_head);
#pragma unroll
            for (int c = 0; c < K::kSteps; ++c) {
                const int d0 = K::kFp8 ? c * 16 + 4 * j : c * 16 + 2 * j;
                const int d1 = K::kFp8 ? d0 + 2 : d0 + 8;
                qf[c][0] = h < hd.count && d0 < a.head_dim ? *reinterpret_cast<const uint32_t*>(q + 2 * d0) : 0u;
                qf[c][1] = h < hd.count && d1 < a.head_dim ? *reinterpret_cast<const uint32_t*>(q + 2 * d1) : 0u;
            }
        };
        load_queries(at);

        // rows of this lane in the loads of a product's operands
        const int k_row = (lane & 7) + ((lane >> 3) & 1) * 8, k_piece = lane >> 4;
        const int v_row = K::kFp8 ? k_row : (lane & 7) + (lane >> 4) * 8, v_piece = K::kFp8 ? k_piece : (lane >> 3) & 1;
        const uint32_t k_at = ring + swizzled<K::kChunks>(k_row, k_piece);
        const uint32_t v_at = ring + T * K::kRow + swizzled<K::kChunks>(v_row, v_piece);
        const float cap = a.softcap * kLog2e;
        int stage = 0, fill = 0;  // the stages of the tile at hand and of the next to be copied
        int32_t done = 0;
        while (done < my_tiles) {
            const int32_t ta = at.t, tb = min(at.nt, ta + my_tiles - done);
            float scale[2], slope[2], less[2], high[2];  // less: m, or 0 while it is -inf; high: what raises m
            {
                // a new item; its queries were loaded while the one before it ended
                const Heads<K::kHeads> hd(a, at.item);
                float back = 1.0f;
                if constexpr (K::kFp8) {
                    // f16 queries, scaled by a power of two to a largest magnitude in [1, 2)
                    float top = 0.0f;
#pragma unroll
                    for (int c = 0; c < K::kSteps; ++c)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(qf[c][x], f0, f1);
                            else unpack2<true>(qf[c][x], f0, f1);
                            top = fmaxf(top, fmaxf(fabsf(f0), fabsf(f1)));
                        }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    const uint32_t field = __float_as_uint(top) >> 23;  // biased exponent
                    const bool scales = field >= 1 && field <= 254;
                    const uint32_t e = min(field, 253u);
                    const float fit = scales ? __uint_as_float((254u - e) << 23) : 1.0f;
                    back = scales ? __uint_as_float(e << 23) : 1.0f;
#pragma unroll
                    for (int c = 0; c < K::kSteps; ++c)
#pragma unroll
                        for (int x = 0; x < 2; ++x) {
                            float f0, f1;
                            if (a.q_f16) unpack2<false>(qf[c][x], f0, f1);
                            else unpack2<true>(qf[c][x], f0, f1);
                            qf[c][x] = pack2<false>(f0 * fit, f1 * fit);
                        }
                }
                const float ks = a.k_scale ? a.k_scale[hd.kv] : 1.0f;
                // head 2j + x of this lane's columns: its scale is with the lanes of row 2j + x
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    const float b = __shfl_sync(0xffffffffu, back, (2 * j + x) * 4);
                    const int hx = member * 8 + 2 * j + x;
                    scale[x] = a.scale * ks * b;
                    scale[x] = a.softcap > 0.0f ? __fdiv_rn(scale[x], a.softcap) * (2.0f * kLog2e) : scale[x] * kLog2e;
                    slope[x] = a.slopes && hx < hd.count ? a.slopes[hd.head0 + hx] * kLog2e : 0.0f;
                    m[x] = high[x] = -INFINITY;
                    less[x] = l[x] = 0.0f;
                }
#pragma unroll
                for (int c = 0; c < K::kSteps; ++c)
#pragma unroll
                    for (int x = 0; x < 4; ++x) o[c][x] = 0.0f;
            }

#pragma unroll 1
            for (int32_t t = done == 0 ? ta - (S - 1) : ta; t < tb; ++t) {  // the first S - 1 rounds only fill the ring
                cp_async_wait<S - 2>();
                team_sync<TM>(team);
                issue(fill);
                fill = fill + 1 == S ? 0 : fill + 1;
                if (t < ta) continue;

                // S^T = K Q^T, two chains of sums
                const uint32_t keys = k_at + stage * K::kStage, values = v_at + stage * K::kStage;
                const uint32_t mask = (partial >> stage) & 1u ? sh.mask[team][stage] : K::kAll;
                float s[K::kBlocks][2][4];
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b) {
                    const uint32_t rows = keys + b * kBlock * K::kRow;
                    if constexpr (!K::kFp8) {
#pragma unroll
                        for (int c = 0; c < K::kSteps; ++c) {
                            uint32_t f[4];
                            ldsm4(f, pieces_on<K::kChunks>(rows, 2 * c));
                            if (c < 2) mma16816<K::kBf16, true>(s[b][c & 1], f, qf[c][0], qf[c][1]);
                            else mma16816<K::kBf16>(s[b][c & 1], f, qf[c][0], qf[c][1]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < K::kSteps; c += 2) {
                            uint32_t f[4];
                            ldsm4(f, pieces_on<K::kChunks>(rows, c));
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                // four codes of a row: elements 4j, 4j+1 take the place of the product's 2j, 2j+1,
                                // elements 4j+2, 4j+3 that of 2j+8, 2j+9 (the queries are laid out alike)
                                uint32_t f16[4];
                                fp8x4_to_f16<MODE>(f[2 * x], f16[0], f16[2]);
                                fp8x4_to_f16<MODE>(f[2 * x + 1], f16[1], f16[3]);
                                if (c == 0) mma16816<false, true>(s[b][x], f16, qf[c + x][0], qf[c + x][1]);
                                else mma16816<false>(s[b][x], f16, qf[c + x][0], qf[c + x][1]);
                            }
                        }
                    }
                }
                // scores of tokens g and g + 8 of each block, heads 2j and 2j + 1, times log2(e)
                float p[K::kBlocks][4], top[2] = {-INFINITY, -INFINITY};
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b)
#pragma unroll
                    for (int x = 0; x < 4; ++x) p[b][x] = (s[b][0][x] + s[b][1][x]) * scale[x & 1];
                if (a.softcap > 0.0f) {
                    float most = 0.0f;
#pragma unroll
                    for (int b = 0; b < K::kBlocks; ++b)
#pragma unroll
                        for (int x = 0; x < 4; ++x) most = fmaxf(most, fabsf(p[b][x]));
                    if (__any_sync(0xffffffffu, most >= kSmallCapped)) {
#pragma unroll
                        for (int b = 0; b < K::kBlocks; ++b)
#pragma unroll
                            for (int x = 0; x < 4; ++x)
                                p[b][x] = fabsf(p[b][x]) < kSmallCapped ? cap_small(p[b][x], a.softcap) : cap_large(p[b][x], cap);
                    } else {
#pragma unroll
                        for (int b = 0; b < K::kBlocks; ++b)
#pragma unroll
                            for (int x = 0; x < 4; ++x) p[b][x] = cap_small(p[b][x], a.softcap);
                    }
                }
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b) {
                    if (a.slopes) {
                        // distance to the newest token, <= 0
                        const float away = static_cast<float>(at.span.base + t * T - (at.span.len - 1) + b * kBlock + g);
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            p[b][x] = __fmaf_rn(slope[x & 1], away + (x & 2 ? 8.0f : 0.0f), p[b][x]);
                    }
                    if (mask != K::kAll) {
#pragma unroll
                        for (int x = 0; x < 4; ++x)
                            p[b][x] = (mask >> (b * kBlock + (x & 2 ? g + 8 : g))) & 1u ? p[b][x] : -INFINITY;
                    }
                    top[0] = fmaxf(top[0], fmaxf(p[b][0], p[b][2]));
                    top[1] = fmaxf(top[1], fmaxf(p[b][1], p[b][3]));
                }
                if (__any_sync(0xffffffffu, top[0] > high[0] || top[1] > high[1])) {
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 4));
                        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 8));
                        top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], 16));
                        const float next = fmaxf(top[x] - K::kBelow, m[x]);
                        const float r = rescale(m[x], next);
                        m[x] = next;
                        high[x] = __fadd_rd(next, K::kAbove);  // down: 2^16 would be past f16
                        less[x] = next == -INFINITY ? 0.0f : next;
                        l[x] *= r;
#pragma unroll
                        for (int c = 0; c < K::kSteps; ++c) {
                            o[c][x] *= r;
                            o[c][x + 2] *= r;
                        }
                    }
                }
                // weights; while nothing is seen, m is -inf and so are the scores: weights of 0
                uint32_t ph[K::kBlocks][2], pl[K::kBlocks][2];
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        p[b][x] = exp2_fast(p[b][x] - less[x & 1]);
                        l[x & 1] += p[b][x];
                    }
                    // high and low terms, tokens x heads -> heads x tokens
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const uint32_t high = pack2<K::kBf16>(p[b][2 * x], p[b][2 * x + 1]);
                        float f0, f1;
                        unpack2<K::kBf16>(high, f0, f1);
                        ph[b][x] = transpose8x8(high);
                        pl[b][x] = transpose8x8(pack2<K::kBf16>(p[b][2 * x] - f0, p[b][2 * x + 1] - f1));
                    }
                }

                // O^T += V^T P^T
#pragma unroll
                for (int b = 0; b < K::kBlocks; ++b) {
                    const uint32_t rows = values + b * kBlock * K::kRow;
                    if constexpr (!K::kFp8) {
#pragma unroll
                        for (int c = 0; c < K::kSteps; ++c) {
                            uint32_t f[4];
                            ldsm4_t(f, pieces_on<K::kChunks>(rows, 2 * c));
                            mma16816<K::kBf16>(o[c], f, ph[b][0], ph[b][1]);
                            mma16816<K::kBf16>(o[c], f, pl[b][0], pl[b][1]);
                        }
                    } else {
#pragma unroll
                        for (int c = 0; c < K::kSteps; c += 2) {
                            uint32_t f[4];
                            ldsm4_t(f, pieces_on<K::kChunks>(rows, c));
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                // a transposed pair of bytes holds elements 2g, 2g+1 of two tokens: row g of the product
                                // is element 2g, row g + 8 element 2g + 1
                                uint32_t f16[4];
                                fp8x4_to_f16_strided<MODE>(f[2 * x], f16[0], f16[1]);
                                fp8x4_to_f16_strided<MODE>(f[2 * x + 1], f16[2], f16[3]);
                                mma16816<false>(o[c + x], f16, ph[b][0], ph[b][1]);
                                mma16816<false>(o[c + x], f16, pl[b][0], pl[b][1]);
                            }
                        }
                    }
                }

                stage = stage + 1 == S ? 0 : stage + 1;
            }
            done += tb - ta;
            Place<T, PART> following = at;
            following.t = tb - 1;
            const bool ends = tb == at.nt, stops = done == my_tiles;  // the item, this team's run
            if (!stops) {
                following.next(a, items);
                load_queries(following);
            }
            {
                const bool all_of_it = ends && ta == 0;
                const Heads<K::kHeads> hd(a, at.item);
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 4);
                    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 8);
                    l[x] += __shfl_xor_sync(0xffffffffu, l[x], 16);
                }
                if (all_of_it) {
                    const float vs = a.v_scale ? a.v_scale[hd.kv] : 1.0f;
                    float f[2];
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int h = member * 8 + 2 * j + x;
                        f[x] = l[x] == 0.0f ? 0.0f : __fdiv_rn(vs, l[x]);
                        if (g == 0 && h < hd.count) store_lse<K, PART>(a, at.r, hd.head0 + h, m[x], l[x]);
                    }
                    char* out = a.out + (PART ? 4 : 2) * (at.r * a.out_req + hd.head0 * a.out_head);
#pragma unroll
                    for (int c = 0; c < K::kSteps; ++c) {
                        if constexpr (PART) {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int h = member * 8 + 2 * j + x;
                                const int d0 = K::kFp8 ? c * 16 + 2 * g : c * 16 + g, d1 = K::kFp8 ? d0 + 1 : d0 + 8;
                                float* to = reinterpret_cast<float*>(out) + h * a.out_head;
                                if (h < hd.count && d0 < a.head_dim) to[d0] = o[c][x] * f[x];
                                if (h < hd.count && d1 < a.head_dim) to[d1] = o[c][x + 2] * f[x];
                            }
                        } else if constexpr (!K::kFp8) {
                            // elements x heads -> heads x elements
                            const uint32_t u = transpose8x8(pack2<K::kBf16>(o[c][0] * f[0], o[c][1] * f[1]));
                            const uint32_t w = transpose8x8(pack2<K::kBf16>(o[c][2] * f[0], o[c][3] * f[1]));
                            const int h = member * 8 + g, d = c * 16 + 2 * j;
                            char* to = out + 2 * (h * a.out_head + d);
                            if (h < hd.count && d < a.head_dim) *reinterpret_cast<uint32_t*>(to) = u;
                            if (h < hd.count && d + 8 < a.head_dim) *reinterpret_cast<uint32_t*>(to + 16) = w;
                        } else {
#pragma unroll
                            for (int x = 0; x < 2; ++x) {
                                const int h = member * 8 + 2 * j + x, d = c * 16 + 2 * g;
                                const float u = o[c][x] * f[x], w = o[c][x + 2] * f[x];
                                const uint32_t two = a.q_f16 ? pack2<false>(u, w) : pack2<true>(u, w);
                                if (h < hd.count && d < a.head_dim) *reinterpret_cast<uint32_t*>(out + 2 * (h * a.out_head + d)) = two;
                            }
                        }
                    }
                } else if (!stops) {
                    // the item began in another team: its end waits in the workspace
                    float* part = a.team_part + static_cast<int64_t>(id) * K::kPart;
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        const int h = member * 8 + 2 * j + x;
                        if (h >= used_heads) break;
                        if (g == 0) {
                            sh.m[2 * team][h] = m[x];
                            sh.l[2 * team][h] = l[x];
                        }
#pragma unroll
                        for (int c = 0; c < K::kSteps; ++c) {
                            const int d0 = K::kFp8 ? c * 16 + 2 * g : c * 16 + g, d1 = K::kFp8 ? d0 + 1 : d0 + 8;
                            part[h * DP + d0] = o[c][x];
                            part[h * DP + d1] = o[c][x + 2];
                        }
                    }
                }
                if (!all_of_it && lane == 0 && member == 0) {
                    Part& p = sh.part[2 * team + (stops ? 1 : 0)];
                    p.start = x0 + done - tb;
                    p.r = at.r;
                    p.item = at.item;
                    p.nt = at.nt;
                    p.ta = ta;
                    p.tb = tb;
                }
            }
            at = following;
        }
        cp_async_wait<0>();
    }
    __syncthreads();  // every ring is done with: the last parts are staged there
    float* staged = reinterpret_cast<float*>(smem);  // [parts][heads][kLd]
    if (sh.part[2 * team].start >= 0) {
        // the first part comes back from the workspace
        const float* from = a.team_part + static_cast<int64_t>(id) * K::kPart + member * 8 * DP;
        const uint32_t to = static_cast<uint32_t>(__cvta_generic_to_shared(staged + (2 * team * K::kHeads + member * 8) * K::kLd));
#pragma unroll 1
        for (int i = lane; i < 8 * K::kFour; i += 32)
            cp_async16(to + (i / K::kFour * K::kLd + i % K::kFour * 4) * 4, from + i * 4, 16u);
    }
    cp_async_commit();
    if (sh.part[2 * team + 1].start >= 0) {
        float* mine = staged + (2 * team + 1) * (K::kHeads * K::kLd);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int h = member * 8 + 2 * j + x;
            if (h >= used_heads) break;
            if (g == 0) {
                sh.m[2 * team + 1][h] = m[x];
                sh.l[2 * team + 1][h] = l[x];
            }
#pragma unroll
            for (int c = 0; c < K::kSteps; ++c) {
                const int d0 = K::kFp8 ? c * 16 + 2 * g : c * 16 + g, d1 = K::kFp8 ? d0 + 1 : d0 + 8;
                mine[h * K::kLd + d0] = o[c][x];
                mine[h * K::kLd + d1] = o[c][x + 2];
            }
        }
    }
    constexpr int kParts = 2 * K::kTeams;
    // the joined items: runs of consecutive parts with one start
    const int32_t start = lane < kParts ? sh.part[lane].start : -1;
    const uint32_t have = __ballot_sync(0xffffffffu, start >= 0), lower = have & ((1u << lane) - 1u);
    const int32_t left = __shfl_sync(0xffffffffu, start, lower ? 31 - __clz(lower) : lane);
    const uint32_t leads = __ballot_sync(0xffffffffu, start >= 0 && (!lower || left != start));
    if (leads == 0) return;
    const uint32_t up_to = leads & (0xffffffffu >> (31 - lane));   // leads at or before this lane
    const uint32_t after = leads & ~(0xffffffffu >> (31 - lane));  // and behind it
    const int lead = up_to ? 31 - __clz(up_to) : lane, end = after ? __ffs(after) - 2 : 31;  // this lane's run of parts
    const int grp = __popc(up_to) - 1;
    if (warp == 0) {
        const uint32_t parts = have & (0xffffffffu << lead) & (0xffffffffu >> (31 - end));
        if (lane == lead && start >= 0) {
            const Part& p = sh.part[lane];
            const Heads<K::kHeads> hd(a, p.item);
            const bool whole = p.ta == 0 && sh.part[31 - __clz(parts)].tb == p.nt;
            sh.joined[grp] = Joined{parts, p.r, hd.kv, hd.head0, hd.count, whole ? -1 : p.ta > 0 ? 0 : 1, p.start, p.nt};
        }
        if (lane == 0) sh.items = __popc(leads);
    }
    __syncthreads();

    // Join the parts of each item inside the CTA.  First the parts' weights: a warp for each head, a lane for each part.
    for (int h = warp; h < used_heads; h += W) {
        const bool is = start >= 0;
        const float mine = is ? sh.m[lane][h] : -INFINITY;
        float top = mine;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const float x = __shfl_up_sync(0xffffffffu, top, d);
            if (lane - d >= lead) top = fmaxf(top, x);
        }
        top = __shfl_sync(0xffffffffu, top, end);
        const float w = rescale(mine, top);
        float sum_l = is ? sh.l[lane][h] * w : 0.0f;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const float x = __shfl_up_sync(0xffffffffu, sum_l, d);
            if (lane - d >= lead) sum_l += x;
        }
        sum_l = __shfl_sync(0xffffffffu, sum_l, end);
        if (is) sh.m[lane][h] = w;
        if (is && lane == lead) {
            sh.joined_m[grp][h] = top;
            sh.joined_l[grp][h] = sum_l;
        }
    }
    cp_async_wait<0>();
    __syncthreads();
    const int32_t joined = sh.items;
    for (int i = tid; i < joined * used_heads * K::kFour; i += K::kThreads) {
        const uint32_t e = static_cast<uint32_t>(i) / K::kFour;
        const int which = e / a.used_heads, h = e - which * used_heads, d = i % K::kFour * 4;
        const Joined& w = sh.joined[which];
        if (h >= w.heads) continue;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (uint32_t parts = w.parts; parts;) {
            float4 f[4];
            int k[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                k[x] = parts ? __ffs(parts) - 1 : -1;
                parts &= parts - 1;
                if (k[x] >= 0) f[x] = *reinterpret_cast<const float4*>(staged + (k[x] * K::kHeads + h) * K::kLd + d);
            }
#pragma unroll
            for (int x = 0; x < 4; ++x)
                if (k[x] >= 0) acc = fma4(f[x], sh.m[k[x]][h], acc);
        }
        const float top = sh.joined_m[which][h], sum_l = sh.joined_l[which][h];
        if (w.slot < 0) {
            const float vs = a.v_scale ? a.v_scale[w.kv] : 1.0f;
            store_out4<PART>(a, w.r, w.head0 + h, d, scale4(acc, sum_l == 0.0f ? 0.0f : __fdiv_rn(vs, sum_l)));
            if (d == 0) store_lse<K, PART>(a, w.r, w.head0 + h, top, sum_l);
        } else {
            float* to = a.cta_part + (static_cast<int64_t>(blockIdx.x) * 3 + w.slot) * K::kPart;
            *reinterpret_cast<float4*>(to + h * DP + d) = acc;
            if (d == 0) {
                to[K::kHeads * DP + h] = top;
                to[K::kHeads * DP + K::kHeads + h] = sum_l;
            }
        }
    }

    // Join between CTAs: the last of an item's CTAs to arrive does it.  More than kJoin join in groups, then the groups.
    if (sh.joined[0].slot != 0 && sh.joined[joined - 1].slot != 1) return;
    __syncthreads();
    if (tid < 64 && lane == 0) {
        const Joined& w = sh.joined[warp == 0 ? 0 : joined - 1];
        if (w.slot == warp) {
            const int32_t first = own ? own_first : by_cta.part_of(w.start);
            const int32_t last = own ? own_last : by_cta.part_of(w.start + w.nt - 1), n = last - first + 1;
            const int32_t size = n <= kJoin ? n : max(12, (n + kJoin - 1) / kJoin);
            const int32_t lo = first + (static_cast<int32_t>(blockIdx.x) - first) / size * size;
            const int32_t here = min(size, last - lo + 1);
            sh.first[warp] = first;
            sh.last[warp] = last;
            sh.size[warp] = size;
            // a group of one has no ticket: that CTA's may be the next item's
            sh.won[warp] = here == 1 || arrive_last(a.tickets + lo, here);
        } else {
            sh.won[warp] = 0;
        }
    }
    __syncthreads();
    constexpr int64_t kCta = 3 * K::kPart;
#pragma unroll 1
    for (int slot = 0; slot < 2; ++slot) {
        if (!sh.won[slot]) continue;
        const Joined w = sh.joined[slot == 0 ? 0 : joined - 1];
        const int32_t first = sh.first[slot], last = sh.last[slot], size = sh.size[slot];
        const int32_t groups = (last - first) / size + 1, lo = first + (static_cast<int32_t>(blockIdx.x) - first) / size * size;
        // a group's result goes to slot 2 of its first CTA; a group of one, an item's last CTA (where the next item may
        // have its first group), is its own result
        int32_t n = min(size, last - lo + 1);
        const float* parts = a.cta_part + lo * kCta;
        const float *at0 = parts + (lo == first ? K::kPart : 0), *at_end = parts + (n - 1) * kCta;
        int64_t stride = kCta;
        float* to = groups == 1 ? nullptr : a.cta_part + lo * kCta + 2 * K::kPart;
#pragma unroll 1
        for (int level = 0; level < 2; ++level) {
            if (level == 1) {
                if (groups == 1) break;
                if (tid == 0) sh.won_groups[slot] = arrive_last(a.tickets + gridDim.x + first, groups);
                __syncthreads();
                if (!sh.won_groups[slot]) break;
                const int32_t in_last = (last - first) % size + 1;
                parts = at0 = a.cta_part + first * kCta + 2 * K::kPart;
                at_end = a.cta_part + (last - in_last + 1) * kCta + (in_last == 1 ? 0 : 2 * K::kPart);
                stride = kCta * size;
                n = groups;
                to = nullptr;
            }
            if (to == nullptr || n > 1) join_parts<K, DP, PART>(a, sh, smem, parts, stride, at0, at_end, n, w, to);
        }
    }
}

// ------------------------------------------------------------------ host

struct Kernel {
    void (*fn)(AttnArgs);
    void (*part_fn)(AttnArgs);
    int threads, shared, part_floats, teams;
};

template <int MODE, int DP, int TM, int W, int T, int S>
Kernel kernel_of() {
    using K = Attn<MODE, DP, TM, W, T, S>;
    static_assert(K::kSharedBytes <= 232448, "shared memory of one CTA");
    return Kernel{paged_attn_kernel<MODE, DP, TM, W, T, S, false>, paged_attn_kernel<MODE, DP, TM, W, T, S, true>, K::kThreads, K::kSharedBytes, K::kPart, K::kTeams};
}

// Warps, tokens of a tile and stages: about 192 KB of ring per SM, the bytes in flight that keep HBM busy.
template <int MODE>
Kernel pick_shape(int group, int head_dim) {
    constexpr bool fp8 = MODE == MF_DT_F8E4M3 || MODE == MF_DT_F8E5M2;
    if (group <= 8) {
        if (head_dim <= 64) return kernel_of<MODE, 64, 1, 12, 32, fp8 ? 4 : 2>();
        if (head_dim <= 128) return kernel_of<MODE, 128, 1, 12, fp8 ? 32 : 16, 2>();
        return kernel_of<MODE, 256, 1, fp8 ? 8 : 6, 16, fp8 ? 3 : 2>();
    }
    if (head_dim <= 64) return kernel_of<MODE, 64, 2, 12, 32, 4>();
    if (head_dim <= 128) return kernel_of<MODE, 128, 2, 12, fp8 ? 32 : 16, 4>();
    return kernel_of<MODE, 256, 2, 12, 16, fp8 ? 4 : 2>();
}
Kernel pick(int cache_dtype, int group, int head_dim) {
    switch (cache_dtype) {
    case MF_DT_BF16: return pick_shape<MF_DT_BF16>(group, head_dim);
    case MF_DT_F16: return pick_shape<MF_DT_F16>(group, head_dim);
    case MF_DT_F8E4M3: return pick_shape<MF_DT_F8E4M3>(group, head_dim);
    default: return pick_shape<MF_DT_F8E5M2>(group, head_dim);
    }
}

}  // namespace
}  // namespace mf

using namespace mf;

struct mf_paged_attn_s {
    mf_paged_attn_config config;
    Kernel kernel;
    AttnArgs args;
    void* workspace;
    int device, ctas;
};

extern "C" int mf_paged_attn_create(const mf_paged_attn_config* config, mf_paged_attn* handle) {
    MF_ENTER();
    if (!config || !handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_paged_attn_create: NULL argument");
    *handle = nullptr;
    const mf_paged_attn_config& c = *config;
    const mf_cache_layout& k = c.cache;
    if (c.q_dtype != MF_DT_BF16 && c.q_dtype != MF_DT_F16)
        return fail(MF_ERR_DTYPE_UNSUPPORTED, "mf_paged_attn_create: queries of dtype %d (BF16 and F16 are supported)", c.q_dtype);
    if (!is_fp8(k.dtype) && k.dtype != c.q_dtype)
        return fail(MF_ERR_DTYPE_MISMATCH, "mf_paged_attn_create: cache dtype %d is neither FP8 nor the queries' %d", k.dtype,
                    c.q_dtype);
    if (k.kv_heads <= 0 || c.q_heads <= 0 || c.q_heads % k.kv_heads || c.q_heads > 65536)
        return fail(MF_ERR_SHAPE_INVALID, "mf_paged_attn_create: %d query heads over %d key-value heads", c.q_heads, k.kv_heads);
    const int step = is_fp8(k.dtype) ? 16 : 8;
    if (k.head_dim <= 0 || k.head_dim > 256 || k.head_dim % step)
        return fail(MF_ERR_SHAPE_INVALID, "mf_paged_attn_create: head_dim %d must be a multiple of %d up to 256", k.head_dim, step);
    if (k.page_size <= 0 || k.n_pages < 0 || c.max_pages <= 0 || c.table_stride < c.max_pages)
        return fail(MF_ERR_SHAPE_INVALID, "mf_paged_attn_create: %lld pages of %d, table rows of %d (stride %lld)",
                    (long long)k.n_pages, k.page_size, c.max_pages, (long long)c.table_stride);
    if (k.page_stride % step || k.token_stride % step || k.head_stride % step)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_paged_attn_create: cache strides must be multiples of 16 bytes");
    const int code = is_fp8(k.dtype) ? 1 : 2;
    if (k.page_stride < 0 || k.token_stride < 0 || k.head_stride < 0 || k.page_stride > 0x7fffffffll / code ||
        k.token_stride > 0x7fffffffll / code / k.page_size)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_paged_attn_create: cache strides may not be negative, a page is below 2 GB");
    if (c.q_token_stride % 2 || c.q_head_stride % 2 || c.out_token_stride % 4 || c.out_head_stride % 4)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_paged_attn_create: query strides must be even, output strides multiples of 4");
    if (c.window < 0 || !(c.softcap >= 0.0f && c.softcap < INFINITY))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_paged_attn_create: window %d, softcap %g", c.window, c.softcap);
    const int group = c.q_heads / k.kv_heads;
    Kernel kernel = pick(k.dtype, group, k.head_dim);
    MF_CUDA_CHECK(cudaFuncSetAttribute(reinterpret_cast<const void*>(kernel.fn), cudaFuncAttributeMaxDynamicSharedMemorySize,
                                       kernel.shared));
    const int ctas = state().sm_count;
    const size_t team_part = static_cast<size_t>(ctas) * kernel.teams * kernel.part_floats * 4;
    const size_t cta_part = static_cast<size_t>(ctas) * 3 * kernel.part_floats * 4;
    const size_t tickets = (static_cast<size_t>(ctas) * 8 + 255) / 256 * 256;
    const size_t bytes = tickets + team_part + cta_part;
    mf_paged_attn_s* h = new (std::nothrow) mf_paged_attn_s{};
    if (!h) return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_paged_attn_create: out of host memory");
    cudaError_t err = cudaMalloc(&h->workspace, bytes);
    if (err != cudaSuccess) {
        cudaGetLastError();
        delete h;
        if (err == cudaErrorMemoryAllocation)
            return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_paged_attn_create: %zu bytes: out of device memory", bytes);
        return cuda_fail(err, "mf_paged_attn_create: cudaMalloc");
    }
    err = cudaMemset(h->workspace, 0, tickets);
    if (err == cudaSuccess) err = cudaStreamSynchronize(nullptr);  // streams that do not wait for the default one may run it
    if (err != cudaSuccess) {
        cudaFree(h->workspace);
        delete h;
        return cuda_fail(err, "mf_paged_attn_create: cudaMemset");
    }
    char* w = static_cast<char*>(h->workspace);
    h->config = c;
    h->kernel = kernel;
    h->device = state().device;
    h->ctas = ctas;
    AttnArgs& a = h->args;
    a.slopes = c.slopes;
    a.k_scale = is_fp8(k.dtype) ? c.k_scale_inv : nullptr;
    a.v_scale = is_fp8(k.dtype) ? c.v_scale_inv : nullptr;
    a.tickets = reinterpret_cast<int32_t*>(w);
    a.team_part = reinterpret_cast<float*>(w + tickets);
    a.cta_part = reinterpret_cast<float*>(w + tickets + team_part);
    a.status = sticky_status_ptr();
    a.q_req = c.q_token_stride;
    a.q_head = c.q_head_stride;
    a.out_req = c.out_token_stride;
    a.out_head = c.out_head_stride;
    a.page_bytes = static_cast<int32_t>(k.page_stride * code);
    a.row_bytes = static_cast<int32_t>(k.token_stride * code);
    a.head_bytes = k.head_stride * code;
    a.table_stride = c.table_stride;
    a.n_pages = static_cast<uint32_t>(k.n_pages < 0x7fffffff ? k.n_pages : 0x7fffffff);
    a.q_heads = c.q_heads;
    a.group = group;
    a.blocks = group <= 8 ? 1 : (group + 15) / 16;
    a.items = k.kv_heads * a.blocks;
    a.head_dim = k.head_dim;
    a.page = k.page_size;
    a.max_pages = c.max_pages;
    a.by_page = divisor(a.page);
    a.used_heads = divisor(group < (group <= 8 ? 8 : 16) ? group : group <= 8 ? 8 : 16);
    a.window = c.window;
    a.q_f16 = c.q_dtype == MF_DT_F16;
    a.scale = c.scale;
    a.softcap = c.softcap;
    if (!a.status) {
        cudaFree(h->workspace);
        delete h;
        return fail(MF_ERR_CUDA, "mf_paged_attn_create: sticky status word unavailable");
    }
    *handle = h;
    return MF_OK;
}

extern "C" int mf_paged_attn_run(mf_paged_attn handle, const void* q, const void* k_cache, const void* v_cache,
                                 const int32_t* table, const int32_t* lens, int32_t n_requests, void* out, float* lse,
                                 mf_stream stream) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_paged_attn_run: handle is NULL");
    if (handle->device != state().device)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_paged_attn_run: the handle belongs to device %d", handle->device);
    if (n_requests < 0 || n_requests > kMaxRequests)
        return fail(MF_ERR_SHAPE_INVALID, "mf_paged_attn_run: %d requests (0 to 2^31 - 2^16)", n_requests);
    if (n_requests == 0) return MF_OK;
    if (!q || !k_cache || !v_cache || !table || !lens || !out)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_paged_attn_run: NULL buffer");
    if (!aligned16(k_cache) || !aligned16(v_cache))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_paged_attn_run: cache buffers must be 16-byte aligned");
    if (reinterpret_cast<uintptr_t>(q) % 4 || reinterpret_cast<uintptr_t>(out) % 8)
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_paged_attn_run: q must be 4-byte and out 8-byte aligned");
    AttnArgs a = handle->args;
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k_cache);
    a.v = static_cast<const char*>(v_cache);
    a.table = table;
    a.lens = lens;
    a.n_requests = n_requests;
    a.out = static_cast<char*>(out);
    a.lse = lse;
    const cudaError_t err = launch_overlapped(handle->kernel.fn, dim3(static_cast<unsigned>(handle->ctas)), handle->kernel.threads,
                                              handle->kernel.shared, static_cast<cudaStream_t>(stream), a);
    if (err != cudaSuccess) return cuda_fail(err, "mf_paged_attn_run");
    return MF_OK;
}

extern "C" int mf_paged_attn_destroy(mf_paged_attn handle) {
    if (!handle) return MF_OK;
    const cudaError_t err = free_workspace(handle->device, handle->workspace);
    delete handle;
    if (err != cudaSuccess) return cuda_fail(err, "mf_paged_attn_destroy");
    return MF_OK;
}

namespace mf {

int paged_attn_enable_parts(mf_paged_attn handle) {
    MF_CUDA_CHECK(cudaFuncSetAttribute(reinterpret_cast<const void*>(handle->kernel.part_fn),
                                       cudaFuncAttributeMaxDynamicSharedMemorySize, handle->kernel.shared));
    return MF_OK;
}

int paged_attn_run_parts(mf_paged_attn handle, const void* q, const void* k_cache, const void* v_cache, const int32_t* table,
                         const int32_t* lens, int32_t n_requests, const int32_t* own_first, const uint32_t* alone, const uint32_t* call,
                         float* out, float2* ml, cudaStream_t stream) {
    AttnArgs a = handle->args;
    a.q = static_cast<const char*>(q);
    a.k = static_cast<const char*>(k_cache);
    a.v = static_cast<const char*>(v_cache);
    a.table = table;
    a.lens = lens;
    a.n_requests = n_requests;
    a.own_first = own_first;
    a.alone = alone;
    a.call = call;
    a.out = reinterpret_cast<char*>(out);
    a.out_head = a.head_dim;
    a.out_req = static_cast<int64_t>(a.q_heads) * a.head_dim;
    a.lse = reinterpret_cast<float*>(ml);
    const cudaError_t err = launch_overlapped(handle->kernel.part_fn, dim3(static_cast<unsigned>(handle->ctas)), handle->kernel.threads,
                                              handle->kernel.shared, stream, a);
    return err == cudaSuccess ? MF_OK : cuda_fail(err, "mf_prefix_attn_run");
}

}  // namespace mf
