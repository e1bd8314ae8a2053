// beam.cu -- mf_beam_select_*: the best continuations over beams and vocabulary.
//
// For row k (a beam) of a batch entry with logits x and score s, token t scores
//   s + x[t] - L,  L = log sum_t exp x[t],
// and the n largest over all beams and tokens are wanted.  Inside a row the
// order of the scores is that of the logits, so a row is cut into segments, and
// a segment gives its n largest logits and its part (maximum, sum of
// exponentials) of L; the last CTA of a batch entry (a ticket) puts the Ls
// together and merges the segments' lists.  One launch, every logit read once.
//
// Bound: HBM, the logits.  A CTA streams its segment once, each thread keeping
// the maximum of what it met and a sum of exponentials relative to it, without a
// barrier; the n-th largest of the maxima is a bound that n logits reach, and only
// what the threads met whose maximum reaches it (n of 1024 parts) is read a second
// time, out of L2.  The few logits that reach the bound are ranked by counting.
// 64 x 8 rows of 128256 BF16 logits: 40.1 us (20 at the copy rate): CTAs end between
// 23 and 35 us, as SMs hold three or four of them, the last 5 of each on the bound,
// the second look and the ticket; the merge takes 4.  Collecting candidates on the
// way took 76: the threads of a warp diverge at each, and the bound has to be
// kept with barriers.  4 rows of 32000: 8.4 us, a chain of twelve dependent steps.
#include <new>

#include "mf_launch.cuh"
#include "mf_runtime.h"
#include "mf_vec.cuh"

namespace mf {
namespace {

constexpr int kThreads = 256;
constexpr int kMostOut = 128;        // results of a batch entry
constexpr int kMostBeams = 1024;     // beams of a batch entry
constexpr int kParts = 4;            // of what a thread meets, with a maximum each
constexpr int kGroups = 32;          // maxima that bound a list of up to kGroups
constexpr int kPicked = 512;         // logits that may be ranked by counting
// CTAs that a batch is cut into for every SM, at least.  Of the 64 x 8 rows below 3 make one segment each; 4 and 6 two (41 us for
// 39.5), 7 three (45).
constexpr int kCtas = 3;
constexpr float kLog2e = 1.44269504088896341f;
constexpr float kReach = 8.0f;       // that logits may exceed what a thread's sum is relative to

struct SelectArgs {
    const char* logits;
    const float* scores;
    const int32_t* ended;
    int64_t row_stride;   // elements
    int32_t vocab, beams, n_out, end_token;
    int32_t segments;     // of a row
    int32_t chunks;       // of a segment
    double* part_sum;     // [rows][segments]
    float* part_max;      // [rows][segments]
    float2* lists;        // [rows][segments][n_out]: logit and token (as bits), the largest first; -inf behind them
    int32_t* tickets;     // [batch], zero between runs
    float* scores_after;
    int32_t* tokens;
    int32_t* parents;
    int32_t* ended_after;
};

// Whether (a, i) comes in front of (b, j): the larger value, of equal ones the lower index.
template <class T>
__device__ __forceinline__ bool in_front(T a, int32_t i, T b, int32_t j) {
    return a > b || (a == b && i < j);
}

__device__ __forceinline__ float exp2_fast(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// Eight or four logits of a 16-byte vector.
template <int DT>
__device__ __forceinline__ void widen(const uint4& v, float* x) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == MF_DT_F32) {
            x[i] = __uint_as_float(w[i]);
        } else if constexpr (DT == MF_DT_BF16) {
            x[2 * i] = __uint_as_float(w[i] << 16);
            x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        } else {
            f16x2_to_f32x2(w[i], x[2 * i], x[2 * i + 1]);
        }
    }
}

// The vector of the logits from token t on, one by one; -inf behind the row.
template <int DT>
__device__ __forceinline__ uint4 some_logits(const char* row, int32_t t, int32_t vocab) {
    uint32_t w[4];
    if constexpr (DT == MF_DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = t + i < vocab ? reinterpret_cast<const uint32_t*>(row)[t + i] : 0xff800000u;
    } else {
        constexpr uint16_t kNone = DT == MF_DT_BF16 ? 0xff80 : 0xfc00;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint16_t lo = t + 2 * i < vocab ? reinterpret_cast<const uint16_t*>(row)[t + 2 * i] : kNone;
            const uint16_t hi = t + 2 * i + 1 < vocab ? reinterpret_cast<const uint16_t*>(row)[t + 2 * i + 1] : kNone;
            w[i] = lo | static_cast<uint32_t>(hi) << 16;
        }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// Bytes off .. off + 15 of two vectors that follow one another, off even and below 16.
__device__ __forceinline__ uint4 shifted(const uint4& lo, const uint4& hi, uint32_t off) {
    const uint32_t w[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t u[6], v[5];
#pragma unroll
    for (int i = 0; i < 6; ++i) u[i] = off & 8u ? w[i + 2] : w[i];
#pragma unroll
    for (int i = 0; i < 5; ++i) v[i] = off & 4u ? u[i + 1] : u[i];
    const uint32_t by = off & 2u ? 0x5432u : 0x3210u;
    return make_uint4(__byte_perm(v[0], v[1], by), __byte_perm(v[1], v[2], by), __byte_perm(v[2], v[3], by), __byte_perm(v[3], v[4], by));
}

template <class T>
struct Bound {
    T group[kGroups];
    T thread[kThreads];   // for more than kGroups results
    T value;
};
// What is ranked by counting.
template <class T>
struct Picked {
    T value[kPicked];
    int32_t index[kPicked];
    int32_t count;
    // how many of the first n are in front of (v, i)
    __device__ __forceinline__ int rank(T v, int32_t i, int n) const {
        int in = 0;
#pragma unroll 8
        for (int o = 0; o < n; ++o) in += in_front(value[o], index[o], v, i);
        return in;
    }
};
template <class T>
struct Best {
    T value[kThreads / 32];
    int32_t index[kThreads / 32];
};
// Two float32 at once.
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
__device__ __forceinline__ float2 mul2(float2 a, float2 b) { return __fmul2_rn(a, b); }

// The largest of a vector's logits; a NaN does not count.
template <int DT>
__device__ __forceinline__ float largest(const uint4& v) {
    if constexpr (DT == MF_DT_F32) {
        return fmaxf(fmaxf(__uint_as_float(v.x), __uint_as_float(v.y)), fmaxf(__uint_as_float(v.z), __uint_as_float(v.w)));
    } else {
        uint32_t m;
        if constexpr (DT == MF_DT_BF16)
            asm("{\n\t.reg .b32 a, b;\n\tmax.bf16x2 a, %1, %2;\n\tmax.bf16x2 b, %3, %4;\n\tmax.bf16x2 %0, a, b;\n\t}"
                : "=r"(m) : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
        else
            asm("{\n\t.reg .b32 a, b;\n\tmax.f16x2 a, %1, %2;\n\tmax.f16x2 b, %3, %4;\n\tmax.f16x2 %0, a, b;\n\t}"
                : "=r"(m) : "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w));
        float lo, hi;
        if constexpr (DT == MF_DT_BF16) {
            lo = __uint_as_float(m << 16);
            hi = __uint_as_float(m & 0xffff0000u);
        } else {
            f16x2_to_f32x2(m, lo, hi);
        }
        return fmaxf(lo, hi);
    }
}

struct SelectShared {
    float warp_max[kThreads / 32];
    double warp_sum[kThreads / 32];
    int32_t last;
    union {
        struct {
            Bound<float> bound;
            Picked<float> picked;
            Best<float> best;
            int32_t part[kPicked];
        } chunk;
        struct {
            Bound<double> bound;
            Picked<double> picked;
            Best<double> best;
        } entry;
    };
};

// A value that at least n of what the threads have reach, given each thread's largest: the n-th largest of the maxima
// over 32 groups of threads, or over the threads.  All threads; -inf where fewer than n maxima are above it.
template <class T>
__device__ __forceinline__ T bound_of(T mine, int n, Bound<T>& sh) {
    const int tid = threadIdx.x, lane = tid & 31;
    if (n <= kGroups) {
        T group = mine;
#pragma unroll
        for (int d = 1; d < kThreads / kGroups; d <<= 1) {
            const T other = __shfl_xor_sync(0xffffffffu, group, d);
            group = other > group ? other : group;
        }
        if (tid % (kThreads / kGroups) == 0) sh.group[tid / (kThreads / kGroups)] = group;
        __syncthreads();
        // every warp ranks the 32 itself, which saves a barrier
        const T v = sh.group[lane];
        int rank = 0;
#pragma unroll
        for (int i = 0; i < kGroups; ++i) rank += in_front(sh.group[i], i, v, lane);
        const uint32_t is = __ballot_sync(0xffffffffu, rank == n - 1);
        return __shfl_sync(0xffffffffu, v, __ffs(is) - 1);
    }
    sh.thread[tid] = mine;
    __syncthreads();
    int rank = 0;
#pragma unroll 4
    for (int i = 0; i < kThreads; ++i) rank += in_front(sh.thread[i], i, mine, tid);
    if (rank == n - 1) sh.value = mine;
    __syncthreads();
    return sh.value;
}

// The first of all threads' (value, index); all threads get it.
template <class T>
__device__ __forceinline__ void first_of_all(T& v, int32_t& i, Best<T>& sh) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 16; d; d >>= 1) {
        const T v2 = __shfl_xor_sync(0xffffffffu, v, d);
        const int32_t i2 = __shfl_xor_sync(0xffffffffu, i, d);
        if (in_front(v2, i2, v, i)) {
            v = v2;
            i = i2;
        }
    }
    __syncthreads();  // the round before has been read
    if (lane == 0) {
        sh.value[warp] = v;
        sh.index[warp] = i;
    }
    __syncthreads();
    for (int w = 0; w < kThreads / 32; ++w) {
        if (in_front(sh.value[w], sh.index[w], v, i)) {
            v = sh.value[w];
            i = sh.index[w];
        }
    }
}

// What the segments of batch entry `entry` left, put together by one CTA.
__device__ void merge_lists(const SelectArgs& a, int32_t entry, SelectShared& sh, double* base) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t row0 = entry * a.beams;
    for (int32_t k = warp; k < a.beams; k += kThreads / 32) {
        const int64_t row = row0 + k;
        double b = static_cast<double>(a.scores[row]);
        if (a.ended == nullptr || a.ended[row] == 0) {
            float top = -INFINITY;
            double sum = 0.0;
            for (int32_t c0 = 0; c0 < a.segments; c0 += 32) {
                const bool in = c0 + lane < a.segments;
                const float m = in ? __ldcg(a.part_max + row * a.segments + c0 + lane) : -INFINITY;
                const double s = in ? __ldcg(a.part_sum + row * a.segments + c0 + lane) : 0.0;
                float most = fmaxf(m, top);
#pragma unroll
                for (int d = 16; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
                // a part of -inf alone has a sum of zero; a NaN stays one
                const double here = m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(most));
                sum = (top == -INFINITY ? sum : sum * exp(static_cast<double>(top) - static_cast<double>(most))) + here;
                top = most;
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            b -= static_cast<double>(top) + log(sum);
        }
        // a beam without a finite sum, or without a finite score, offers nothing
        if (lane == 0) base[k] = b > -INFINITY && b < INFINITY ? b : -INFINITY;
    }
    __syncthreads();
    const int32_t n_lists = a.beams * a.segments;
    // entry e of list l, -inf if there is none
    auto get = [&](int32_t l, int32_t e, double& v, int32_t& i) {
        const int32_t k = l / a.segments;
        const double b = base[k];
        v = -INFINITY;
        i = 0x7fffffff;
        if (b == -INFINITY) return;
        if (a.ended != nullptr && a.ended[row0 + k] != 0) {
            if (e > 0 || l != k * a.segments) return;
            v = b;
            i = k * a.vocab + a.end_token;
            return;
        }
        const float2 x = __ldcg(a.lists + (static_cast<int64_t>(row0) * a.segments + l) * a.n_out + e);
        v = b + static_cast<double>(x.x);
        if (x.x != -INFINITY) i = k * a.vocab + __float_as_int(x.y);
    };
    auto put = [&](int32_t j, double v, int32_t i) {
        const int64_t to = static_cast<int64_t>(entry) * a.n_out + j;
        const bool there = v > -INFINITY;
        const int32_t k = there ? i / a.vocab : 0, token = there ? i - k * a.vocab : -1;
        a.scores_after[to] = static_cast<float>(v);
        a.tokens[to] = token;
        a.parents[to] = there ? row0 + k : -1;
        if (a.ended_after) a.ended_after[to] = there && token == a.end_token;
    };
    // Every thread's largest entry; entries that follow one another go to different groups of threads.  From one round to the next
    // the threads turn by some 3/8 of a list, an odd number: else a group has entries of one rank where n_out divides kGroups, and
    // the bound lets too many through (8 beams of 122286 in 480 lists, 16 results: 98 us).
    const int32_t entries = n_lists * a.n_out, first = tid % (kThreads / kGroups) * kGroups + tid / (kThreads / kGroups);
    const int32_t turn = ((a.n_out * 3 / 8 | 1) + a.n_out - kThreads % a.n_out) % a.n_out;
    double mine = -INFINITY, v;
    int32_t i;
#pragma unroll 4
    for (int32_t x0 = 0, at = first; x0 < entries; x0 += kThreads, at = (at + turn) & (kThreads - 1)) {
        const int32_t x = x0 + at;
        if (x >= entries) continue;
        const int32_t l = x / a.n_out;
        get(l, x - l * a.n_out, v, i);
        mine = v > mine ? v : mine;
    }
    const double bound = bound_of(mine, a.n_out, sh.entry.bound);
    auto& picked = sh.entry.picked;
    if (tid == 0) picked.count = 0;
    __syncthreads();
#pragma unroll 4
    for (int32_t x = tid; x < entries; x += kThreads) {
        const int32_t l = x / a.n_out;
        get(l, x - l * a.n_out, v, i);
        if (v >= bound && v > -INFINITY) {
            const int at = atomicAdd(&picked.count, 1);
            if (at < kPicked) {
                picked.value[at] = v;
                picked.index[at] = i;
            }
        }
    }
    __syncthreads();
    const int n = picked.count;
    if (n <= kPicked) {
        for (int x = tid; x < n; x += kThreads) {
            v = picked.value[x];
            i = picked.index[x];
            const int rank = picked.rank(v, i, n);
            if (rank < a.n_out) put(rank, v, i);
        }
        for (int j = n + tid; j < a.n_out; j += kThreads) put(j, -INFINITY, -1);
        return;
    }
    // many equal scores: one after the other, each the first behind the one before
    double last_v = INFINITY;
    int32_t last_i = -1;
#pragma unroll 1
    for (int j = 0; j < a.n_out; ++j) {
        double best = -INFINITY;
        int32_t best_i = 0x7fffffff;
        for (int32_t x = tid; x < entries; x += kThreads) {
            const int32_t l = x / a.n_out;
            get(l, x - l * a.n_out, v, i);
            if (in_front(last_v, last_i, v, i) && in_front(v, i, best, best_i)) {
                best = v;
                best_i = i;
            }
        }
        first_of_all(best, best_i, sh.entry.best);
        if (tid == 0) put(j, best, best_i);
        last_v = best;
        last_i = best_i;
    }
}

// The vector of the logits from token t on, wherever in memory the row begins: a thread's tokens do not depend on that, so
// that equal rows have equal sums, to the bit.
template <int DT>
__device__ __forceinline__ uint4 load_vector(const char* row, int32_t t, int32_t vocab) {
    constexpr int kPer = DT == MF_DT_F32 ? 4 : 8, kBytes = 16 / kPer;  // logits of a vector, bytes of one
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u);
    const int32_t lead = off / kBytes;
    if (t < lead || t + 2 * kPer > vocab) return some_logits<DT>(row, t, vocab);
    const uint4* p = reinterpret_cast<const uint4*>(row - off) + t / kPer;
    return off == 0 ? *p : shifted(p[0], p[1], off);
}

// A thread's vectors of the chunk from token `first` on.
template <int DT, int V>
__device__ __forceinline__ void load_chunk(uint4 (&vec)[V], const char* row, int32_t first, int32_t vocab) {
    constexpr int kPer = DT == MF_DT_F32 ? 4 : 8, kBytes = 16 / kPer;
    const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15u);
    const int32_t lead = off / kBytes, mine = first + static_cast<int>(threadIdx.x) * kPer;
    if (first < lead || first + kThreads * V * kPer + kPer > vocab) {  // the row's beginning, where it is not aligned, and its end
#pragma unroll
        for (int v = 0; v < V; ++v) vec[v] = load_vector<DT>(row, mine + v * (kThreads * kPer), vocab);
    } else {
        const uint4* p = reinterpret_cast<const uint4*>(row - off) + mine / kPer;
        if (off == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) vec[v] = p[v * kThreads];
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) vec[v] = shifted(p[v * kThreads], p[v * kThreads + 1], off);
        }
    }
}

// DT: dtype of the logits; V: 16-byte vectors of a thread and chunk.
template <int DT, int V>
__global__ void __launch_bounds__(kThreads, 4) beam_select_kernel(const SelectArgs a) {
    constexpr int kPer = DT == MF_DT_F32 ? 4 : 8;
    constexpr int kBytes = 16 / kPer;
    constexpr int kChunk = kThreads * V * kPer;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ SelectShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.segments;
    const int32_t segment = blockIdx.x - row * a.segments;
    const int32_t entry = row / a.beams;
    const int64_t list = row * a.segments + segment;
    after_previous();
    let_next_start();
    if (a.ended == nullptr || a.ended[row] == 0) {
        const char* begin = a.logits + row * a.row_stride * kBytes;
        const int32_t first0 = segment * a.chunks * kChunk;
        const int32_t chunks = min(a.chunks, (a.vocab - first0 + kChunk - 1) / kChunk);
        uint4 vec[V], ahead[V];
        load_chunk<DT, V>(ahead, begin, first0, a.vocab);
        // Sums of exp(x - ref), ref a maximum that the thread met: differences of near logits are exact.  It is replaced where a
        // logit exceeds it by kReach, so that what is left of earlier terms (3e-4) makes the factor's error nothing, however often
        // the maximum rises.  The terms of a chunk are added in pairs in float32 (five steps), the chunks in float64: one float32 sum
        // of 256 chunks was 4e-6 off.
        float ref = -INFINITY, of_part[kParts];
        double sum = 0.0;
        const int32_t each = (chunks + kParts - 1) / kParts;  // chunks of a part
#pragma unroll
        for (int part = 0; part < kParts; ++part) {
            of_part[part] = -INFINITY;
#pragma unroll 1
            for (int32_t c = part * each; c < min(chunks, (part + 1) * each); ++c) {
#pragma unroll
                for (int v = 0; v < V; ++v) vec[v] = ahead[v];
                if (c + 1 < chunks) load_chunk<DT, V>(ahead, begin, first0 + (c + 1) * kChunk, a.vocab);
                float top = -INFINITY;
#pragma unroll
                for (int v = 0; v < V; ++v) top = fmaxf(top, largest<DT>(vec[v]));
                of_part[part] = fmaxf(of_part[part], top);
                if (top > ref + kReach) {
                    sum *= static_cast<double>(exp2_fast((ref - top) * kLog2e));  // the first time it is 0 times 0
                    ref = top;
                }
                const float less = ref == -INFINITY ? 0.0f : ref;
                float2 of_vec[V];
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float x[kPer];
                    float2 e[kPer / 2];
                    widen<DT>(vec[v], x);
#pragma unroll
                    for (int i = 0; i < kPer / 2; ++i) {
                        e[i] = mul2(add2(make_float2(x[2 * i], x[2 * i + 1]), make_float2(-less, -less)), make_float2(kLog2e, kLog2e));
                        e[i] = make_float2(exp2_fast(e[i].x), exp2_fast(e[i].y));
                    }
                    of_vec[v] = add2(e[0], e[1]);
                    if constexpr (kPer == 8) of_vec[v] = add2(of_vec[v], add2(e[2], e[3]));
                }
#pragma unroll
                for (int d = 1; d < V; d *= 2)
#pragma unroll
                    for (int v = 0; v + d < V; v += 2 * d) of_vec[v] = add2(of_vec[v], of_vec[v + d]);
                sum += static_cast<double>(of_vec[0].x + of_vec[0].y);
            }
        }
        // sums of a warp and of the segment in float64
        float most = of_part[0], all = ref;
#pragma unroll
        for (int part = 1; part < kParts; ++part) most = fmaxf(most, of_part[part]);
#pragma unroll
        for (int d = 16; d; d >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
        double of_warp = ref == -INFINITY ? sum : sum * static_cast<double>(exp2_fast((ref - all) * kLog2e));
#pragma unroll
        for (int d = 16; d; d >>= 1) of_warp += __shfl_xor_sync(0xffffffffu, of_warp, d);
        if (lane == 0) {
            sh.warp_max[warp] = all;
            sh.warp_sum[warp] = of_warp;
        }
        auto& picked = sh.chunk.picked;
        if (tid == 0) picked.count = 0;
        // the threads' parts with the n_out largest maxima, and the least of those; more parts where maxima are equal
        float bound = bound_of(most, a.n_out, sh.chunk.bound);
        if (warp == 0) {
            const float m = lane < kThreads / 32 ? sh.warp_max[lane] : -INFINITY;
            double s = lane < kThreads / 32 ? sh.warp_sum[lane] : 0.0;
            float top = m;
#pragma unroll
            for (int d = 4; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            if (m != -INFINITY) s *= static_cast<double>(exp2_fast((m - top) * kLog2e));
#pragma unroll
            for (int d = 4; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            if (lane == 0) {
                a.part_max[list] = top;
                a.part_sum[list] = s;
            }
        }
        auto keep = [&](float x, int32_t i) {
            const int at = atomicAdd(&picked.count, 1);
            if (at < kPicked) {
                picked.value[at] = x;
                picked.index[at] = i;
            }
        };
#pragma unroll
        for (int part = 0; part < kParts; ++part)
            if (of_part[part] >= bound && of_part[part] > -INFINITY) keep(of_part[part], part * kThreads + tid);
        __syncthreads();
        const int parts = picked.count;
        if (parts <= kPicked) {
            for (int x = tid; x < parts; x += kThreads) {
                const float v = picked.value[x];
                const int32_t i = picked.index[x];
                if (picked.rank(v, i, parts) == a.n_out - 1) sh.chunk.bound.value = v;
                sh.chunk.part[x] = i;
            }
            __syncthreads();
            if (parts >= a.n_out) bound = sh.chunk.bound.value;
            if (tid == 0) picked.count = 0;
            __syncthreads();
            // their logits again
            const int32_t vectors = each * V;
#pragma unroll 2
            for (int32_t x = tid; x < parts * vectors; x += kThreads) {
                const int32_t j = x / parts, part = sh.chunk.part[x - j * parts];
                if (part / kThreads * each * V + j >= chunks * V) continue;
                const int32_t t = first0 + ((part / kThreads * vectors + j) * kThreads + part % kThreads) * kPer;
                const uint4 again = load_vector<DT>(begin, t, a.vocab);
                const float top = largest<DT>(again);
                if (!(top >= bound && top > -INFINITY)) continue;
                float v[kPer];
                widen<DT>(again, v);
#pragma unroll
                for (int i = 0; i < kPer; ++i)
                    if (v[i] >= bound && v[i] > -INFINITY) keep(v[i], t + i);
            }
            __syncthreads();
        }
        const int n = picked.count;
        float2* to = a.lists + list * a.n_out;
        if (n <= kPicked) {
            for (int x = tid; x < n; x += kThreads) {
                const float v = picked.value[x];
                const int32_t i = picked.index[x];
                const int rank = picked.rank(v, i, n);
                if (rank < a.n_out) to[rank] = make_float2(v, __int_as_float(i));
            }
            for (int j = n + tid; j < a.n_out; j += kThreads) to[j] = make_float2(-INFINITY, 0.0f);
        } else {
            // mostly equal logits: one after the other, each the first behind the one before
            float last_v = INFINITY;
            int32_t last_i = -1;
#pragma unroll 1
            for (int j = 0; j < a.n_out; ++j) {
                float best = -INFINITY;
                int32_t best_i = 0x7fffffff;
                for (int32_t x = 0; x < chunks * V; ++x) {
                    const int32_t t = first0 + (x * kThreads + tid) * kPer;
                    float v[kPer];
                    widen<DT>(load_vector<DT>(begin, t, a.vocab), v);
#pragma unroll
                    for (int i = 0; i < kPer; ++i)
                        if (in_front(last_v, last_i, v[i], t + i) && in_front(v[i], t + i, best, best_i)) {
                            best = v[i];
                            best_i = t + i;
                        }
                }
                first_of_all(best, best_i, sh.chunk.best);
                last_v = best;
                last_i = best_i;
                if (tid == 0) to[j] = make_float2(best, __int_as_float(best_i));
            }
        }
        __syncthreads();
    }
    if (tid == 0) {
        int32_t old;
        const int32_t parts = a.beams * a.segments;
        asm volatile("atom.acq_rel.gpu.global.add.s32 %0, [%1], 1;" : "=r"(old) : "l"(a.tickets + entry) : "memory");
        sh.last = old == parts - 1;
        if (sh.last) a.tickets[entry] = 0;
    }
    __syncthreads();
    if (sh.last) merge_lists(a, entry, sh, reinterpret_cast<double*>(smem));
}

struct SelectKernel {
    void (*fn)(SelectArgs);
    int chunk;
};
template <int DT>
SelectKernel select_kernel(bool small) {
    constexpr int per = DT == MF_DT_F32 ? 4 : 8;
    if (small) return {beam_select_kernel<DT, 8 / per>, kThreads * 8};
    return {beam_select_kernel<DT, 4>, kThreads * 4 * per};
}
SelectKernel pick(int dtype, bool small) {
    return dtype == MF_DT_F32 ? select_kernel<MF_DT_F32>(small) : dtype == MF_DT_BF16 ? select_kernel<MF_DT_BF16>(small)
                                                                                     : select_kernel<MF_DT_F16>(small);
}

// How a batch of `rows` rows is cut: the kernel, and the chunks of a segment.
struct Cuts {
    SelectKernel kernel;
    int32_t chunks, segments;
};
Cuts cuts_of(int64_t rows, int32_t vocab, int dtype, int sms) {
    // Small chunks where large ones would not give every SM two; else segments of as many as leave every SM kCtas.
    Cuts c{pick(dtype, false), 1, 1};
    int64_t chunks = (vocab + c.kernel.chunk - 1) / c.kernel.chunk;
    if (rows * chunks <= 2 * sms) {
        c.kernel = pick(dtype, true);
        chunks = (vocab + c.kernel.chunk - 1) / c.kernel.chunk;
    } else {
        const int64_t want = (kCtas * sms + rows - 1) / rows;  // segments of a row
        c.chunks = static_cast<int32_t>(want >= chunks ? 1 : (chunks + want - 1) / want);
    }
    c.segments = static_cast<int32_t>((chunks + c.chunks - 1) / c.chunks);
    c.chunks = static_cast<int32_t>((chunks + c.segments - 1) / c.segments);
    return c;
}

}  // namespace
}  // namespace mf

using namespace mf;

struct mf_beam_select_s {
    mf_beam_select_config config;
    SelectArgs args;
    void* workspace;
    int device, sm_count;
    int64_t lists;  // that the workspace has room for
};

extern "C" int mf_beam_select_create(const mf_beam_select_config* config, mf_beam_select* handle) {
    MF_ENTER();
    if (!config || !handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_create: NULL argument");
    *handle = nullptr;
    const mf_beam_select_config& c = *config;
    if (!is_float_store_dtype(c.dtype))
        return fail(MF_ERR_DTYPE_UNSUPPORTED, "mf_beam_select_create: logits of dtype %d (F32, BF16 and F16 are supported)", c.dtype);
    if (c.vocab <= 0 || c.vocab > (1 << 30) || c.beams <= 0 || c.beams > kMostBeams || static_cast<int64_t>(c.beams) * c.vocab > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_beam_select_create: %d beams (1 to %d) of %d tokens (1 to 2^30), below 2^31 together", c.beams,
                    kMostBeams, c.vocab);
    if (c.n_out <= 0 || c.n_out > kMostOut)
        return fail(MF_ERR_SHAPE_INVALID, "mf_beam_select_create: %d results (1 to %d)", c.n_out, kMostOut);
    if (c.max_batch <= 0 || static_cast<int64_t>(c.max_batch) * c.beams > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_beam_select_create: batch of up to %d", c.max_batch);
    if (c.row_stride < c.vocab)
        return fail(MF_ERR_SHAPE_MISMATCH, "mf_beam_select_create: row stride %lld is below the row's %d logits",
                    (long long)c.row_stride, c.vocab);
    if (c.end_token < -1 || c.end_token >= c.vocab)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_create: end token %d of %d", c.end_token, c.vocab);
    // The workspace holds what the segments of any batch leave.  More rows mean fewer segments of each, and no more than
    // `most` in all until a row is one.
    const int sms = state().sm_count;
    const int64_t rows = static_cast<int64_t>(c.max_batch) * c.beams, least = c.beams;
    const int64_t large = (c.vocab + kThreads * 16 - 1) / (kThreads * 16);
    const int64_t most = 64ll * sms + 4 * least * large;
    const int64_t lists = rows > most ? rows : most < 4 * rows * large ? most : 4 * rows * large;
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t at_max = up(static_cast<size_t>(c.max_batch) * 4), at_sum = at_max + up(lists * 4);
    const size_t at_lists = at_sum + up(lists * 8), bytes = at_lists + static_cast<size_t>(lists) * c.n_out * 8;
    mf_beam_select_s* h = new (std::nothrow) mf_beam_select_s{};
    if (!h) return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_beam_select_create: out of host memory");
    cudaError_t err = cudaMalloc(&h->workspace, bytes);
    if (err != cudaSuccess) {
        cudaGetLastError();
        delete h;
        if (err == cudaErrorMemoryAllocation)
            return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_beam_select_create: %zu bytes: out of device memory", bytes);
        return cuda_fail(err, "mf_beam_select_create: cudaMalloc");
    }
    err = cudaMemset(h->workspace, 0, at_max);
    if (err == cudaSuccess) err = cudaStreamSynchronize(nullptr);  // streams that do not wait for the default one may run it
    if (err != cudaSuccess) {
        cudaFree(h->workspace);
        delete h;
        return cuda_fail(err, "mf_beam_select_create: cudaMemset");
    }
    char* w = static_cast<char*>(h->workspace);
    h->config = c;
    h->device = state().device;
    h->sm_count = sms;
    h->lists = lists;
    SelectArgs& a = h->args;
    a.row_stride = c.row_stride;
    a.vocab = c.vocab;
    a.beams = c.beams;
    a.n_out = c.n_out;
    a.end_token = c.end_token;
    a.tickets = reinterpret_cast<int32_t*>(w);
    a.part_max = reinterpret_cast<float*>(w + at_max);
    a.part_sum = reinterpret_cast<double*>(w + at_sum);
    a.lists = reinterpret_cast<float2*>(w + at_lists);
    *handle = h;
    return MF_OK;
}

extern "C" int mf_beam_select_run(mf_beam_select handle, const void* logits, const float* scores, const int32_t* ended,
                                  int32_t batch, float* scores_after, int32_t* tokens, int32_t* parents, int32_t* ended_after,
                                  mf_stream stream) {
    MF_ENTER();
    if (!handle) return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_run: handle is NULL");
    if (handle->device != state().device)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_run: the handle belongs to device %d", handle->device);
    const mf_beam_select_config& c = handle->config;
    if (batch < 0 || batch > c.max_batch)
        return fail(MF_ERR_SHAPE_INVALID, "mf_beam_select_run: batch of %d (0 to %d)", batch, c.max_batch);
    if (batch == 0) return MF_OK;
    if (!logits || !scores || !scores_after || !tokens || !parents)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_run: NULL buffer");
    if (reinterpret_cast<uintptr_t>(logits) % (c.dtype == MF_DT_F32 ? 4 : 2))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_beam_select_run: logits are not aligned to their dtype");
    if (ended && c.end_token < 0)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_run: ended beams need an end token");
    if (scores_after == scores || (ended && ended_after == ended))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_beam_select_run: outputs may not be the inputs (scores_after, ended_after)");
    const int64_t rows = static_cast<int64_t>(batch) * c.beams;
    const Cuts cuts = cuts_of(rows, c.vocab, c.dtype, handle->sm_count);
    if (rows * cuts.segments > handle->lists) return fail(MF_ERR_ALLOCATOR_EXHAUSTED, "mf_beam_select_run: workspace of %lld lists", (long long)handle->lists);
    SelectArgs a = handle->args;
    a.logits = static_cast<const char*>(logits);
    a.scores = scores;
    a.ended = ended;
    a.segments = cuts.segments;
    a.chunks = cuts.chunks;
    a.scores_after = scores_after;
    a.tokens = tokens;
    a.parents = parents;
    a.ended_after = ended_after;
    const cudaError_t err = launch_overlapped(cuts.kernel.fn, dim3(static_cast<unsigned>(rows * a.segments)), kThreads, c.beams * 8,
                                              static_cast<cudaStream_t>(stream), a);
    if (err != cudaSuccess) return cuda_fail(err, "mf_beam_select_run");
    return MF_OK;
}

extern "C" int mf_beam_select_destroy(mf_beam_select handle) {
    if (!handle) return MF_OK;
    const cudaError_t err = free_workspace(handle->device, handle->workspace);
    delete handle;
    if (err != cudaSuccess) return cuda_fail(err, "mf_beam_select_destroy");
    return MF_OK;
}
