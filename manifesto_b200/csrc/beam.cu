// beam.cu -- mf_beam_select_*: the best continuations over beams and vocabulary.
//
// For row k (a beam) of a batch entry with logits x and score s, token t scores
//   s + x[t] - L,  L = log sum_t exp x[t],
// and the n largest over all beams and tokens are wanted.  Inside a row the
// order of the scores is that of the logits, so a row is cut into chunks, and a
// chunk gives its n largest logits and its part (maximum, sum of exponentials)
// of L; the last CTA of a batch entry (a ticket) puts the Ls together and
// merges the chunks' lists.  One launch, every logit read once.
//
// Bound: HBM, the logits.  A chunk stays in registers (32 logits a thread), so
// the second look at it is free: the n-th largest of 32 maxima (of 8 threads
// each) is a bound that n logits reach, only threads whose maximum reaches it
// look at their logits again, and the few that do are ranked by counting.
#include <new>

#include "mf_launch.cuh"
#include "mf_runtime.h"
#include "mf_vec.cuh"

namespace mf {
namespace {

constexpr int kThreads = 256;
constexpr int kMostOut = 128;        // results of a batch entry
constexpr int kMostBeams = 1024;     // beams of a batch entry
constexpr int kGroups = 32;          // maxima that bound a list of up to kGroups
constexpr int kPicked = 1024;        // logits of a chunk that may be ranked by counting
constexpr float kLog2e = 1.44269504088896341f;

struct SelectArgs {
    const char* logits;
    const float* scores;
    const int32_t* ended;
    int64_t row_stride;   // elements
    int32_t vocab, beams, n_out, end_token;
    int32_t chunks;       // of a row
    double* part_sum;     // [rows][chunks]
    float* part_max;      // [rows][chunks]
    int32_t* part_n;      // [rows][chunks]: entries of the list
    float2* lists;        // [rows][chunks][n_out]: logit and token (as bits), the largest first
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
__device__ __noinline__ uint4 some_logits(const char* row, int32_t t, int32_t vocab) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = DT == MF_DT_F32 ? 0xff800000u : DT == MF_DT_BF16 ? 0xff80ff80u : 0xfc00fc00u;
    if constexpr (DT == MF_DT_F32) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (t + i < vocab) w[i] = reinterpret_cast<const uint32_t*>(row)[t + i];
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (t + i < vocab)
                w[i / 2] = __byte_perm(w[i / 2], reinterpret_cast<const uint16_t*>(row)[t + i], i & 1 ? 0x5410 : 0x3254);
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
};
struct SelectShared {
    float warp_max[kThreads / 32];
    double warp_sum[kThreads / 32];
    int32_t last;
    union {
        struct {
            Bound<float> bound;
            Picked<float> picked;
        } chunk;
        struct {
            Bound<double> bound;
            Picked<double> picked;
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
__device__ __forceinline__ void first_of_all(T& v, int32_t& i, Picked<T>& sh) {
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

// What the chunks of batch entry `entry` left, put together by one CTA.
__device__ void merge_lists(const SelectArgs& a, int32_t entry, SelectShared& sh, double* base) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int32_t row0 = entry * a.beams;
    for (int32_t k = warp; k < a.beams; k += kThreads / 32) {
        const int64_t row = row0 + k;
        double b = static_cast<double>(a.scores[row]);
        if (a.ended == nullptr || a.ended[row] == 0) {
            float top = -INFINITY;
            for (int32_t c = lane; c < a.chunks; c += 32) top = fmaxf(top, __ldcg(a.part_max + row * a.chunks + c));
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            double sum = 0.0;
            for (int32_t c = lane; c < a.chunks; c += 32) {
                const float m = __ldcg(a.part_max + row * a.chunks + c);
                const double s = __ldcg(a.part_sum + row * a.chunks + c);
                // a chunk of -inf alone has a sum of zero; a NaN stays one
                sum += m == -INFINITY ? s : s * exp(static_cast<double>(m) - static_cast<double>(top));
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
            b -= static_cast<double>(top) + log(sum);
        }
        // a beam without a finite sum, or without a finite score, offers nothing
        if (lane == 0) base[k] = b > -INFINITY && b < INFINITY ? b : -INFINITY;
    }
    __syncthreads();
    const int32_t n_lists = a.beams * a.chunks;
    // entry e of list l; false behind the list's end
    auto get = [&](int32_t l, int32_t e, double& v, int32_t& i) {
        const int32_t k = l / a.chunks;
        const double b = base[k];
        if (b == -INFINITY) return false;
        if (a.ended != nullptr && a.ended[row0 + k] != 0) {
            v = b;
            i = k * a.vocab + a.end_token;
            return e == 0 && l == k * a.chunks;
        }
        const int64_t list = static_cast<int64_t>(row0) * a.chunks + l;
        if (e >= __ldcg(a.part_n + list)) return false;
        const float2 x = __ldcg(a.lists + list * a.n_out + e);
        v = b + static_cast<double>(x.x);
        i = k * a.vocab + __float_as_int(x.y);
        return true;
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
    double mine = -INFINITY, v;
    int32_t i;
    for (int32_t l = tid; l < n_lists; l += kThreads)
        if (get(l, 0, v, i) && v > mine) mine = v;
    const double bound = bound_of(mine, a.n_out, sh.entry.bound);
    auto& picked = sh.entry.picked;
    if (tid == 0) picked.count = 0;
    __syncthreads();
    for (int32_t l = tid; l < n_lists; l += kThreads)
        for (int32_t e = 0; e < a.n_out && get(l, e, v, i) && v >= bound; ++e) {
            const int at = atomicAdd(&picked.count, 1);
            if (at < kPicked) {
                picked.value[at] = v;
                picked.index[at] = i;
            }
        }
    __syncthreads();
    const int n = picked.count;
    if (n <= kPicked) {
        for (int x = tid; x < n; x += kThreads) {
            v = picked.value[x];
            i = picked.index[x];
            int rank = 0;
            for (int o = 0; o < n; ++o) rank += in_front(picked.value[o], picked.index[o], v, i);
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
        for (int32_t l = tid; l < n_lists; l += kThreads)
            for (int32_t e = 0; e < a.n_out && get(l, e, v, i); ++e) {
                if (!in_front(last_v, last_i, v, i)) continue;
                if (in_front(v, i, best, best_i)) {
                    best = v;
                    best_i = i;
                }
                break;  // a list is in order
            }
        first_of_all(best, best_i, picked);
        if (tid == 0) put(j, best, best_i);
        last_v = best;
        last_i = best_i;
    }
}

// DT: dtype of the logits; V: 16-byte vectors of a thread.
template <int DT, int V>
__global__ void __launch_bounds__(kThreads) beam_select_kernel(const SelectArgs a) {
    constexpr int kPer = DT == MF_DT_F32 ? 4 : 8;     // logits of a vector
    constexpr int kBytes = 16 / kPer;
    constexpr int kChunk = kThreads * V * kPer;
    extern __shared__ __align__(16) unsigned char smem[];
    __shared__ SelectShared sh;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t row = blockIdx.x / a.chunks;
    const int32_t chunk = blockIdx.x - row * a.chunks;
    const int32_t entry = row / a.beams;
    const int64_t list = row * a.chunks + chunk;
    after_previous();
    let_next_start();
    if (a.ended == nullptr || a.ended[row] == 0) {
        // A thread's tokens do not depend on where the row begins in memory: equal rows have equal sums, to the bit.
        const char* begin = a.logits + row * a.row_stride * kBytes;
        const uint32_t off = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(begin) & 15u);
        const int32_t lead = off / kBytes, first = chunk * kChunk;
        uint4 vec[V];
        if (off == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int32_t t = first + (v * kThreads + tid) * kPer;
                vec[v] = t + kPer <= a.vocab ? __ldcs(reinterpret_cast<const uint4*>(begin) + t / kPer) : some_logits<DT>(begin, t, a.vocab);
            }
        } else {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const int32_t t = first + (v * kThreads + tid) * kPer;
                if (t >= lead && t - lead + 2 * kPer <= a.vocab) {
                    const uint4* p = reinterpret_cast<const uint4*>(begin + static_cast<int64_t>(t - lead) * kBytes);
                    vec[v] = shifted(p[0], p[1], off);
                } else {
                    vec[v] = some_logits<DT>(begin, t, a.vocab);
                }
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float x[kPer];
            widen<DT>(vec[v], x);
#pragma unroll
            for (int i = 0; i < kPer; ++i) top = fmaxf(top, x[i]);
        }
        // the sum relative to the thread's own maximum: differences of near logits are exact
        const float less = top == -INFINITY ? 0.0f : top;
        float sum = 0.0f;
#pragma unroll
        for (int v = 0; v < V; ++v) {
            float x[kPer];
            widen<DT>(vec[v], x);
#pragma unroll
            for (int i = 0; i < kPer; ++i) sum += exp2_fast((x[i] - less) * kLog2e);
        }
        // sums of a warp and of the chunk in float64
        float all = top;
#pragma unroll
        for (int d = 16; d; d >>= 1) all = fmaxf(all, __shfl_xor_sync(0xffffffffu, all, d));
        double of_warp = top == -INFINITY ? sum : static_cast<double>(sum * exp2_fast((top - all) * kLog2e));
#pragma unroll
        for (int d = 16; d; d >>= 1) of_warp += __shfl_xor_sync(0xffffffffu, of_warp, d);
        if (lane == 0) {
            sh.warp_max[warp] = all;
            sh.warp_sum[warp] = of_warp;
        }
        auto& picked = sh.chunk.picked;
        if (tid == 0) picked.count = 0;
        const float bound = bound_of(top, a.n_out, sh.chunk.bound);
        if (warp == 0) {
            const float m = lane < kThreads / 32 ? sh.warp_max[lane] : -INFINITY;
            double s = lane < kThreads / 32 ? sh.warp_sum[lane] : 0.0;
            float most = m;
#pragma unroll
            for (int d = 4; d; d >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, d));
            if (m != -INFINITY) s *= static_cast<double>(exp2_fast((m - most) * kLog2e));
#pragma unroll
            for (int d = 4; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
            if (lane == 0) {
                a.part_max[list] = most;
                a.part_sum[list] = s;
            }
        }
        if (top >= bound && top > -INFINITY) {
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float x[kPer];
                widen<DT>(vec[v], x);
#pragma unroll
                for (int i = 0; i < kPer; ++i) {
                    if (x[i] >= bound && x[i] > -INFINITY) {
                        const int at = atomicAdd(&picked.count, 1);
                        if (at < kPicked) {
                            picked.value[at] = x[i];
                            picked.index[at] = first + (v * kThreads + tid) * kPer + i;
                        }
                    }
                }
            }
        }
        __syncthreads();
        const int n_picked = picked.count;
        float2* to = a.lists + list * a.n_out;
        if (n_picked <= kPicked) {
            for (int x = tid; x < n_picked; x += kThreads) {
                const float v = picked.value[x];
                const int32_t i = picked.index[x];
                int rank = 0;
                for (int o = 0; o < n_picked; ++o) rank += in_front(picked.value[o], picked.index[o], v, i);
                if (rank < a.n_out) to[rank] = make_float2(v, __int_as_float(i));
            }
            if (tid == 0) a.part_n[list] = min(n_picked, a.n_out);
        } else {
            // a chunk of mostly equal logits: one after the other, each the first behind the one before
            float last_v = INFINITY;
            int32_t last_i = -1;
            int n = 0;
#pragma unroll 1
            for (; n < a.n_out; ++n) {
                float best = -INFINITY;
                int32_t best_i = 0x7fffffff;
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float x[kPer];
                    widen<DT>(vec[v], x);
#pragma unroll
                    for (int i = 0; i < kPer; ++i) {
                        const int32_t t = first + (v * kThreads + tid) * kPer + i;
                        if (in_front(last_v, last_i, x[i], t) && in_front(x[i], t, best, best_i)) {
                            best = x[i];
                            best_i = t;
                        }
                    }
                }
                first_of_all(best, best_i, picked);
                if (best == -INFINITY) break;
                last_v = best;
                last_i = best_i;
                if (tid == 0) to[n] = make_float2(best, __int_as_float(best_i));
            }
            if (tid == 0) a.part_n[list] = n;
        }
        __syncthreads();
    }
    if (tid == 0) {
        int32_t old;
        const int32_t parts = a.beams * a.chunks;
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
    return {beam_select_kernel<DT, 32 / per>, kThreads * 32};
}
SelectKernel pick(int dtype, bool small) {
    return dtype == MF_DT_F32 ? select_kernel<MF_DT_F32>(small) : dtype == MF_DT_BF16 ? select_kernel<MF_DT_BF16>(small)
                                                                                     : select_kernel<MF_DT_F16>(small);
}

int64_t chunks_of(int64_t vocab, int chunk) { return (vocab + chunk - 1) / chunk; }

// Up to how many rows take small chunks: where large ones would not give every SM two.
int64_t small_rows(int64_t large_chunks, int sms) { return 2 * sms / large_chunks; }

}  // namespace
}  // namespace mf

using namespace mf;

struct mf_beam_select_s {
    mf_beam_select_config config;
    SelectArgs args;
    void* workspace;
    int device, sm_count;
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
    // the workspace holds what the chunks of any batch leave; small chunks are for batches that leave SMs idle
    const int sms = state().sm_count;
    const int64_t rows = static_cast<int64_t>(c.max_batch) * c.beams;
    const int64_t large = chunks_of(c.vocab, kThreads * 32), small = chunks_of(c.vocab, kThreads * 8);
    const int64_t few = rows < small_rows(large, sms) ? rows : small_rows(large, sms);
    const int64_t lists = rows * large > few * small ? rows * large : few * small;
    if (lists > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "mf_beam_select_create: a batch of %d x %d x %d logits", c.max_batch, c.beams, c.vocab);
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t at_max = up(static_cast<size_t>(c.max_batch) * 4), at_n = at_max + up(lists * 4), at_sum = at_n + up(lists * 4);
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
    SelectArgs& a = h->args;
    a.row_stride = c.row_stride;
    a.vocab = c.vocab;
    a.beams = c.beams;
    a.n_out = c.n_out;
    a.end_token = c.end_token;
    a.tickets = reinterpret_cast<int32_t*>(w);
    a.part_max = reinterpret_cast<float*>(w + at_max);
    a.part_n = reinterpret_cast<int32_t*>(w + at_n);
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
    const bool small = rows <= small_rows(chunks_of(c.vocab, kThreads * 32), handle->sm_count);
    const SelectKernel kernel = pick(c.dtype, small);
    SelectArgs a = handle->args;
    a.logits = static_cast<const char*>(logits);
    a.scores = scores;
    a.ended = ended;
    a.chunks = static_cast<int32_t>(chunks_of(c.vocab, kernel.chunk));
    a.scores_after = scores_after;
    a.tokens = tokens;
    a.parents = parents;
    a.ended_after = ended_after;
    const cudaError_t err = launch_overlapped(kernel.fn, dim3(static_cast<unsigned>(rows * a.chunks)), kThreads, c.beams * 8,
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
