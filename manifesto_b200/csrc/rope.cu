// rope.cu -- rotary positions (mf_rope) and the cache write of a step
// (mf_rope_append): queries and keys rotated, keys and values stored in their
// slots, encoded to the cache's dtype.
//
// One kernel serves both: a token is a list of up to three segments of heads
// (queries, keys, values), each with its source, its destination (an array or
// the paged cache) and whether it turns.  A CTA takes a few tokens, makes their
// cosines and sines once in shared memory (float64 product and reduction to a
// fraction of a turn, then float32 cos/sin of it), and then walks the heads'
// units of 2 * VEC elements with all threads.
//
// Bound: HBM, every element read and written once; issue slots are next (212
// instructions per 16 elements, 65% busy; 275 before divisions became
// multiplications and the test for NaN one per vector).  Occupancy hides the
// loads: 40 registers; keeping several heads of a thread in flight in 64 to 80
// registers was slower (48 to 73 us for the 44 below).  For the few tokens of a
// decoding step, the launch.  Measured: 16384 tokens of 32 heads of 128 in BF16
// 43.7 us (0.94 of the copy rate), 32771 tokens of 32/8 heads into an E4M3 cache
// 123 us (0.92), 48 tokens 2.1 us.
#include <cmath>
#include <initializer_list>

#include "mf_divisor.cuh"
#include "mf_launch.cuh"
#include "mf_runtime.h"
#include "mf_vec.cuh"

namespace mf {
namespace {

constexpr int kRopeThreads = 256;
constexpr int kMaxRot = 1024;
constexpr int kRopeTableFloats = 2048;  // cosines and sines of a CTA's tokens: 2 * tokens * rot / 2

struct RopeSegment {
    const void* src;
    void* dst;
    int32_t src_token, src_head;
    int32_t dst_token, dst_head;  // an array's strides; a cache's are in RopeArgs
    const float* scale_inv;
    int32_t heads;
    int32_t first;                // heads in front of this segment
    bool turns, cached;
};

struct RopeArgs {
    RopeSegment seg[3];
    Divisor per_token, units, half;  // units of a token and of a head, rotated pairs
    const float* inv_freq;
    const int32_t* positions;
    const int64_t* slots;
    int64_t cache_slots, page_stride, token_stride, head_stride;
    int32_t* status;
    int32_t tokens, n_seg, heads, head_dim, rot, page_size, tokens_per_cta;
    int32_t interleaved, inverse, compat;
    float magnitude;
};

// N consecutive elements of a 16- or 32-bit dtype.
template <int DT, int N>
__device__ __forceinline__ void load_n(const void* p, int64_t i, float (&v)[N]) {
    const char* at = static_cast<const char*>(p) + i * dtype_bytes(DT);
    if constexpr (N == 1) {
        v[0] = load_as_f32<DT>(at, 0);
    } else {
        constexpr int kWords = N * dtype_bytes(DT) / 4;
        uint32_t w[kWords];
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k) {
                const uint4 x = *reinterpret_cast<const uint4*>(at + 16 * k);
                w[4 * k] = x.x, w[4 * k + 1] = x.y, w[4 * k + 2] = x.z, w[4 * k + 3] = x.w;
            }
        } else {
            const uint2 x = *reinterpret_cast<const uint2*>(at);
            w[0] = x.x, w[1] = x.y;
        }
#pragma unroll
        for (int q = 0; q < N / 4; ++q) {
            float f[4];
            decode4<DT>(w + q * dtype_bytes(DT), f);
#pragma unroll
            for (int k = 0; k < 4; ++k) v[4 * q + k] = f[k];
        }
    }
}

// N elements of v as stored in DT.  A sum of all of them is not a number when
// one of them is not (or when infinities meet): only then does each element
// take the encoder's rule for NaN.
template <int DT, int N>
__device__ __forceinline__ void encode_n(const float (&v)[N], uint32_t* w, int compat) {
    if constexpr (DT == MF_DT_BF16 || DT == MF_DT_F16) {
        float all = v[0];
#pragma unroll
        for (int k = 1; k < N; ++k) all += v[k];
        if (all == all) {
#pragma unroll
            for (int k = 0; k < N; k += 2)
                w[k / 2] = DT == MF_DT_BF16 ? f32x2_to_bf16x2_nonan(v[k], v[k + 1]) : f32x2_to_f16x2_nonan(v[k], v[k + 1]);
            return;
        }
    }
#pragma unroll
    for (int q = 0; q < N / 4; ++q) {
        const float f[4] = {v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
        encode4<DT>(f, w + q * dtype_bytes(DT), compat);
    }
}

template <int DT, int N>
__device__ __forceinline__ void store_n(void* p, int64_t i, const float (&v)[N], int compat) {
    char* at = static_cast<char*>(p) + i * dtype_bytes(DT);
    if constexpr (N == 1) {
        store_code<DT>(at, 0, encode_f32<DT>(v[0], compat));
    } else {
        constexpr int kWords = N * dtype_bytes(DT) / 4;
        uint32_t w[kWords];
        encode_n<DT, N>(v, w, compat);
        if constexpr (kWords % 4 == 0) {
#pragma unroll
            for (int k = 0; k < kWords / 4; ++k)
                *reinterpret_cast<uint4*>(at + 16 * k) = make_uint4(w[4 * k], w[4 * k + 1], w[4 * k + 2], w[4 * k + 3]);
        } else if constexpr (kWords == 2) {
            *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
        } else {
            *reinterpret_cast<uint32_t*>(at) = w[0];
        }
    }
}

// Cosine and sine of position * frequency, times the magnitude.  The product
// in turns is off by 2^-52 of itself at most (1e-7 of a turn at 2^31 turns);
// what is left after whole turns go is exact, and rounded to float32 there: up
// to 2^-26 of a turn, 9e-8 of the pair's length, as cosine and sine are
// themselves (a 16-bit result hides both).
__device__ __forceinline__ float2 turn_of(int32_t position, float inv_freq, float magnitude, bool inverse) {
    constexpr double kInvTwoPi = 0.15915494309189533577;
    double t = static_cast<double>(position) * (static_cast<double>(inv_freq) * kInvTwoPi);
    t -= rint(t);
    float s, c;
    sincospif(2.0f * static_cast<float>(t), &s, &c);
    return make_float2(c * magnitude, (inverse ? -s : s) * magnitude);
}

// IN: source dtype; CACHE: dtype of cached segments; VEC: elements per access.
// A unit is 2 * VEC elements of one head: the two halves of VEC pairs (HALF),
// VEC pairs side by side (INTERLEAVED), or elements that pass through.
template <int IN, int CACHE, int VEC>
__global__ void __launch_bounds__(kRopeThreads) rope_kernel(const RopeArgs a) {
    __shared__ __align__(16) float s_cos[kRopeTableFloats / 2];
    __shared__ __align__(16) float s_sin[kRopeTableFloats / 2];
    const int32_t t0 = static_cast<int32_t>(blockIdx.x * a.tokens_per_cta);
    after_previous();
    let_next_start();
    const int n_tok = min(a.tokens_per_cta, a.tokens - t0);
    const int half = a.rot >> 1;
    for (int i = threadIdx.x; i < n_tok * half; i += kRopeThreads) {
        const int tok = static_cast<uint32_t>(i) / a.half;
        const float2 cs = turn_of(a.positions[t0 + tok], a.inv_freq[i - tok * half], a.magnitude, a.inverse);
        s_cos[i] = cs.x;
        s_sin[i] = cs.y;
    }
    __syncthreads();
    // per head; the last may be one element short (VEC 1)
    const int units = a.units.d, per_token = a.per_token.d;
    const int step = kRopeThreads * gridDim.y;
    for (int i = blockIdx.y * kRopeThreads + threadIdx.x; i < n_tok * per_token; i += step) {
        const int tok = static_cast<uint32_t>(i) / a.per_token, in_tok = i - tok * per_token;
        int h = static_cast<uint32_t>(in_tok) / a.units;
        const int u = in_tok - h * units;
        const RopeSegment& g = a.seg[(a.n_seg > 1 && h >= a.seg[1].first) + (a.n_seg > 2 && h >= a.seg[2].first)];
        h -= g.first;
        const int32_t t = t0 + tok;
        // the two places of the unit
        const int e = u * 2 * VEC;
        const bool turning = g.turns && e < a.rot;
        int ea, eb;
        if (turning && !a.interleaved) {
            ea = u * VEC;
            eb = ea + half;
        } else {
            ea = e;
            eb = e + VEC;
        }
        const bool second = VEC > 1 || eb < a.head_dim;
        const int64_t from = static_cast<int64_t>(t) * g.src_token + static_cast<int64_t>(h) * g.src_head;
        float x[VEC], y[VEC];
        load_n<IN, VEC>(g.src, from + ea, x);
        if (second) load_n<IN, VEC>(g.src, from + eb, y);
        else y[0] = 0.0f;
        if (turning) {
            const float* pc = s_cos + tok * half + u * VEC;
            const float* ps = s_sin + tok * half + u * VEC;
            if (a.interleaved) {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    // pair k of the unit: elements 2k, 2k + 1 of the run x, y
                    float& p = 2 * k < VEC ? x[(2 * k) % VEC] : y[(2 * k) % VEC];
                    float& q = 2 * k + 1 < VEC ? x[(2 * k + 1) % VEC] : y[(2 * k + 1) % VEC];
                    const float c = pc[k], s = ps[k], p0 = p, q0 = q;
                    p = __fmaf_rn(p0, c, -__fmul_rn(q0, s));
                    q = __fmaf_rn(q0, c, __fmul_rn(p0, s));
                }
            } else {
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    const float c = pc[k], s = ps[k], p0 = x[k], q0 = y[k];
                    x[k] = __fmaf_rn(p0, c, -__fmul_rn(q0, s));
                    y[k] = __fmaf_rn(q0, c, __fmul_rn(p0, s));
                }
            }
        }
        if (!g.cached) {
            const int64_t to = static_cast<int64_t>(t) * g.dst_token + static_cast<int64_t>(h) * g.dst_head;
            store_n<IN, VEC>(g.dst, to + ea, x, 0);
            if (second) store_n<IN, VEC>(g.dst, to + eb, y, 0);
            continue;
        }
        if constexpr (CACHE != MF_DT_INVALID) {
            const int64_t slot = a.slots[t];
            if (slot < 0) continue;
            if (slot >= a.cache_slots) {
                atomicExch(a.status, MF_DEVICE_BAD_PAGE);
                continue;
            }
            const int64_t to = slot / a.page_size * a.page_stride + slot % a.page_size * a.token_stride + h * a.head_stride;
            if constexpr (dtype_bytes(CACHE) == 1) {
                if (g.scale_inv) {
                    const float inv = __fdiv_rn(1.0f, g.scale_inv[h]);
#pragma unroll
                    for (int k = 0; k < VEC; ++k) {
                        x[k] = __fmul_rn(x[k], inv);
                        y[k] = __fmul_rn(y[k], inv);
                    }
                }
            }
            store_n<CACHE, VEC>(g.dst, to + ea, x, a.compat);
            if (second) store_n<CACHE, VEC>(g.dst, to + eb, y, a.compat);
        }
    }
}

template <int IN, int CACHE>
cudaError_t launch_rope(const RopeArgs& a, int vec, dim3 grid, cudaStream_t s) {
    if (vec == 8) return launch_overlapped(rope_kernel<IN, CACHE, 8>, grid, kRopeThreads, 0, s, a);
    if (vec == 4) return launch_overlapped(rope_kernel<IN, CACHE, 4>, grid, kRopeThreads, 0, s, a);
    return launch_overlapped(rope_kernel<IN, CACHE, 1>, grid, kRopeThreads, 0, s, a);
}

// Whether accesses of `vec` elements are aligned: base address, both strides.
bool fits_vec(int vec, int bytes, const void* p, int64_t s0, int64_t s1, int64_t s2 = 0) {
    const int access = vec * bytes < 16 ? vec * bytes : 16;
    return reinterpret_cast<uintptr_t>(p) % access == 0 && s0 % vec == 0 && s1 % vec == 0 && s2 % vec == 0;
}

int check_rope(const char* name, const mf_rope_config* c, int64_t tokens) {
    if (!is_float_store_dtype(c->dtype)) return fail(MF_ERR_DTYPE_UNSUPPORTED, "%s: unsupported dtype %d", name, c->dtype);
    if (c->head_dim <= 0) return fail(MF_ERR_SHAPE_INVALID, "%s: head_dim %d must be positive", name, c->head_dim);
    if (c->rot_dim < 0 || c->rot_dim % 2 || c->rot_dim > c->head_dim || c->rot_dim > kMaxRot)
        return fail(MF_ERR_SHAPE_INVALID, "%s: rot_dim %d must be even, at most head_dim %d and at most %d", name, c->rot_dim,
                    c->head_dim, kMaxRot);
    if (c->layout != MF_ROPE_HALF && c->layout != MF_ROPE_INTERLEAVED)
        return fail(MF_ERR_INVALID_ARGUMENT, "%s: unknown layout %d", name, c->layout);
    if (c->rot_dim > 0 && !c->inv_freq) return fail(MF_ERR_INVALID_ARGUMENT, "%s: inv_freq is NULL", name);
    if (tokens < 0 || tokens > 0x7fffffffll)
        return fail(MF_ERR_SHAPE_INVALID, "%s: %lld tokens (0 to 2^31 - 1)", name, (long long)tokens);
    return MF_OK;
}

// Sizes of the launch: several tokens per CTA where there are many (up to 1024
// units: 44 us for 16384 tokens of 32 heads of 128, 47.5 with twice and 46 with
// half as many), several CTAs per token (grid.y) where there are few.
int finish_and_launch(const char* name, RopeArgs& a, const mf_rope_config* c, int cache_dt, int vec, cudaStream_t s) {
    a.inv_freq = c->inv_freq;
    a.head_dim = c->head_dim;
    a.rot = c->rot_dim;
    a.interleaved = c->layout == MF_ROPE_INTERLEAVED;
    a.magnitude = c->magnitude;
    const int per_head = (a.head_dim + 2 * vec - 1) / (2 * vec);
    const int64_t units = static_cast<int64_t>(a.heads) * per_head;
    a.per_token = divisor(static_cast<int32_t>(units));
    a.units = divisor(per_head);
    a.half = divisor(a.rot > 1 ? a.rot / 2 : 1);
    const int sms = state().sm_count;
    const int room = a.rot ? kRopeTableFloats / a.rot : 16;  // tokens whose cosines fit
    int per = 1;
    while (per * 2 <= room && per < 16 && a.tokens / (per * 2) >= 8ll * sms && per * units < 4 * kRopeThreads) per *= 2;
    a.tokens_per_cta = per;
    const int64_t blocks = (static_cast<int64_t>(a.tokens) + per - 1) / per;
    int64_t split = 1;
    if (blocks < sms) {
        split = (units + kRopeThreads - 1) / kRopeThreads;
        if (split > sms / blocks) split = sms / blocks;
        if (split < 1) split = 1;
    }
    const dim3 grid(static_cast<unsigned>(blocks), static_cast<unsigned>(split));
    cudaError_t err;
    switch (c->dtype) {
    case MF_DT_F32:
        if (cache_dt == MF_DT_F32) err = launch_rope<MF_DT_F32, MF_DT_F32>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E4M3) err = launch_rope<MF_DT_F32, MF_DT_F8E4M3>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E5M2) err = launch_rope<MF_DT_F32, MF_DT_F8E5M2>(a, vec, grid, s);
        else err = launch_rope<MF_DT_F32, MF_DT_INVALID>(a, vec, grid, s);
        break;
    case MF_DT_BF16:
        if (cache_dt == MF_DT_BF16) err = launch_rope<MF_DT_BF16, MF_DT_BF16>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E4M3) err = launch_rope<MF_DT_BF16, MF_DT_F8E4M3>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E5M2) err = launch_rope<MF_DT_BF16, MF_DT_F8E5M2>(a, vec, grid, s);
        else err = launch_rope<MF_DT_BF16, MF_DT_INVALID>(a, vec, grid, s);
        break;
    default:
        if (cache_dt == MF_DT_F16) err = launch_rope<MF_DT_F16, MF_DT_F16>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E4M3) err = launch_rope<MF_DT_F16, MF_DT_F8E4M3>(a, vec, grid, s);
        else if (cache_dt == MF_DT_F8E5M2) err = launch_rope<MF_DT_F16, MF_DT_F8E5M2>(a, vec, grid, s);
        else err = launch_rope<MF_DT_F16, MF_DT_INVALID>(a, vec, grid, s);
    }
    if (err != cudaSuccess) return cuda_fail(err, name);
    return MF_OK;
}

bool fits_int(std::initializer_list<int64_t> strides) {
    for (int64_t s : strides)
        if (s < -0x7fffffffll || s > 0x7fffffffll) return false;
    return true;
}

// The widest access that the head's split allows (both parts whole units).
bool dims_fit(const mf_rope_config* c, int vec) {
    return c->rot_dim % (2 * vec) == 0 && (c->head_dim - c->rot_dim) % (2 * vec) == 0;
}

}  // namespace
}  // namespace mf

using namespace mf;

extern "C" int mf_rope(const mf_rope_config* config, int inverse, const void* src, int64_t src_token_stride,
                       int64_t src_head_stride, void* dst, int64_t dst_token_stride, int64_t dst_head_stride,
                       const int32_t* positions, int64_t tokens, int32_t heads, mf_stream stream) {
    MF_ENTER();
    if (!config) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope: config is NULL");
    if (int rc = check_rope("mf_rope", config, tokens)) return rc;
    if (heads < 0) return fail(MF_ERR_SHAPE_INVALID, "mf_rope: negative head count %d", heads);
    if (tokens == 0 || heads == 0) return MF_OK;
    if (!src || !dst || !positions) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope: NULL buffer");
    if (static_cast<int64_t>(heads) * config->head_dim > (1 << 26))
        return fail(MF_ERR_SHAPE_INVALID, "mf_rope: %d heads of %d elements", heads, config->head_dim);
    if (src == dst && (src_token_stride != dst_token_stride || src_head_stride != dst_head_stride))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_rope: in place needs equal strides");
    if (!fits_int({src_token_stride, src_head_stride, dst_token_stride, dst_head_stride}))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_rope: a stride is over 2^31 - 1 elements");
    const int bytes = dtype_bytes(config->dtype);
    int vec = 1;
    for (int v : {8, 4})
        if (vec == 1 && dims_fit(config, v) && fits_vec(v, bytes, src, src_token_stride, src_head_stride) &&
            fits_vec(v, bytes, dst, dst_token_stride, dst_head_stride))
            vec = v;
    RopeArgs a{};
    auto stride = [](int64_t s) { return static_cast<int32_t>(s); };
    a.seg[0] = RopeSegment{src, dst, stride(src_token_stride), stride(src_head_stride), stride(dst_token_stride),
                           stride(dst_head_stride), nullptr, heads, 0, true, false};
    a.n_seg = 1;
    a.heads = heads;
    a.positions = positions;
    a.tokens = static_cast<int32_t>(tokens);
    a.inverse = inverse != 0;
    return finish_and_launch("mf_rope", a, config, MF_DT_INVALID, vec, static_cast<cudaStream_t>(stream));
}

extern "C" int mf_rope_append(const mf_rope_append_config* config, const void* q, const void* k, const void* v,
                              void* q_out, void* k_cache, void* v_cache, const int32_t* positions, const int64_t* slots,
                              int64_t tokens, mf_stream stream) {
    MF_ENTER();
    if (!config) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_append: config is NULL");
    const mf_rope_append_config& c = *config;
    const mf_cache_layout& cache = c.cache;
    if (int rc = check_rope("mf_rope_append", &c.rope, tokens)) return rc;
    if (!is_fp8(cache.dtype) && cache.dtype != c.rope.dtype)
        return fail(MF_ERR_DTYPE_MISMATCH, "mf_rope_append: cache dtype %d is neither FP8 nor the inputs' %d", cache.dtype,
                    c.rope.dtype);
    if (cache.head_dim != c.rope.head_dim)
        return fail(MF_ERR_SHAPE_MISMATCH, "mf_rope_append: the cache's head_dim %d is not %d", cache.head_dim,
                    c.rope.head_dim);
    if (cache.kv_heads <= 0 || cache.page_size <= 0 || cache.n_pages < 0 || c.q_heads < 0)
        return fail(MF_ERR_SHAPE_INVALID, "mf_rope_append: %d query and %d key heads, %lld pages of %d", c.q_heads,
                    cache.kv_heads, (long long)cache.n_pages, cache.page_size);
    if (c.compat != MF_COMPAT_REFERENCE && c.compat != MF_COMPAT_OCP)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_append: unknown compat mode %d", c.compat);
    const int64_t heads = static_cast<int64_t>(c.q_heads) + 2ll * cache.kv_heads;
    if (heads * cache.head_dim > (1 << 26))
        return fail(MF_ERR_SHAPE_INVALID, "mf_rope_append: %lld heads of %d elements", (long long)heads, cache.head_dim);
    if (tokens == 0) return MF_OK;
    if (!k || !v || !k_cache || !v_cache || !positions || !slots || (c.q_heads > 0 && (!q || !q_out)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_append: NULL buffer");
    if (q == q_out && c.q_heads > 0 && (c.q_token_stride != c.out_token_stride || c.q_head_stride != c.out_head_stride))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_rope_append: in place needs equal strides");
    if (!fits_int({c.q_token_stride, c.q_head_stride, c.k_token_stride, c.k_head_stride, c.v_token_stride, c.v_head_stride,
                   c.out_token_stride, c.out_head_stride}))
        return fail(MF_ERR_LAYOUT_UNSUPPORTED, "mf_rope_append: a stride is over 2^31 - 1 elements");
    const int bytes = dtype_bytes(c.rope.dtype), code = dtype_bytes(cache.dtype);
    int vec = 1;
    for (int w : {8, 4})
        if (vec == 1 && dims_fit(&c.rope, w) && cache.head_dim % (2 * w) == 0 &&
            (c.q_heads == 0 || (fits_vec(w, bytes, q, c.q_token_stride, c.q_head_stride) &&
                                fits_vec(w, bytes, q_out, c.out_token_stride, c.out_head_stride))) &&
            fits_vec(w, bytes, k, c.k_token_stride, c.k_head_stride) &&
            fits_vec(w, bytes, v, c.v_token_stride, c.v_head_stride) &&
            fits_vec(w, code, k_cache, cache.page_stride, cache.token_stride, cache.head_stride) &&
            fits_vec(w, code, v_cache, cache.page_stride, cache.token_stride, cache.head_stride))
            vec = w;
    RopeArgs a{};
    auto stride = [](int64_t s) { return static_cast<int32_t>(s); };
    a.seg[0] = RopeSegment{q, q_out, stride(c.q_token_stride), stride(c.q_head_stride), stride(c.out_token_stride),
                           stride(c.out_head_stride), nullptr, c.q_heads, 0, true, false};
    a.seg[1] = RopeSegment{k, k_cache, stride(c.k_token_stride), stride(c.k_head_stride), 0, 0, c.k_scale_inv,
                           cache.kv_heads, c.q_heads, true, true};
    a.seg[2] = RopeSegment{v, v_cache, stride(c.v_token_stride), stride(c.v_head_stride), 0, 0, c.v_scale_inv,
                           cache.kv_heads, c.q_heads + cache.kv_heads, false, true};
    a.n_seg = 3;
    a.heads = static_cast<int32_t>(heads);
    a.positions = positions;
    a.slots = slots;
    a.tokens = static_cast<int32_t>(tokens);
    a.cache_slots = cache.n_pages * cache.page_size;
    a.page_size = cache.page_size;
    a.page_stride = cache.page_stride;
    a.token_stride = cache.token_stride;
    a.head_stride = cache.head_stride;
    a.compat = c.compat;
    a.status = sticky_status_ptr();
    if (!a.status) return fail(MF_ERR_CUDA, "mf_rope_append: sticky status word unavailable");
    return finish_and_launch("mf_rope_append", a, &c.rope, cache.dtype, vec, static_cast<cudaStream_t>(stream));
}

extern "C" int mf_rope_frequencies(int32_t rot_dim, double base, int scaling, double factor, double original_length,
                                   double low_turns, double high_turns, float* inv_freq) {
    if (rot_dim < 0 || rot_dim % 2 || rot_dim > kMaxRot)
        return fail(MF_ERR_SHAPE_INVALID, "mf_rope_frequencies: rot_dim %d must be even and at most %d", rot_dim, kMaxRot);
    if (scaling < MF_ROPE_NONE || scaling > MF_ROPE_BANDS)
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_frequencies: unknown scaling %d", scaling);
    if (!(base > 0.0) || (scaling != MF_ROPE_NONE && !(factor > 0.0)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_frequencies: base %g and factor %g must be positive", base, factor);
    if (scaling == MF_ROPE_BANDS && (!(original_length > 0.0) || !(high_turns > low_turns)))
        return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_frequencies: original length %g, turns from %g to %g", original_length,
                    low_turns, high_turns);
    if (rot_dim > 0 && !inv_freq) return fail(MF_ERR_INVALID_ARGUMENT, "mf_rope_frequencies: inv_freq is NULL");
    if (scaling == MF_ROPE_BASE && rot_dim > 2) base *= std::pow(factor, double(rot_dim) / (rot_dim - 2));
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == MF_ROPE_LINEAR) {
            f /= factor;
        } else if (scaling == MF_ROPE_BANDS) {
            const double turns = original_length * f / (2.0 * 3.14159265358979323846);
            double ramp = (turns - low_turns) / (high_turns - low_turns);
            ramp = ramp < 0.0 ? 0.0 : ramp > 1.0 ? 1.0 : ramp;
            f = (1.0 - ramp) * f / factor + ramp * f;
        }
        inv_freq[i] = static_cast<float>(f);
    }
    return MF_OK;
}
