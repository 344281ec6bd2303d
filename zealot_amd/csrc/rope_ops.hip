// rope_ops.hip -- norms of the query and key heads and the rotary position
// embedding in one pass over a fused projection's output, with or without the
// write of K and V into the pages.
//
// For a head row x of D values at position p, weight w (optional) and a table
// row of R / 2 cosines c and R / 2 sines s:
//   y = x * rsqrt(mean(x^2) + eps) * w          (y = x without a weight)
//   (y_a, y_b) -> (y_a c_i - y_b s_i, y_b c_i + y_a s_i)   for i < R / 2
// with (a, b) = (i, i + R / 2), or (2 i, 2 i + 1) interleaved; dimensions from
// R on keep y.  Everything is computed in f32 from the inputs; a result is
// rounded once, to the type of where it goes (a fused call's K goes to the
// pool's type without the step over the source's).
//
// The reference has neither (its runner applies no rotary embedding,
// src/cuda_runner.rs:373-461); its norm is attention/kernels/rms_norm.cu:4-55.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "rope_ops.h"
#include "zk_common.h"

using namespace zk;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;  // of the generic kernel's LDS row

template <typename T> struct Elt;
template <> struct Elt<float> {
    static constexpr int V = 4;  // of a 16-byte vector
    static __device__ __forceinline__ void load(const float *p, float *x) {
        const f32x4 v = *reinterpret_cast<const f32x4 *>(p);
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = v[e];
    }
    static __device__ __forceinline__ void store(float *p, const float *x) {
        *reinterpret_cast<f32x4 *>(p) = f32x4{x[0], x[1], x[2], x[3]};
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float x) { *p = x; }
};
template <> struct Elt<uint16_t> {  // bf16 bits
    static constexpr int V = 8;
    static __device__ __forceinline__ void load(const uint16_t *p, float *x) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16lo(v[i]);
            x[2 * i + 1] = bf16hi(v[i]);
        }
    }
    static __device__ __forceinline__ void store(uint16_t *p, const float *x) {
        *reinterpret_cast<u32x4 *>(p) = u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                              pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
    }
    static __device__ __forceinline__ float get(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ __forceinline__ void put(uint16_t *p, float x) { *p = (uint16_t)f32_to_bf16_bits(x); }
};

// V values to element `at` of a pool of type `dt`, inv: 1 / scale of an fp8 pool.
template <int V>
__device__ __forceinline__ void store_pool(void *pool, int dt, size_t at, const float *x, float inv) {
    if (dt == ZK_BF16) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j) {
            const u32x2 w = {pack_bf16x2(x[4 * j], x[4 * j + 1]), pack_bf16x2(x[4 * j + 2], x[4 * j + 3])};
            reinterpret_cast<u32x2 *>((uint16_t *)pool + at)[j] = w;
        }
    } else if (dt == ZK_F32) {
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
            reinterpret_cast<f32x4 *>((float *)pool + at)[j] = f32x4{x[4 * j], x[4 * j + 1], x[4 * j + 2], x[4 * j + 3]};
    } else {
#pragma unroll
        for (int j = 0; j < V / 4; ++j)
            reinterpret_cast<uint32_t *>((uint8_t *)pool + at)[j] =
                e4m3x4(x[4 * j] * inv, x[4 * j + 1] * inv, x[4 * j + 2] * inv, x[4 * j + 3] * inv);
    }
}
__device__ __forceinline__ void put_pool(void *pool, int dt, size_t at, float x, float inv) {
    if (dt == ZK_BF16) ((uint16_t *)pool)[at] = (uint16_t)f32_to_bf16_bits(x);
    else if (dt == ZK_F32) ((float *)pool)[at] = x;
    else ((uint8_t *)pool)[at] = (uint8_t)(e4m3x4(x * inv, 0.f, 0.f, 0.f) & 0xffu);
}

// Where a token's K and V rows go: the row index in the pools (of head 0,
// heads are block_size rows apart), or -1.
__device__ __forceinline__ int64_t pool_row(const RopeArgs &a, int64_t t) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) return -1;
    const int64_t blk = slot / a.block_size;
    return blk * a.num_kv_heads * a.block_size + (slot - blk * a.block_size);
}

// One workgroup per token (gridDim.y workgroups when there are few): `lanes`
// lanes (a power of two) hold one head, V values in one 16-byte vector each,
// the cosines, sines and weights of a lane's dimensions stay in registers over
// its heads.  The sum of squares and the partner's half of a rotation cross
// lanes by shuffles; a lane writes what it read, so outputs may be the inputs.
// Bound by HBM.
template <typename T>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(RopeArgs a) {
    constexpr int V = Elt<T>::V;
    const int64_t t = blockIdx.x;
    const int D = a.head_dim, half = a.rot_dim / 2;
    const int lanes = a.lanes, l = threadIdx.x & (lanes - 1), d0 = l * V;
    const int group = threadIdx.x / lanes, groups = kThreads / lanes;
    const bool live = d0 < D;
    const bool pool = a.k_pool != nullptr;
    const int heads = a.num_heads + (pool ? 2 : 1) * a.num_kv_heads;
    const int64_t pos = a.rot_dim ? a.positions[t] : 0;
    const bool zero = a.rot_dim && (pos < 0 || pos >= a.max_positions);
    const int64_t prow = pool ? pool_row(a, t) : 0;
    const bool rotated = live && d0 < a.rot_dim;
    const bool second = !a.interleaved && d0 >= half;  // holds the y_b of its pairs
    const int partner = a.interleaved ? threadIdx.x : second ? threadIdx.x - half / V : threadIdx.x + half / V;
    float c[V], s[V], wq[V], wk[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        c[e] = 1.0f;
        s[e] = 0.0f;
        wq[e] = wk[e] = 1.0f;
    }
    if (rotated && !zero) {
        const float *row = a.rope + (size_t)pos * a.rot_dim;
        if (a.interleaved) {
#pragma unroll
            for (int e = 0; e < V; e += 2) {
                c[e] = c[e + 1] = row[(d0 + e) / 2];
                s[e] = s[e + 1] = row[half + (d0 + e) / 2];
            }
        } else {
            const int i = second ? d0 - half : d0;
#pragma unroll
            for (int e = 0; e < V; e += 4) {
                const f32x4 cv = *reinterpret_cast<const f32x4 *>(row + i + e);
                const f32x4 sv = *reinterpret_cast<const f32x4 *>(row + half + i + e);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    c[e + j] = cv[j];
                    s[e + j] = sv[j];
                }
            }
        }
    }
    if (live && a.q_weight) Elt<T>::load((const T *)a.q_weight + d0, wq);
    if (live && a.k_weight) Elt<T>::load((const T *)a.k_weight + d0, wk);
    const int step = groups * gridDim.y;
    for (int h0 = blockIdx.y * groups; h0 < heads; h0 += step) {
        const int h = h0 + group;
        const bool is_q = h < a.num_heads, is_v = h >= a.num_heads + a.num_kv_heads;
        const int kh = is_v ? h - a.num_heads - a.num_kv_heads : h - a.num_heads;
        const bool on = live && h < heads;
        float x[V];
        if (on) {
            const T *src = is_q   ? (const T *)a.q + t * a.q_stride + (size_t)h * D
                           : is_v ? (const T *)a.v + t * a.v_stride + (size_t)kh * D
                                  : (const T *)a.k + t * a.k_stride + (size_t)kh * D;
            Elt<T>::load(src + d0, x);
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) x[e] = 0.0f;
        }
        float y[V];
        const bool norm = is_q ? a.q_weight != nullptr : a.k_weight != nullptr;
        float inv = 1.0f;
        if (a.q_weight || a.k_weight) {  // (all lanes: the shuffles need their partners)
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < V; ++e) ss += x[e] * x[e];
            for (int o = lanes / 2; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
            inv = rsqrtf(ss / (float)D + a.eps);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = !norm || is_v ? x[e] : x[e] * inv * (is_q ? wq[e] : wk[e]);
        if (a.rot_dim && !is_v) {  // (is_v is the same for a head's lanes)
            float z[V];
            if (a.interleaved) {
#pragma unroll
                for (int e = 0; e < V; e += 2) {
                    z[e] = y[e] * c[e] - y[e + 1] * s[e];
                    z[e + 1] = y[e + 1] * c[e] + y[e] * s[e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float p = __shfl(y[e], partner & 63);
                    z[e] = second ? y[e] * c[e] + p * s[e] : y[e] * c[e] - p * s[e];
                }
            }
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = zero ? 0.0f : rotated ? z[e] : y[e];
        }
        if (!on) continue;
        if (is_q) {
            Elt<T>::store((T *)a.q_out + t * a.q_out_stride + (size_t)h * D + d0, y);
        } else if (!pool) {
            Elt<T>::store((T *)a.k_out + t * a.k_out_stride + (size_t)kh * D + d0, y);
        } else if (prow >= 0) {
            float f = 1.0f;
            if (a.cache_dtype == ZK_FP8_E4M3)
                f = 1.0f / (is_v ? a.v_scales : a.k_scales)[(size_t)a.token_row[t] * a.num_kv_heads + kh];
            const size_t at = ((size_t)prow + (size_t)kh * a.block_size) * D + d0;
            store_pool<V>(is_v ? a.v_pool : a.k_pool, a.cache_dtype, at, y, f);
        }
    }
}

// Any shape and alignment up to kMaxDim: one wave per (token, head), the row
// in LDS.
template <typename T>
__global__ void __launch_bounds__(64) qk_norm_rope_generic_kernel(RopeArgs a) {
    __shared__ float row[kMaxDim];
    const int64_t t = blockIdx.x;
    const int h = blockIdx.y, lane = threadIdx.x, D = a.head_dim, half = a.rot_dim / 2;
    const bool pool = a.k_pool != nullptr;
    const bool is_q = h < a.num_heads, is_v = h >= a.num_heads + a.num_kv_heads;
    const int kh = is_v ? h - a.num_heads - a.num_kv_heads : h - a.num_heads;
    const T *src = is_q   ? (const T *)a.q + t * a.q_stride + (size_t)h * D
                   : is_v ? (const T *)a.v + t * a.v_stride + (size_t)kh * D
                          : (const T *)a.k + t * a.k_stride + (size_t)kh * D;
    const T *w = is_v ? nullptr : (const T *)(is_q ? a.q_weight : a.k_weight);
    float ss = 0.0f;
    for (int i = lane; i < D; i += 64) {
        const float x = Elt<T>::get(src + i);
        row[i] = x;
        ss += x * x;
    }
    for (int o = 32; o > 0; o >>= 1) ss += __shfl_xor(ss, o);
    const float inv = rsqrtf(ss / (float)D + a.eps);
    if (w)
        for (int i = lane; i < D; i += 64) row[i] = row[i] * inv * Elt<T>::get(w + i);
    __syncthreads();
    const int64_t pos = a.rot_dim ? a.positions[t] : 0;
    const bool zero = !is_v && a.rot_dim && (pos < 0 || pos >= a.max_positions);
    const float *cs = a.rope + (zero || is_v ? 0 : (size_t)pos * a.rot_dim);
    const int64_t prow = pool && !is_q ? pool_row(a, t) : 0;
    if (prow < 0) return;
    float f = 1.0f;
    if (pool && !is_q && a.cache_dtype == ZK_FP8_E4M3)
        f = 1.0f / (is_v ? a.v_scales : a.k_scales)[(size_t)a.token_row[t] * a.num_kv_heads + kh];
    for (int i = lane; i < D; i += 64) {
        float y = row[i];
        if (zero) {
            y = 0.0f;
        } else if (!is_v && i < a.rot_dim) {
            const int j = a.interleaved ? i >> 1 : i < half ? i : i - half;
            const bool second = a.interleaved ? (i & 1) != 0 : i >= half;
            const float p = row[a.interleaved ? i ^ 1 : second ? i - half : i + half];
            y = second ? y * cs[j] + p * cs[half + j] : y * cs[j] - p * cs[half + j];
        }
        if (is_q) Elt<T>::put((T *)a.q_out + t * a.q_out_stride + (size_t)h * D + i, y);
        else if (!pool) Elt<T>::put((T *)a.k_out + t * a.k_out_stride + (size_t)kh * D + i, y);
        else
            put_pool(is_v ? a.v_pool : a.k_pool, a.cache_dtype, ((size_t)prow + (size_t)kh * a.block_size) * D + i, y, f);
    }
}

int bad(const char *what) {
    return set_error(ZK_ERR_INVALID_ARGUMENT, std::string("Internal error: zk_qk_norm_rope: ") + what);
}

// Whether rows (t * stride, width values) of two tensors of the same element
// size share memory.  Columns of one fused buffer (equal strides) do not.
bool rows_overlap(const void *a, int64_t a_stride, int64_t a_width, const void *b, int64_t b_stride, int64_t b_width,
                  int64_t rows, int elt) {
    const int64_t pa = (int64_t)(uintptr_t)a, pb = (int64_t)(uintptr_t)b;
    const int64_t ea = pa + ((rows - 1) * a_stride + a_width) * elt, eb = pb + ((rows - 1) * b_stride + b_width) * elt;
    if (ea <= pb || eb <= pa) return false;
    if (a_stride != b_stride || rows == 1) return true;
    const int64_t s = a_stride * elt, d = ((pb - pa) % s + s) % s;
    return d < a_width * elt || d + b_width * elt > s;
}

template <typename T>
void launch(const RopeArgs &a, bool vec, int heads, hipStream_t s) {
    if (vec) {
        // Few tokens: the heads of a token over several workgroups, down to one
        // pass of 256 / lanes heads each.
        const int passes = (heads * a.lanes + kThreads - 1) / kThreads;
        const int y = (int)std::max<int64_t>(1, std::min<int64_t>(passes, 2048 / std::max<int64_t>(1, a.num_tokens)));
        qk_norm_rope_kernel<T><<<dim3((unsigned)a.num_tokens, y), kThreads, 0, s>>>(a);
    } else {
        qk_norm_rope_generic_kernel<T><<<dim3((unsigned)a.num_tokens, heads), 64, 0, s>>>(a);
    }
}

}  // namespace

int zk::qk_norm_rope(const RopeArgs &in, hipStream_t s) {
    RopeArgs a = in;
    if (a.dtype != ZK_F32 && a.dtype != ZK_BF16) return bad("dtype must be f32 or bf16");
    const int64_t qw = (int64_t)a.num_heads * a.head_dim, kw = (int64_t)a.num_kv_heads * a.head_dim;
    if (a.num_tokens < 0 || a.num_tokens > 0xffffff || a.num_heads <= 0 || a.num_kv_heads <= 0 || a.head_dim <= 0 ||
        (int64_t)a.num_heads + 2 * (int64_t)a.num_kv_heads > 65535)
        return bad("bad shape");
    if (a.head_dim > kMaxDim) return bad("head_dim above 1024");
    if (a.rot_dim < 0 || a.rot_dim > a.head_dim || a.rot_dim % 2) return bad("rot_dim must be even and at most head_dim");
    const bool pool = a.k_pool || a.v_pool;
    if (a.q_stride == 0) a.q_stride = qw;
    if (a.k_stride == 0) a.k_stride = kw;
    if (a.v_stride == 0) a.v_stride = kw;
    if (a.q_out_stride == 0) a.q_out_stride = qw;
    if (a.k_out_stride == 0) a.k_out_stride = kw;
    if (a.q_stride < qw || a.k_stride < kw || a.q_out_stride < qw || (pool && a.v_stride < kw) ||
        (!pool && a.k_out_stride < kw))
        return bad("token stride below the row's width");
    if (pool) {
        if (!valid_dtype(a.cache_dtype)) return bad("unsupported cache dtype");
        if (a.block_size <= 0 || a.num_blocks <= 0) return bad("bad pool shape");
        const bool fp8 = a.cache_dtype == ZK_FP8_E4M3;
        if (fp8 && (!a.k_scales || !a.v_scales || !a.token_row)) return bad("fp8 pool needs scales and token_row");
        if (!fp8 && (a.k_scales || a.v_scales || a.token_row)) return bad("scales given for a non-fp8 pool");
        a.num_slots = a.num_blocks * a.block_size;
    }
    if (a.num_tokens == 0) return ZK_OK;
    if (!a.q || !a.k || !a.q_out || (pool ? !a.v || !a.k_pool || !a.v_pool || !a.slots : !a.k_out) ||
        (a.rot_dim && (!a.positions || !a.rope)))
        return bad("NULL pointer");
    if (a.rot_dim && a.max_positions <= 0) return bad("empty position table");
    const int e = elt_size(a.dtype);
    const int64_t T = a.num_tokens;
    auto apart = [&](const void *o, int64_t os, int64_t ow, const void *i, int64_t is, int64_t iw, bool same_ok) {
        return (same_ok && o == i && os == is) || !rows_overlap(o, os, ow, i, is, iw, T, e);
    };
    if (!apart(a.q_out, a.q_out_stride, qw, a.q, a.q_stride, qw, true) ||
        !apart(a.q_out, a.q_out_stride, qw, a.k, a.k_stride, kw, false) ||
        (pool && !apart(a.q_out, a.q_out_stride, qw, a.v, a.v_stride, kw, false)) ||
        (!pool && (!apart(a.k_out, a.k_out_stride, kw, a.k, a.k_stride, kw, true) ||
                   !apart(a.k_out, a.k_out_stride, kw, a.q, a.q_stride, qw, false) ||
                   !apart(a.k_out, a.k_out_stride, kw, a.q_out, a.q_out_stride, qw, false))))
        return bad("an output overlaps another operand (only the input of the same name, in its own layout, may be it)");
    const int V = 16 / e, D = a.head_dim, half = a.rot_dim / 2;
    auto mult = [&](int64_t stride) { return stride % V == 0; };
    auto al = [](const void *p) { return ((uintptr_t)p & 15u) == 0; };
    bool vec = D % V == 0 && D / V <= 64 && (a.interleaved ? a.rot_dim % V == 0 : half % V == 0) && mult(a.q_stride) &&
               mult(a.k_stride) && mult(a.q_out_stride) && al(a.q) && al(a.k) && al(a.q_out) && al(a.q_weight) &&
               al(a.k_weight) && (!a.rot_dim || al(a.rope));
    if (pool) vec = vec && mult(a.v_stride) && al(a.v) && al(a.k_pool) && al(a.v_pool);
    else vec = vec && mult(a.k_out_stride) && al(a.k_out);
    int lanes = 1;
    while (lanes * V < D) lanes *= 2;
    a.lanes = lanes;
    const int heads = a.num_heads + (pool ? 2 : 1) * a.num_kv_heads;
    KernelTimer timer("qk_norm_rope", s);
    if (a.dtype == ZK_BF16) launch<uint16_t>(a, vec, heads, s);
    else launch<float>(a, vec, heads, s);
    if (hipError_t er = hipGetLastError(); er != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_qk_norm_rope: ") + hipGetErrorString(er));
    return ZK_OK;
}

extern "C" {

int zk_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, zk_dtype dtype,
                    int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, const void *q_weight,
                    const void *k_weight, float eps, const int32_t *positions, const float *rope,
                    int64_t max_positions, int rot_dim, int interleaved, void *q_out, int64_t q_out_stride,
                    void *k_out, int64_t k_out_stride, void *stream) {
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.dtype = dtype;
    a.num_tokens = num_tokens;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.positions = positions;
    a.rope = rope;
    a.max_positions = max_positions;
    a.rot_dim = rot_dim;
    a.interleaved = interleaved != 0;
    a.q_out = q_out;
    a.q_out_stride = q_out_stride;
    a.k_out = k_out;
    a.k_out_stride = k_out_stride;
    return zk::qk_norm_rope(a, (hipStream_t)stream);
}

int zk_qk_norm_rope_append(void *k_pool, void *v_pool, zk_dtype cache_dtype, const void *q, int64_t q_stride,
                           const void *k, int64_t k_stride, const void *v, int64_t v_stride, zk_dtype dtype,
                           int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, const void *q_weight,
                           const void *k_weight, float eps, const int32_t *positions, const float *rope,
                           int64_t max_positions, int rot_dim, int interleaved, void *q_out, int64_t q_out_stride,
                           const int64_t *slot_mapping, int block_size, int64_t num_blocks, const float *k_scales,
                           const float *v_scales, const int32_t *token_row, void *stream) {
    if (num_tokens != 0 && (!k_pool || !v_pool)) return bad("NULL pool");
    RopeArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.v_stride = v_stride;
    a.dtype = dtype;
    a.num_tokens = num_tokens;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.q_weight = q_weight;
    a.k_weight = k_weight;
    a.eps = eps;
    a.positions = positions;
    a.rope = rope;
    a.max_positions = max_positions;
    a.rot_dim = rot_dim;
    a.interleaved = interleaved != 0;
    a.q_out = q_out;
    a.q_out_stride = q_out_stride;
    a.k_pool = k_pool;
    a.v_pool = v_pool;
    a.cache_dtype = cache_dtype;
    a.slots = slot_mapping;
    a.block_size = block_size;
    a.num_blocks = num_blocks;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    a.token_row = token_row;
    return zk::qk_norm_rope(a, (hipStream_t)stream);
}

}  // extern "C"
