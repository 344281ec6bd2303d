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

#include "attn_device.h"
#include "rope_ops.h"
#include "zk_common.h"

using namespace zk;

namespace {

constexpr int kThreads = 256;
constexpr int kMaxDim = 1024;  // of the generic kernel's LDS row

template <typename T> struct Elt;
template <> struct Elt<float> {
    static constexpr int V = 4;  // of a 16-byte vector
    static __device__ __forceinline__ void unpack(u32x4 v, float *x) {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
    }
    static __device__ __forceinline__ u32x4 pack(const float *x) {
        return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
    }
    static __device__ __forceinline__ float squares(u32x4 v) {
        float s = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) s = fmaf(__uint_as_float(v[e]), __uint_as_float(v[e]), s);
        return s;
    }
    static __device__ __forceinline__ float get(const float *p) { return *p; }
    static __device__ __forceinline__ void put(float *p, float x) { *p = x; }
};
template <> struct Elt<uint16_t> {  // bf16 bits
    static constexpr int V = 8;
    static __device__ __forceinline__ void unpack(u32x4 v, float *x) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = bf16lo(v[i]);
            x[2 * i + 1] = bf16hi(v[i]);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float *x) {
        return u32x4{bf16x2_rne(x[0], x[1]), bf16x2_rne(x[2], x[3]), bf16x2_rne(x[4], x[5]), bf16x2_rne(x[6], x[7])};
    }
    static __device__ __forceinline__ float squares(u32x4 v) {  // exact products, f32 sums
        typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
        float s = 0.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = v[i];
            s = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_t, w), __builtin_bit_cast(bf16x2_t, w), s, false);
        }
        return s;
    }
    static __device__ __forceinline__ float get(const uint16_t *p) { return __uint_as_float((uint32_t)*p << 16); }
    static __device__ __forceinline__ void put(uint16_t *p, float x) { *p = (uint16_t)f32_to_bf16_bits(x); }
};

// A vector of the element type T at p: one access at its own alignment (nontemporal
// where NT), or accesses of T for operands off it (OFF).
template <typename T, bool OFF, bool NT>
__device__ __forceinline__ u32x4 load_vec(const T *p) {
    if constexpr (OFF) {
        u32x4 v;
        __builtin_memcpy(&v, p, 16);
        return v;
    } else if constexpr (NT) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p));
    } else {
        return *reinterpret_cast<const u32x4 *>(p);
    }
}
template <typename T, bool OFF>
__device__ __forceinline__ void store_vec(T *p, u32x4 v) {
    if constexpr (OFF) __builtin_memcpy(p, &v, 16);
    else __builtin_nontemporal_store(v, reinterpret_cast<u32x4 *>(p));
}

__device__ __forceinline__ void put_pool(void *pool, int dt, size_t at, float x, float inv) {
    if (dt == ZK_BF16) ((uint16_t *)pool)[at] = (uint16_t)f32_to_bf16_bits(x);
    else if (dt == ZK_F32) ((float *)pool)[at] = x;
    else ((uint8_t *)pool)[at] = (uint8_t)(e4m3x4(x * inv, 0.f, 0.f, 0.f) & 0xffu);
}
// V values to element `at` of a pool of type `dt`, inv: 1 / scale of an fp8 pool.
template <int V, bool OFF>
__device__ __forceinline__ void store_pool(void *pool, int dt, size_t at, const float *x, float inv) {
    if constexpr (OFF) {
#pragma unroll
        for (int e = 0; e < V; ++e) put_pool(pool, dt, at + e, x[e], inv);
    } else if (dt == ZK_BF16) {
        if constexpr (V == 8) {
            __builtin_nontemporal_store(Elt<uint16_t>::pack(x), reinterpret_cast<u32x4 *>((uint16_t *)pool + at));
        } else {
            const u32x2 w = {bf16x2_rne(x[0], x[1]), bf16x2_rne(x[2], x[3])};
            *reinterpret_cast<u32x2 *>((uint16_t *)pool + at) = w;
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

// Row index in the pools of a slot's token (of head 0; heads are block_size
// rows apart), or -1.
__device__ __forceinline__ int64_t pool_row(const RopeArgs &a, int64_t slot) {
    if (slot < 0 || slot >= a.num_slots) return -1;
    const int64_t blk = slot / a.block_size;
    return blk * a.num_kv_heads * a.block_size + (slot - blk * a.block_size);
}

// Sum over aligned groups of `lanes` lanes, in every lane of a group: within 16
// by the VALU's lane permutations (pairs, pairs of pairs, then mirrored halves,
// whose lanes agree by then).
__device__ __forceinline__ float lane_sum(float x, int lanes) {
    if (lanes > 1) x += dpp<0xb1>(x);   // lane ^ 1
    if (lanes > 2) x += dpp<0x4e>(x);   // lane ^ 2
    if (lanes > 4) x += dpp<0x141>(x);  // mirrored in 8
    if (lanes > 8) x += dpp<0x140>(x);  // mirrored in 16
    if (lanes > 16) x += xor16(x);
    if (lanes > 32) x += xor32(x);
    return x;
}

// One workgroup per token (gridDim.y of them share its heads when tokens are
// few or heads many); `lanes` lanes (a power of two) hold one head, V values in
// one 16-byte vector each, NP heads a lane, all loaded before any is used.  A
// lane writes what it read, so outputs may be the inputs.
//
// 32768 tokens, 32 + 2 x 8 heads of 128 bf16 (810 MB): 133 us, 6.1 TB/s (a copy
// reaches 6.7).  Between HBM and the VALU (busy 104 us of it), so what a head
// needs is kept small: cosines and sines times the weights once a token, the
// norm's factor applied to the rotated value, sums of squares by dot products of
// packed pairs, partners exchanged packed, V copied (before: 187 us, and 233 with
// plain loads and stores).  And its waves must be many (83 registers, five a
// SIMD): workgroups that walk the tokens and load the next one ahead hold 180-200
// registers, two waves a SIMD, and took 178-217 us.
//
// Sums and products are written out as they are to be rounded (fmaf), so that a row's
// result is the same in every variant, whatever the call's other operands are: the
// fused call's K is bit for bit the separate calls'.  OFF: operands off a vector's
// alignment.
template <typename T, int NP, bool INTER, bool OFF>
__global__ void __launch_bounds__(kThreads) qk_norm_rope_kernel(RopeArgs a) {
    constexpr int V = Elt<T>::V, TV = INTER ? V / 2 : V;  // cosines of a lane
    // read only: scalar loads, apart from the vector loads' order
    typedef const __attribute__((address_space(4))) int32_t *cint_t;
    typedef const __attribute__((address_space(4))) int64_t *clong_t;
    const int D = a.head_dim, half = a.rot_dim / 2;
    const int lanes = a.lanes, l = threadIdx.x & (lanes - 1), d0 = l * V;
    const int groups = (int)blockDim.x / lanes, step = groups * gridDim.y;
    const int hg = blockIdx.y * groups + threadIdx.x / lanes;  // this lane's heads: hg + j * step
    const bool live = d0 < D, pool = a.k_pool != nullptr;
    const int heads = a.num_heads + (pool ? 2 : 1) * a.num_kv_heads;
    const bool rot = a.rot_dim > 0, part = a.rot_dim < D, rotated = live && d0 < a.rot_dim;
    const bool second = !INTER && d0 >= half;  // holds the y_b of its pairs
    const int away = !rotated || INTER ? 0 : second ? -(half / V) : half / V;  // the partner's lane
    const int partner = ((int)threadIdx.x + away) & 63;
    const int at_table = !rotated ? 0 : INTER ? d0 / 2 : second ? d0 - half : d0;

    // weights of this lane's dimensions and (rotate-half) its partner's, packed
    u32x4 wq, wk, uq, uk;
    {
        float one[V];
#pragma unroll
        for (int e = 0; e < V; ++e) one[e] = 1.0f;
        wq = wk = uq = uk = Elt<T>::pack(one);
        if (live && a.q_weight) {
            wq = load_vec<T, OFF, false>((const T *)a.q_weight + d0);
            uq = load_vec<T, OFF, false>((const T *)a.q_weight + d0 + away * V);
        }
        if (live && a.k_weight) {
            wk = load_vec<T, OFF, false>((const T *)a.k_weight + d0);
            uk = load_vec<T, OFF, false>((const T *)a.k_weight + d0 + away * V);
        }
    }
    // Workgroups go to the 8 XCDs in turn: of each 128 tokens an XCD takes 16 in a row,
    // whose pieces of a page follow each other (32768 tokens 135.4 us in order, 133.6)
    const int bx = blockIdx.x, t = (bx | 127) < (int)gridDim.x ? (bx & ~127) | (bx & 7) << 4 | (bx >> 3 & 15) : bx;
    u32x4 raw[NP];                      // this lane's values of its heads
    bool has_q = false, has_k = false;  // whether query or key heads are among them
#pragma unroll
    for (int j = 0; j < NP; ++j) {
        const int h = hg + j * step, kh = h - a.num_heads, vh = kh - a.num_kv_heads;
        // (a lane without a head loads the row's start, not used: no branch around a load)
        const bool q_row = kh < 0 || h >= heads || !live;
        const int64_t stride = q_row ? a.q_stride : vh < 0 ? a.k_stride : a.v_stride;
        const T *p = q_row ? (const T *)a.q : vh < 0 ? (const T *)a.k : (const T *)a.v;
        if (live && h < heads) p += (size_t)(kh < 0 ? h : vh < 0 ? kh : vh) * D + d0;
        if constexpr (OFF) raw[j] = load_vec<T, true, true>(p + t * stride);
        else raw[j] = load_vec<T, false, true>((const T *)((const char *)p + (uint64_t)(uint32_t)t * (uint32_t)(sizeof(T) * stride)));
        has_q = has_q || kh < 0;
        has_k = has_k || (kh >= 0 && vh < 0);
    }
    const int64_t pos = rot ? ((cint_t)a.positions)[t] : 0;
    const bool zero = rot && (pos < 0 || pos >= a.max_positions);
    f32x4 cs[V / 4], sn[V / 4];  // cosines and sines of this lane's pairs
    if (rot) {
        const float *row = a.rope + (zero ? 0 : (size_t)pos * a.rot_dim) + at_table;
        if constexpr (OFF) {
#pragma unroll
            for (int e = 0; e < TV; ++e) {
                cs[e / 4][e % 4] = row[e];
                sn[e / 4][e % 4] = row[half + e];
            }
        } else if constexpr (TV >= 4) {
#pragma unroll
            for (int e = 0; e < TV / 4; ++e) {
                cs[e] = *reinterpret_cast<const f32x4 *>(row + 4 * e);
                sn[e] = *reinterpret_cast<const f32x4 *>(row + half + 4 * e);
            }
        } else {
            const f32x2 cv = *reinterpret_cast<const f32x2 *>(row), sv = *reinterpret_cast<const f32x2 *>(row + half);
            cs[0] = f32x4{cv[0], cv[1], 0.f, 0.f};
            sn[0] = f32x4{sv[0], sv[1], 0.f, 0.f};
        }
    }
    // cosines times this lane's weights, sines times those of what they meet (and its sign)
    struct Turn {
        float c[V], s[V];
    };
    auto make = [&](u32x4 w_, u32x4 u_, Turn &m) {
        float w[V], u[V];
        Elt<T>::unpack(w_, w);
        Elt<T>::unpack(u_, u);
#pragma unroll
        for (int e = 0; e < V; ++e) {
            const int i = INTER ? e / 2 : e;
            const bool minus = INTER ? !(e & 1) : !second;
            const float c = rotated ? cs[i / 4][i % 4] : 1.0f, s = rotated ? sn[i / 4][i % 4] : 0.0f;
            m.c[e] = c * w[e];
            m.s[e] = (minus ? -s : s) * (INTER ? w[e ^ 1] : u[e]);
        }
    };
    // y = (x * c + its partner * s) * the norm's factor
    auto turn = [&](u32x4 v, const Turn &m, bool norm, float *y) {
        float x[V];
        Elt<T>::unpack(v, x);
        float inv = 1.0f;
        if (norm) {
            const float ss = Elt<T>::squares(v);
            inv = rsqrtf(fmaf(lane_sum(live ? ss : 0.0f, lanes), a.inv_dim, a.eps));
        }
        if (!rot) {
#pragma unroll
            for (int e = 0; e < V; ++e) y[e] = x[e] * m.c[e] * inv;
            return;
        }
        float p[V];
        if constexpr (INTER) {
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = x[e ^ 1];
        } else {
            u32x4 other;
#pragma unroll
            for (int i = 0; i < 4; ++i) other[i] = (uint32_t)__shfl((int)v[i], partner);
            Elt<T>::unpack(other, p);
        }
        if (part)  // behind rot_dim an infinity times the sine of 0 must not count
#pragma unroll
            for (int e = 0; e < V; ++e) p[e] = rotated ? p[e] : 0.0f;
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = fmaf(x[e], m.c[e], p[e] * m.s[e]) * inv;
    };
    const int64_t prow = pool ? pool_row(a, ((clong_t)a.slots)[t]) : 0;
    auto to_pool = [&](bool is_v, int hd, const float *y) {
        if (prow < 0) return;
        float f = 1.0f;
        if (a.cache_dtype == ZK_FP8_E4M3)
            f = 1.0f / (is_v ? a.v_scales : a.k_scales)[(size_t)((cint_t)a.token_row)[t] * a.num_kv_heads + hd];
        store_pool<V, OFF>(is_v ? a.v_pool : a.k_pool, a.cache_dtype, ((size_t)prow + (size_t)hd * a.block_size) * D + d0, y, f);
    };
    // queries, keys, values: a wave skips what none of its lanes holds
    if (has_q) {
        Turn m;
        make(wq, uq, m);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int h = hg + j * step;
            if (h >= a.num_heads) continue;
            float y[V];
            turn(raw[j], m, a.q_weight != nullptr, y);
            u32x4 w = Elt<T>::pack(y);
            if (zero) w = u32x4{0u, 0u, 0u, 0u};
            if (live) store_vec<T, OFF>((T *)a.q_out + t * a.q_out_stride + (size_t)h * D + d0, w);
        }
    }
    if (has_k) {
        Turn m;
        make(wk, uk, m);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int kh = hg + j * step - a.num_heads;
            if (kh < 0 || kh >= a.num_kv_heads) continue;
            float y[V];
            turn(raw[j], m, a.k_weight != nullptr, y);
            if (zero)
#pragma unroll
                for (int e = 0; e < V; ++e) y[e] = 0.0f;
            if (!live) continue;
            if (pool) to_pool(false, kh, y);
            else store_vec<T, OFF>((T *)a.k_out + t * a.k_out_stride + (size_t)kh * D + d0, Elt<T>::pack(y));
        }
    }
    if (pool)
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int vh = hg + j * step - a.num_heads - a.num_kv_heads;
            if (vh < 0 || vh >= a.num_kv_heads || !live) continue;
            float y[V];
            Elt<T>::unpack(raw[j], y);
            to_pool(true, vh, y);
        }
}

// Head sizes and rotations that are not whole vectors, up to kMaxDim: one wave per
// (token, head), the row in LDS.
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
    const int64_t prow = pool && !is_q ? pool_row(a, a.slots[t]) : 0;
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

// vec: rows are whole vectors (by the shape alone); off: some operand is off their
// alignment, or its rows are too far apart for 32-bit steps.
template <typename T>
void launch(const RopeArgs &a, bool vec, bool off, int heads, hipStream_t s) {
    if (!vec) {
        qk_norm_rope_generic_kernel<T><<<dim3((unsigned)a.num_tokens, heads), 64, 0, s>>>(a);
        return;
    }
    // What a wave does once a token is shared by its heads, so a token gets as few
    // waves as four passes over them allow (8000 tokens of 20 + 2 x 4 heads of 96: 26 us
    // with four waves a token, 22 with two).
    int threads = kThreads;
    while (threads > 64 && heads * a.lanes <= threads / 2 * 4) threads /= 2;
    // Few tokens: the heads of a token over several workgroups, down to one
    // pass of threads / lanes heads each; many heads: at most five passes (8000 tokens of
    // 64 + 2 x 8 heads: 61 us as two workgroups of three, 57; six passes of f32 62.4 as
    // two of three, 63.2 as one).
    const int passes = (heads * a.lanes + threads - 1) / threads;
    if (off) {  // one head a lane
        const dim3 grid((unsigned)a.num_tokens, passes);
        (a.interleaved ? qk_norm_rope_kernel<T, 1, true, true> : qk_norm_rope_kernel<T, 1, false, true>)<<<grid, threads, 0, s>>>(a);
        return;
    }
    const int64_t fill = 2048 / std::max<int64_t>(1, a.num_tokens);
    const int y = std::max((passes + 4) / 5, (int)std::max<int64_t>(1, std::min<int64_t>(passes, fill)));
    const int np = (passes + y - 1) / y;
    const dim3 grid((unsigned)a.num_tokens, y);
    auto go = [&](auto rotate_half, auto inter) { (a.interleaved ? inter : rotate_half)<<<grid, threads, 0, s>>>(a); };
    if (np <= 1) go(qk_norm_rope_kernel<T, 1, false, false>, qk_norm_rope_kernel<T, 1, true, false>);
    else if (np <= 2) go(qk_norm_rope_kernel<T, 2, false, false>, qk_norm_rope_kernel<T, 2, true, false>);
    else if (np <= 3) go(qk_norm_rope_kernel<T, 3, false, false>, qk_norm_rope_kernel<T, 3, true, false>);
    else if (np <= 4) go(qk_norm_rope_kernel<T, 4, false, false>, qk_norm_rope_kernel<T, 4, true, false>);
    else go(qk_norm_rope_kernel<T, 5, false, false>, qk_norm_rope_kernel<T, 5, true, false>);
}

}  // namespace

namespace {

void default_strides(RopeArgs &a) {
    const int64_t qw = (int64_t)a.num_heads * a.head_dim, kw = (int64_t)a.num_kv_heads * a.head_dim;
    if (a.q_stride == 0) a.q_stride = qw;
    if (a.k_stride == 0) a.k_stride = kw;
    if (a.v_stride == 0) a.v_stride = kw;
    if (a.q_out_stride == 0) a.q_out_stride = qw;
    if (a.k_out_stride == 0) a.k_out_stride = kw;
}

}  // namespace

int zk::check_qk_norm_rope(const RopeArgs &in, bool by_cache) {
    RopeArgs a = in;
    if (a.dtype != ZK_F32 && a.dtype != ZK_BF16) return bad("dtype must be f32 or bf16");
    if (a.num_tokens < 0 || a.num_tokens > 0xffffff || a.num_heads <= 0 || a.num_kv_heads <= 0 || a.head_dim <= 0 ||
        (int64_t)a.num_heads + 2 * (int64_t)a.num_kv_heads > 65535)
        return bad("bad shape");
    if (a.head_dim > kMaxDim) return bad("head_dim above 1024");
    if (a.rot_dim < 0 || a.rot_dim > a.head_dim || a.rot_dim % 2) return bad("rot_dim must be even and at most head_dim");
    const int64_t qw = (int64_t)a.num_heads * a.head_dim, kw = (int64_t)a.num_kv_heads * a.head_dim;
    const bool pool = a.k_pool || a.v_pool;
    default_strides(a);
    if (a.q_stride < qw || a.k_stride < kw || a.q_out_stride < qw || (pool && a.v_stride < kw) ||
        (!pool && a.k_out_stride < kw))
        return bad("token stride below the row's width");
    if (pool) {
        if (!valid_dtype(a.cache_dtype)) return bad("unsupported cache dtype");
        if (a.block_size <= 0 || a.num_blocks <= 0) return bad("bad pool shape");
        const bool fp8 = a.cache_dtype == ZK_FP8_E4M3;
        if (!by_cache && fp8 && (!a.k_scales || !a.v_scales || !a.token_row))
            return bad("fp8 pool needs scales and token_row");
        if (!fp8 && (a.k_scales || a.v_scales || a.token_row)) return bad("scales given for a non-fp8 pool");
    }
    if (a.num_tokens == 0) return ZK_OK;
    if (!a.q || !a.k || !a.q_out || (pool ? !a.v || !a.k_pool || !a.v_pool || (!by_cache && !a.slots) : !a.k_out) ||
        (a.rot_dim && ((!by_cache && !a.positions) || !a.rope)))
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
    return ZK_OK;
}

int zk::qk_norm_rope(const RopeArgs &in, hipStream_t s) {
    if (int rc = check_qk_norm_rope(in, false)) return rc;
    if (in.num_tokens == 0) return ZK_OK;
    RopeArgs a = in;
    default_strides(a);
    const bool pool = a.k_pool != nullptr;
    if (pool) a.num_slots = a.num_blocks * a.block_size;
    const int e = elt_size(a.dtype);
    const int V = 16 / e, D = a.head_dim, half = a.rot_dim / 2;
    auto mult = [&](int64_t stride) { return stride % V == 0; };
    auto al = [](const void *p) { return ((uintptr_t)p & 15u) == 0; };
    const bool vec = D % V == 0 && D / V <= 64 && (a.interleaved ? a.rot_dim % V == 0 : half % V == 0);
    bool on = mult(a.q_stride) && mult(a.k_stride) && mult(a.q_out_stride) && al(a.q) && al(a.k) && al(a.q_out) &&
              al(a.q_weight) && al(a.k_weight) && (!a.rot_dim || al(a.rope));
    if (pool) on = on && mult(a.v_stride) && al(a.v) && al(a.k_pool) && al(a.v_pool);
    else on = on && mult(a.k_out_stride) && al(a.k_out);
    on = on && std::max({a.q_stride, a.k_stride, pool ? a.v_stride : 0}) * e < (1ll << 32);  // (32-bit steps)
    int lanes = 1;
    while (lanes * V < D) lanes *= 2;
    a.lanes = lanes;
    a.inv_dim = 1.0f / (float)D;
    const int heads = a.num_heads + (pool ? 2 : 1) * a.num_kv_heads;
    KernelTimer timer("qk_norm_rope", s);
    if (a.dtype == ZK_BF16) launch<uint16_t>(a, vec, !on, heads, s);
    else launch<float>(a, vec, !on, heads, s);
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
