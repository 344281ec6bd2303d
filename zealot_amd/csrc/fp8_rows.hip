// fp8_rows.hip -- rows in 8 bits for the 8-bit projections: RMSNorm (with the
// residual add before it) and SiLU(gate) * up whose results are written as
// e4m3 values and one f32 scale a row.
//
// A row y is held as s = max(max |y| / 448, 2^-126) and q = e4m3(y / s), to
// nearest even (448: the largest e4m3 value; 2^-126 keeps 1 / s finite and a
// row of zeros zero).  A row with a NaN has NaN for its scale and all values.
//   norm: t = x (+ residual, rounded to the tensors' type and written),
//         y = t * rsqrt(mean(t^2) + eps) * w
//   SiLU: y = g / (1 + exp(-g)) * u
// y itself is f32 and rounded once, to e4m3: the 16-bit row that the unfused
// sequence writes and reads again never exists.  The reference has neither
// (its projections are f32, src/attention/cublas.rs:72-114).
//
// Both are bound by HBM (32768 rows of 4096 with a residual 158 us, 6.0 TB/s; SiLU of
// 8192 rows of 14336 102 us, 5.8 TB/s), a few rows by latency: a row is read once
// into registers, its sum of squares and its largest |t w| (which is the largest
// |y| up to the factor of the row) go through one reduction, and it is written from
// the registers.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "zk_common.h"

using namespace zk;

namespace {

constexpr float kTop = 448.0f;        // e4m3's largest value
constexpr float kLeast = 0x1p-126f;   // smallest scale

struct RowArgs {
    const void *x, *other;  // norm: x and the residual (or null); SiLU: gate and up
    const void *weight;     // norm
    uint8_t *q;
    float *scales;
    void *sum_out;          // norm with a residual
    const int64_t *rows;    // norm: the input row of each output row, or null
    int64_t in_rows;        // rows of x; one outside them is a row of zeros
    int64_t x_stride, other_stride, num_rows;
    int dim;
    float eps;
};

// What a thread loads at once: VEC values, as they are in memory, at their own
// alignment (one instruction all the same).
template <typename T, int VEC> struct __attribute__((packed, aligned(sizeof(T)))) Raw { T v; };
template <> struct __attribute__((packed, aligned(4))) Raw<float, 4> { f32x4 v; };
template <> struct __attribute__((packed, aligned(2))) Raw<uint16_t, 8> { u32x4 v; };

template <typename T, int VEC>
__device__ __forceinline__ Raw<T, VEC> load(const T *p) { return *reinterpret_cast<const Raw<T, VEC> *>(p); }
__device__ __forceinline__ void values(const Raw<float, 1> &r, float (&v)[1]) { v[0] = r.v; }
__device__ __forceinline__ void values(const Raw<float, 4> &r, float (&v)[4]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = r.v[e];
}
__device__ __forceinline__ void values(const Raw<uint16_t, 1> &r, float (&v)[1]) { v[0] = __uint_as_float((uint32_t)r.v << 16); }
__device__ __forceinline__ void values(const Raw<uint16_t, 8> &r, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v[2 * e] = bf16lo(r.v[e]);
        v[2 * e + 1] = bf16hi(r.v[e]);
    }
}
// v rounded to the tensor's type (to nearest even, the machine's conversion)
__device__ __forceinline__ Raw<float, 1> rounded(const float (&v)[1], float) { return {v[0]}; }
__device__ __forceinline__ Raw<float, 4> rounded(const float (&v)[4], float) { return {f32x4{v[0], v[1], v[2], v[3]}}; }
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2_t));
}
__device__ __forceinline__ Raw<uint16_t, 1> rounded(const float (&v)[1], uint16_t) { return {(uint16_t)bf16_pair(v[0], v[0])}; }
__device__ __forceinline__ Raw<uint16_t, 8> rounded(const float (&v)[8], uint16_t) {
    return {u32x4{bf16_pair(v[0], v[1]), bf16_pair(v[2], v[3]), bf16_pair(v[4], v[5]), bf16_pair(v[6], v[7])}};
}
typedef uint32_t __attribute__((aligned(1))) u32_any;
typedef u32x2 __attribute__((aligned(1))) u32x2_any;
// (FINITE: every value is, and at most 448 before its rounding)
template <bool FINITE, int VEC>
__device__ __forceinline__ void store_q(uint8_t *p, const float (&v)[VEC]) {
    auto four = [](float a, float b, float c, float d) { return FINITE ? e4m3x4_in_range(a, b, c, d) : e4m3x4(a, b, c, d); };
    if constexpr (VEC == 1) {
        *p = (uint8_t)four(v[0], 0.f, 0.f, 0.f);
    } else if constexpr (VEC == 4) {
        *reinterpret_cast<u32_any *>(p) = four(v[0], v[1], v[2], v[3]);
    } else {
        *reinterpret_cast<u32x2_any *>(p) = u32x2{four(v[0], v[1], v[2], v[3]), four(v[4], v[5], v[6], v[7])};
    }
}
// g / (1 + exp(-g)) with the machine's exp2 and reciprocal, as g (1 / (1 / 4 + exp(-g) / 4)
// / 4): the machine's reciprocal gives no numbers below 2^-126, exp(-g) may be up to 2^128.
// (Below -87.3 the last quarter loses two bits; a quarter of g would lose them of gates
// near 2^-149.)  0 below -88.72, where exp(-g) is no f32.  The exponent -g log2(e) - 2 is off by 2^-25 of
// its first term at most (the constant's) and 2^-24 of the whole (its rounding): 2^-24 (2.2 |g| + 2),
// and the value by log(2) of that where g is far below zero, by half and less of it above;
// beside it exp2 and the reciprocal 2 steps of 2^-24 each, the sum and the product one: 6.
// With expf and a division the instructions bind, not memory (8192 rows of 14336 129 us).
__device__ __forceinline__ float silu(float g) {
    const float e = __builtin_amdgcn_exp2f(fmaf(g, -1.44269504088896341f, -2.0f));
    return g * (0.25f * __builtin_amdgcn_rcpf(0.25f + e));
}

// W waves a row, MAXV vectors a thread, R rows a workgroup (more than one where a
// row is one wave's).  Each sum is written by the thread that read its terms, so
// sum_out may be x or residual.  Loads past the row's end repeat its last vector,
// so that none waits for a branch; what they give (in place: the vector or its sum)
// is not used.
template <bool NORM, typename T, int VEC, int MAXV, int W, int R>
__global__ void __launch_bounds__(64 * W * R) fp8_rows_kernel(RowArgs a) {
    static_assert(W == 1 || R == 1, "rows of several waves meet at barriers");
    constexpr int THREADS = 64 * W;
    __shared__ float red_sum[W];
    __shared__ uint32_t red_max[W];
    const int t = R > 1 ? threadIdx.x & 63 : threadIdx.x;
    const int64_t row = (int64_t)blockIdx.x * R + (R > 1 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) : 0);
    if (R > 1 && row >= a.num_rows) return;
    int64_t in = row;
    if (NORM && a.rows) {
        in = a.rows[row];
        if ((uint64_t)in >= (uint64_t)a.in_rows) {  // no such row: zeros
            for (int i = t; i < a.dim; i += THREADS) {
                a.q[(size_t)row * a.dim + i] = 0;
                if (a.other) ((T *)a.sum_out)[(size_t)row * a.dim + i] = T(0);
            }
            if (t == 0) a.scales[row] = kLeast;
            return;
        }
    }
    const T *x = (const T *)a.x + (size_t)in * a.x_stride;
    const T *o = a.other ? (const T *)a.other + (size_t)in * a.other_stride : nullptr;
    Raw<T, VEC> rx[MAXV], ro[MAXV], rw[MAXV];
    const int last = a.dim - VEC;
#pragma unroll
    for (int j = 0; j < MAXV; ++j) rx[j] = load<T, VEC>(x + min((j * THREADS + t) * VEC, last));
    if (!NORM || o) {
#pragma unroll
        for (int j = 0; j < MAXV; ++j) ro[j] = load<T, VEC>(o + min((j * THREADS + t) * VEC, last));
    }
    if (NORM) {
#pragma unroll
        for (int j = 0; j < MAXV; ++j) rw[j] = load<T, VEC>((const T *)a.weight + min((j * THREADS + t) * VEC, last));
    }
    float v[MAXV][VEC];
    float ss = 0.0f;
    uint32_t top = 0;  // of |value| as bits: NaN above infinity above the numbers
#pragma unroll
    for (int j = 0; j < MAXV; ++j) {
        const int i = (j * THREADS + t) * VEC;
        values(rx[j], v[j]);
        float other[VEC];
        if (NORM) {
            if (o) {
                values(ro[j], other);
#pragma unroll
                for (int e = 0; e < VEC; ++e) v[j][e] += other[e];
                const Raw<T, VEC> sum = rounded(v[j], T());
                values(sum, v[j]);
                if (i < a.dim) *reinterpret_cast<Raw<T, VEC> *>((T *)a.sum_out + (size_t)row * a.dim + i) = sum;
            }
            float part = 0.0f;
#pragma unroll
            for (int e = 0; e < VEC; ++e) part += v[j][e] * v[j][e];
            ss += i < a.dim ? part : 0.0f;
            values(rw[j], other);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] *= other[e];
        } else {
            values(ro[j], other);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[j][e] = silu(v[j][e]) * other[e];
        }
        uint32_t most = 0;
#pragma unroll
        for (int e = 0; e < VEC; ++e) most = max(most, __float_as_uint(v[j][e]) & 0x7fffffffu);
        top = max(top, i < a.dim ? most : 0u);
    }
#pragma unroll
    for (int k = 32; k > 0; k >>= 1) {
        if (NORM) ss += __shfl_xor(ss, k);
        top = max(top, (uint32_t)__shfl_xor((int)top, k));
    }
    if (W > 1) {
        const int wave = threadIdx.x >> 6;
        if ((threadIdx.x & 63) == 0) {
            red_sum[wave] = ss;
            red_max[wave] = top;
        }
        __syncthreads();
        ss = 0.0f;
#pragma unroll
        for (int k = 0; k < W; ++k) {
            ss += red_sum[k];
            top = max(top, red_max[k]);
        }
    }
    const float inv = NORM ? rsqrtf(ss / (float)a.dim + a.eps) : 1.0f;
    const float most = __uint_as_float(top) * inv / kTop;
    const float s = most < kLeast ? kLeast : most;  // (NaN stays)
    const float r = 1.0f / s;
    if (t == 0) a.scales[row] = s;
    auto write = [&](auto finite) {
        constexpr bool kFinite = decltype(finite)::value;
#pragma unroll
        for (int j = 0; j < MAXV; ++j) {
            const int i = (j * THREADS + t) * VEC;
            if (i < a.dim) {
                float q[VEC];
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float y = NORM ? v[j][e] * inv : v[j][e];
                    q[e] = kFinite ? quotient(y, s, r) : y * r;
                }
                store_q<kFinite>(a.q + (size_t)row * a.dim + i, q);
            }
        }
    };
    // A row whose scale is infinite or NaN (the same over the row) has no quotients to round: NaN, and zeros beside an infinity.
    if (__builtin_amdgcn_readfirstlane(__float_as_uint(s)) < 0x7f800000u) write(std::true_type{});
    else write(std::false_type{});
}

// Waves a row: a wave for short rows, four rows a workgroup (32768 rows of 1024,
// two vectors a thread 43 us, a workgroup a row 51).  Longer rows of the norm take two to four
// vectors a thread (8192 rows of 16384: eight 163 us, four 160, two 164; 32768 of
// 4096: two 158, one 160), SiLU, whose threads compute more between two loads, as few
// as 16 waves allow (8192 of 14336: eight 110, four 109, two 100; 16384 of 4096: two
// 60.5, one 57.7).  Rows that are no whole vectors go value by value: eight a thread
// (8192 of 2001: 31 us, four 36, two 49).
template <bool NORM, typename T, int VEC>
bool launch_vec(const RowArgs &a, hipStream_t s) {
    const int n = (a.dim + VEC - 1) / VEC;
    auto go = [&](auto kernel, int threads, int rows) {
        kernel<<<(unsigned)((a.num_rows + rows - 1) / rows), threads, 0, s>>>(a);
    };
    if (n <= 64) go(fp8_rows_kernel<NORM, T, VEC, 1, 1, 4>, 256, 4);
    else if (n <= 128) go(fp8_rows_kernel<NORM, T, VEC, 2, 1, 4>, 256, 4);
    else if (n <= 256) go(fp8_rows_kernel<NORM, T, VEC, 1, 4, 1>, 256, 1);
    else if constexpr (VEC == 1) {
        if (n <= 512) go(fp8_rows_kernel<NORM, T, VEC, 2, 4, 1>, 256, 1);
        else if (n <= 2048) go(fp8_rows_kernel<NORM, T, VEC, 8, 4, 1>, 256, 1);
        else if (n <= 4096) go(fp8_rows_kernel<NORM, T, VEC, 8, 8, 1>, 512, 1);
        else return false;
    } else if constexpr (NORM) {
        if (n <= 512) go(fp8_rows_kernel<NORM, T, VEC, 2, 4, 1>, 256, 1);
        else if (n <= 1024) go(fp8_rows_kernel<NORM, T, VEC, 2, 8, 1>, 512, 1);
        else if (n <= 2048) go(fp8_rows_kernel<NORM, T, VEC, 4, 8, 1>, 512, 1);
        else if (n <= 4096) go(fp8_rows_kernel<NORM, T, VEC, 4, 16, 1>, 1024, 1);
        else return false;
    } else {
        if (n <= 512) go(fp8_rows_kernel<NORM, T, VEC, 1, 8, 1>, 512, 1);
        else if (n <= 1024) go(fp8_rows_kernel<NORM, T, VEC, 1, 16, 1>, 1024, 1);
        else if (n <= 2048) go(fp8_rows_kernel<NORM, T, VEC, 2, 16, 1>, 1024, 1);
        else if (n <= 4096) go(fp8_rows_kernel<NORM, T, VEC, 4, 16, 1>, 1024, 1);
        else return false;
    }
    return true;
}

template <bool NORM>
int launch(const RowArgs &a, zk_dtype dtype, const char *name, hipStream_t s) {
    const bool vec = a.dim % (dtype == ZK_BF16 ? 8 : 4) == 0;
    bool ok;
    if (dtype == ZK_BF16)
        ok = vec ? launch_vec<NORM, uint16_t, 8>(a, s) : launch_vec<NORM, uint16_t, 1>(a, s);
    else
        ok = vec ? launch_vec<NORM, float, 4>(a, s) : launch_vec<NORM, float, 1>(a, s);
    if (!ok)
        return set_error(ZK_ERR_INVALID_ARGUMENT,
                         std::string("Internal error: ") + name + ": rows of " + std::to_string(a.dim) +
                             " too long (at most 32768 bf16 / 16384 f32 elements in whole vectors of 16 bytes, 4096 otherwise)");
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: ") + name + ": " + hipGetErrorString(e));
    return ZK_OK;
}

struct Span {
    const void *p;
    int64_t bytes;
};
bool meet(const Span &u, const Span &v) {
    const uintptr_t a = (uintptr_t)u.p, b = (uintptr_t)v.p;
    return u.p && v.p && u.bytes > 0 && v.bytes > 0 && a < b + v.bytes && b < a + u.bytes;
}

}  // namespace

extern "C" {

int zk_rms_norm_fp8(const void *x, const void *residual, const void *weight, void *q, float *scales,
                    void *residual_out, const int64_t *rows, int64_t x_rows, int64_t num_rows, int64_t dim, float eps,
                    zk_dtype dtype, void *stream) {
    if (dtype != ZK_F32 && dtype != ZK_BF16)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_rms_norm_fp8: dtype must be f32 or bf16");
    if (num_rows < 0 || x_rows < 0 || dim <= 0 || dim > 32768 || num_rows > 0x7fffffff || x_rows > 0x7fffffff ||
        (!rows && x_rows != num_rows))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_rms_norm_fp8: bad shape");
    if (num_rows == 0) return ZK_OK;
    if (!x || !weight || !q || !scales || (residual && !residual_out))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_rms_norm_fp8: NULL pointer");
    const int64_t e = elt_size(dtype);
    const Span in[] = {{x, x_rows * dim * e}, {residual, x_rows * dim * e}, {weight, dim * e}, {rows, 8 * num_rows}};
    const Span out[] = {{q, num_rows * dim}, {scales, 4 * num_rows}, {residual ? residual_out : nullptr, num_rows * dim * e}};
    for (int i = 0; i < 3; ++i) {
        for (int j = 0; j < 4; ++j)  // (a row's own sum may take its place)
            if (meet(out[i], in[j]) && !(i == 2 && j < 2 && !rows && out[i].p == in[j].p))
                return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_rms_norm_fp8: an output overlaps an input");
        for (int j = 0; j < i; ++j)
            if (meet(out[i], out[j]))
                return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_rms_norm_fp8: outputs overlap");
    }
    RowArgs a{};
    a.x = x;
    a.other = residual;
    a.weight = weight;
    a.q = (uint8_t *)q;
    a.scales = scales;
    a.sum_out = residual ? residual_out : nullptr;
    a.rows = rows;
    a.in_rows = x_rows;
    a.num_rows = num_rows;
    a.x_stride = a.other_stride = dim;
    a.dim = (int)dim;
    a.eps = eps;
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("rms_norm_fp8", s);
    return launch<true>(a, dtype, "zk_rms_norm_fp8", s);
}

int zk_silu_mul_fp8(const void *gate, const void *up, void *q, float *scales, int64_t rows, int64_t cols,
                    int64_t gate_stride, int64_t up_stride, zk_dtype dtype, void *stream) {
    if (dtype != ZK_F32 && dtype != ZK_BF16)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_silu_mul_fp8: dtype must be f32 or bf16");
    if (rows < 0 || cols <= 0 || cols > 32768 || rows > 0x7fffffff)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_silu_mul_fp8: bad shape");
    if (gate_stride == 0) gate_stride = cols;
    if (up_stride == 0) up_stride = cols;
    if (gate_stride < cols || up_stride < cols || gate_stride > (1ll << 31) || up_stride > (1ll << 31))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_silu_mul_fp8: bad row stride");
    if (rows == 0) return ZK_OK;
    if (!gate || !up || !q || !scales)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_silu_mul_fp8: NULL pointer");
    const int64_t e = elt_size(dtype);
    const Span in[] = {{gate, ((rows - 1) * gate_stride + cols) * e}, {up, ((rows - 1) * up_stride + cols) * e}};
    const Span out[] = {{q, rows * cols}, {scales, 4 * rows}};
    if (meet(out[0], in[0]) || meet(out[0], in[1]) || meet(out[1], in[0]) || meet(out[1], in[1]) || meet(out[0], out[1]))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_silu_mul_fp8: an output overlaps another operand");
    RowArgs a{};
    a.x = gate;
    a.other = up;
    a.num_rows = rows;
    a.q = (uint8_t *)q;
    a.scales = scales;
    a.x_stride = gate_stride;
    a.other_stride = up_stride;
    a.dim = (int)cols;
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("silu_mul_fp8", s);
    return launch<false>(a, dtype, "zk_silu_mul_fp8", s);
}

}  // extern "C"
