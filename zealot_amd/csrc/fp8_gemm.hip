// fp8_gemm.hip -- y[m, n] = s_m t_n sum_k q[m, k] W[n, k]: products of rows in
// 8 bits (e4m3 with one scale a row, fp8_rows.hip) with weights in 8 bits (e4m3
// with one scale an output column), on the matrix cores with f32 sums.  No
// counterpart in the reference (its projections are f32 sgemms,
// src/attention/cublas.rs:72-114).
//
// Weights are packed once into the order in which waves take them, zeros
// behind row n and column k:
//   [ceil(n / 64)][4 tiles][ceil(k / 128)][8 units][16 rows][16 bytes]
// unit u holds columns 16 u .. 16 u + 15 of its 128, and row i of tile t of
// group G is weight row 64 G + 16 (i / 4) + 4 t + i % 4.  The 16x16x128 matrix
// instruction takes from lane l 32 values of row l % 16 of either operand
// (units l / 16 and l / 16 + 4 here: any order of k does, as long as both
// operands have it) and leaves D[4 (l / 16) + r][l % 16], r < 4; with weights as
// the first operand lane l ends with rows 64 G + 16 (l / 16) + 4 t + r: over the
// four tiles 16 consecutive columns of y for one row of x.  So a half tile is
// one load of 1 KiB in a row, without LDS or with it, free of bank conflicts,
// and y is written in whole 16-byte pieces.
//
// bf16 results come from the 8-bit instruction without scales (the intrinsic with
// constant zeros; row and column scales are applied to the sums).  It adds eight
// consecutive products at a time, each cut to a multiple of 2^-13 of the largest
// one's power of two (measured, on this card), and those sums in f32: of normal
// values a result is off by 1.5e-5 of itself, against the 2^-9 of its rounding.
// f32 results take the operands as bf16 (exact) to the bf16 instruction, whose
// sums keep all of f32 (6e-8), at half the rate.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "zk_common.h"

using namespace zk;

namespace {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 128;  // k of one matrix instruction
constexpr int kTile = 2048;  // bytes of 16 packed rows of a chunk

struct GemmArgs {
    const uint8_t *x;
    const float *xs;
    const uint8_t *w;
    const float *ws;
    void *y;
    int m, n, k, chunks, tiles;  // tiles: packed 16-row tiles
    int tiles_m, tiles_n;        // of workgroups
};

// what lanes behind column k of x read
__device__ __align__(16) const uint8_t kZeros[16] = {};

__device__ __forceinline__ i32x8 join(const u32x4 &lo, const u32x4 &hi) {
    return i32x8{(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
}
// values 8 q .. 8 q + 7 of an operand as bf16
__device__ __forceinline__ bf16x8 eight(const i32x8 &v, int q) {
    const u32x2 lo = e4m3x4_to_bf16x4((uint32_t)v[2 * q]), hi = e4m3x4_to_bf16x4((uint32_t)v[2 * q + 1]);
    return __builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]});
}
// acc[f][t] += w[f] x[t], one chunk
template <bool F32, int NT, int MT>
__device__ __forceinline__ void multiply(const i32x8 (&w)[NT], const i32x8 (&x)[MT], f32x4 (&acc)[NT][MT]) {
    if constexpr (F32) {
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            bf16x8 xq[MT];
#pragma unroll
            for (int t = 0; t < MT; ++t) xq[t] = eight(x[t], q);
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const bf16x8 wq = eight(w[f], q);
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[f][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wq, xq[t], acc[f][t], 0, 0, 0);
            }
        }
    } else {
#pragma unroll
        for (int f = 0; f < NT; ++f)
#pragma unroll
            for (int t = 0; t < MT; ++t)
                acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[f], x[t], acc[f][t], 0, 0, 0, 0, 0, 0);
    }
}

// The weight row of row i of tile T.
__device__ __forceinline__ int row_of(int T, int i) { return 64 * (T >> 2) + 16 * (i >> 2) + 4 * (T & 3) + (i & 3); }

// y[row, n0 .. n0 + 3] = v * xs * ws
template <bool F32>
__device__ __forceinline__ void store4(const GemmArgs &a, int row, int n0, f32x4 v, float xs) {
    float o[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) o[r] = n0 + r < a.n ? v[r] * xs * a.ws[n0 + r] : 0.0f;
    const size_t at = (size_t)row * a.n + n0;
    if (a.n % 4 == 0) {  // (y is 16-byte aligned)
        if (n0 >= a.n) return;
        if (F32) *reinterpret_cast<f32x4 *>((float *)a.y + at) = f32x4{o[0], o[1], o[2], o[3]};
        else *reinterpret_cast<u32x2 *>((uint16_t *)a.y + at) = u32x2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (n0 + r < a.n) {
                if (F32) ((float *)a.y)[at + r] = o[r];
                else ((uint16_t *)a.y)[at + r] = (uint16_t)f32_to_bf16_bits(o[r]);
            }
    }
}

// ------------------------------------------------------------ few rows of x
// A workgroup owns NT tiles of 16 weight rows and all of k, its KW waves every
// KW-th chunk of it: weights and x come from memory straight into the
// registers of the instruction, U chunks at a time, and the waves' sums meet
// in LDS, in the order of the waves.
template <int NT, int MT, int KW, int U, bool F32>
__global__ void __launch_bounds__(64 * KW) fp8_stream_kernel(GemmArgs a) {
    __shared__ f32x4 sums[KW][NT * MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int T0 = blockIdx.x * NT;
    const uint8_t *wp = a.w + (size_t)T0 * a.chunks * kTile + lane * 16;
    const uint8_t *xp[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) xp[t] = a.x + (size_t)min(16 * t + r16, a.m - 1) * a.k + 16 * g;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int f = 0; f < NT; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < a.chunks; c0 += KW * U) {
        u32x4 wv[U][NT][2], xv[U][MT][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int c = c0 + u * KW;
            if (c < a.chunks) {
#pragma unroll
                for (int f = 0; f < NT; ++f)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        wv[u][f][h] = __builtin_nontemporal_load(
                            reinterpret_cast<const u32x4 *>(wp + ((size_t)f * a.chunks + c) * kTile + 1024 * h));
#pragma unroll
                for (int t = 0; t < MT; ++t)
#pragma unroll
                    for (int h = 0; h < 2; ++h) {
                        const bool in = c * kChunk + 64 * h + 16 * g < a.k;
                        xv[u][t][h] = *reinterpret_cast<const u32x4 *>(in ? xp[t] + c * kChunk + 64 * h : kZeros);
                    }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
#pragma unroll
                    for (int f = 0; f < NT; ++f) wv[u][f][h] = u32x4{0, 0, 0, 0};
#pragma unroll
                    for (int t = 0; t < MT; ++t) xv[u][t][h] = u32x4{0, 0, 0, 0};
                }
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            i32x8 w[NT], x[MT];
#pragma unroll
            for (int f = 0; f < NT; ++f) w[f] = join(wv[u][f][0], wv[u][f][1]);
#pragma unroll
            for (int t = 0; t < MT; ++t) x[t] = join(xv[u][t][0], xv[u][t][1]);
            multiply<F32>(w, x, acc);
        }
    }
#pragma unroll
    for (int f = 0; f < NT; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) sums[wave][f * MT + t][lane] = acc[f][t];
    __syncthreads();
#pragma unroll
    for (int j = wave; j < NT * MT; j += KW) {
        f32x4 v = sums[0][j][lane];
#pragma unroll
        for (int k = 1; k < KW; ++k) v += sums[k][j][lane];
        const int T = T0 + j / MT, row = 16 * (j % MT) + r16;
        if (row < a.m && T < a.tiles) store4<F32>(a, row, row_of(T, 4 * g), v, a.xs[row]);
    }
}

// ------------------------------------------------------------- many rows of x
typedef __attribute__((address_space(3))) void lds_void;
__device__ __forceinline__ void g2l16(const void *g, lds_void *l) { __builtin_amdgcn_global_load_lds(g, l, 16, 0, 0); }
template <int N>
__device__ __forceinline__ void wait_vmcnt() {
    static_assert(N >= 0 && N <= 63, "vmcnt range");
    __builtin_amdgcn_s_waitcnt((N & 15) | (7 << 4) | (15 << 8) | ((N >> 4) << 14));
}
// workgroup barrier without the fences of __syncthreads (those would wait for
// every load in flight); the memory clobber keeps LDS accesses on their side
__device__ __forceinline__ void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

// A workgroup owns 16 MT WM rows of x and 16 NT WN weight rows; chunks of both
// come to LDS by DMA, two stages.  Weights stay in their packed order; a row of
// x has its eight units at u ^ (row % 8), so the eight rows of a DMA are whole
// 128-byte lines and the reads of a unit of 16 rows hit every bank alike.
template <int MT, int NT, int WM, int WN, bool F32>
__global__ void __launch_bounds__(64 * WM * WN) fp8_gemm_kernel(GemmArgs a) {
    constexpr int kWaves = WM * WN;
    constexpr int BM = 16 * MT * WM, BT = NT * WN;  // rows of x, weight tiles
    constexpr int WQ = BT * 2, XQ = BM / 8;         // DMA instructions a chunk
    constexpr int WL = WQ / kWaves, XL = XQ / kWaves;
    static_assert(WQ % kWaves == 0 && XQ % kWaves == 0 && NT % 4 == 0, "split over the waves");
    __shared__ u32x4 lds[2][(BT * kTile + BM * kChunk) / 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    // An XCD takes a run of tiles, eight m-tiles side by side: workgroups that
    // run at once share their rows and weights in its L2.
    const int all = a.tiles_m * a.tiles_n, per = (all + 7) / 8;
    const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || tile >= all) return;
    const int band = tile / (8 * a.tiles_n), high = min(8, a.tiles_m - 8 * band), in = tile - band * 8 * a.tiles_n;
    const int tm = 8 * band + in % high, tn = in / high;
    const int m0 = tm * BM, T0 = tn * BT;

    const uint8_t *wsrc[WL], *xsrc[XL];
    int xcol[XL];
#pragma unroll
    for (int j = 0; j < WL; ++j) {
        const int q = wave * WL + j;
        wsrc[j] = a.w + (size_t)min(T0 + (q >> 1), a.tiles - 1) * a.chunks * kTile + 1024 * (q & 1) + lane * 16;
    }
#pragma unroll
    for (int j = 0; j < XL; ++j) {
        const int r = 8 * (wave * XL + j) + (lane >> 3);
        xcol[j] = 16 * ((lane & 7) ^ (r & 7));
        xsrc[j] = a.x + (size_t)min(m0 + r, a.m - 1) * a.k + xcol[j];
    }
    auto issue = [&](int c) {
        u32x4 *st = lds[c & 1];
#pragma unroll
        for (int j = 0; j < WL; ++j) g2l16(wsrc[j] + (size_t)c * kTile, (lds_void *)(st + 64 * (wave * WL + j)));
#pragma unroll
        for (int j = 0; j < XL; ++j)
            g2l16(c * kChunk + xcol[j] < a.k ? xsrc[j] + c * kChunk : kZeros,
                  (lds_void *)(st + BT * kTile / 16 + 64 * (wave * XL + j)));
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int f = 0; f < NT; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int wm = wave % WM, wn = wave / WM;
    issue(0);
    for (int c = 0; c < a.chunks; ++c) {
        // the chunk is in, everywhere; every wave has left the other stage
        wait_vmcnt<0>();
        wg_barrier();
        const u32x4 *st = lds[c & 1];
        const u32x4 *wl = st + wn * NT * (kTile / 16) + lane;
        const u32x4 *xl = st + BT * kTile / 16 + (wm * MT * 16 + r16) * 8;
        i32x8 wv[NT], xv[MT];
#pragma unroll
        for (int f = 0; f < NT; ++f) wv[f] = join(wl[f * (kTile / 16)], wl[f * (kTile / 16) + 64]);
#pragma unroll
        for (int t = 0; t < MT; ++t)
            xv[t] = join(xl[t * 128 + (g ^ (r16 & 7))], xl[t * 128 + ((g + 4) ^ (r16 & 7))]);
        if (c + 1 < a.chunks) issue(c + 1);
        multiply<F32>(wv, xv, acc);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = m0 + (wm * MT + t) * 16 + r16;
        if (row < a.m) {
            const float xs = a.xs[row];
#pragma unroll
            for (int f = 0; f < NT; ++f) {
                const int T = T0 + wn * NT + f;
                store4<F32>(a, row, row_of(T, 4 * g), acc[f][t], xs);
            }
        }
    }
}

// ----------------------------------------------------------------- packing
// One workgroup a packed row: its largest value, then its values in order.
__global__ void __launch_bounds__(256) fp8_pack_kernel(const void *w, int dtype, uint8_t *out, float *scales, int n, int k,
                                                       int chunks) {
    __shared__ uint32_t red[4];
    const int T = blockIdx.x >> 4, i = blockIdx.x & 15, row = row_of(T, i);
    const bool real = row < n;
    auto value = [&](int c) {
        return dtype == ZK_F32 ? ((const float *)w)[(size_t)row * k + c]
                               : __uint_as_float((uint32_t)((const uint16_t *)w)[(size_t)row * k + c] << 16);
    };
    float r = 0.0f;
    if (dtype != ZK_FP8_E4M3 && real) {
        uint32_t top = 0;  // as bits: NaN above infinity above the numbers
        for (int c = threadIdx.x; c < k; c += 256) top = max(top, __float_as_uint(value(c)) & 0x7fffffffu);
        for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o));
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = top;
        __syncthreads();
        top = max(max(red[0], red[1]), max(red[2], red[3]));
        const float most = __uint_as_float(top) / 448.0f, s = most < 0x1p-126f ? 0x1p-126f : most;
        if (threadIdx.x == 0) scales[row] = s;
        r = 1.0f / s;
    }
    uint8_t *to = out + (size_t)T * chunks * kTile + i * 16;
    for (int c = threadIdx.x; c < chunks * kChunk; c += 256) {
        uint8_t q = 0;
        if (real && c < k)
            q = dtype == ZK_FP8_E4M3 ? ((const uint8_t *)w)[(size_t)row * k + c]
                                     : (uint8_t)e4m3x4(value(c) * r, 0.f, 0.f, 0.f);
        to[(size_t)(c / kChunk) * kTile + (c % kChunk) / 16 * 256 + c % 16] = q;
    }
}

bool meet(const void *p, int64_t pb, const void *q, int64_t qb) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return pb > 0 && qb > 0 && a < b + qb && b < a + pb;
}
int bad(const char *what) { return set_error(ZK_ERR_INVALID_ARGUMENT, std::string("Internal error: ") + what); }
bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }

template <bool F32>
void launch(GemmArgs a, hipStream_t s) {
    if (a.m <= 64) {
        const dim3 grid((unsigned)a.tiles);
        if (a.m <= 16) fp8_stream_kernel<1, 1, 8, 4, F32><<<grid, 512, 0, s>>>(a);
        else if (a.m <= 32) fp8_stream_kernel<1, 2, 8, 4, F32><<<grid, 512, 0, s>>>(a);
        else fp8_stream_kernel<1, 4, 8, 2, F32><<<grid, 512, 0, s>>>(a);
        return;
    }
    auto go = [&](auto kernel, int bm, int bt, int threads) {
        a.tiles_m = (a.m + bm - 1) / bm;
        a.tiles_n = (a.tiles + bt - 1) / bt;
        const int64_t all = (int64_t)a.tiles_m * a.tiles_n;
        kernel<<<(unsigned)(8 * ((all + 7) / 8)), threads, 0, s>>>(a);
    };
    const int64_t big = (int64_t)((a.m + 255) / 256) * ((a.tiles + 15) / 16);
    if constexpr (!F32)
        if (big >= 256) return go(fp8_gemm_kernel<8, 4, 2, 4, false>, 256, 16, 512);
    go(fp8_gemm_kernel<4, 4, 2, 2, F32>, 128, 8, 256);
}

}  // namespace

extern "C" {

size_t zk_fp8_weight_bytes(int64_t n, int64_t k) {
    if (n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24)) return 0;
    return (size_t)((n + 63) / 64) * 4 * ((k + kChunk - 1) / kChunk) * kTile;
}

int zk_fp8_weight(const void *w, zk_dtype dtype, void *packed, float *scales, int64_t n, int64_t k, void *stream) {
    if (!valid_dtype(dtype)) return bad("zk_fp8_weight: unknown dtype");
    if (n <= 0 || k <= 0 || n > (1 << 24) || k > (1 << 24)) return bad("zk_fp8_weight: bad shape");
    if (!w || !packed || (!scales && dtype != ZK_FP8_E4M3)) return bad("zk_fp8_weight: NULL pointer");
    if (!aligned16(packed)) return bad("zk_fp8_weight: the packed weight must be 16-byte aligned");
    const int64_t bytes = (int64_t)zk_fp8_weight_bytes(n, k), in = n * k * elt_size(dtype);
    const int64_t out = dtype == ZK_FP8_E4M3 ? 0 : 4 * n;  // (its scales are the caller's)
    if (meet(packed, bytes, w, in) || meet(scales, out, w, in) || meet(scales, out, packed, bytes))
        return bad("zk_fp8_weight: operands overlap");
    hipStream_t s = (hipStream_t)stream;
    const int chunks = (int)((k + kChunk - 1) / kChunk);
    fp8_pack_kernel<<<(unsigned)((n + 63) / 64 * 64), 256, 0, s>>>(w, dtype, (uint8_t *)packed, scales, (int)n, (int)k, chunks);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_fp8_weight: ") + hipGetErrorString(e));
    return ZK_OK;
}

int zk_linear_fp8(const void *x, const float *x_scales, const void *packed, const float *w_scales, void *y, int64_t m,
                  int64_t n, int64_t k, zk_dtype out_dtype, void *stream) {
    if (out_dtype != ZK_F32 && out_dtype != ZK_BF16) return bad("zk_linear_fp8: the output must be f32 or bf16");
    if (m < 0 || n <= 0 || k <= 0 || m > (1 << 24) || n > (1 << 24) || k > (1 << 24)) return bad("zk_linear_fp8: bad shape");
    if (k % 16) return bad("zk_linear_fp8: k must be a multiple of 16");
    if (m == 0) return ZK_OK;
    if (!x || !x_scales || !packed || !w_scales || !y) return bad("zk_linear_fp8: NULL pointer");
    if (!aligned16(x) || !aligned16(packed) || !aligned16(y)) return bad("zk_linear_fp8: x, the weight and y must be 16-byte aligned");
    const int64_t out = m * n * elt_size(out_dtype);
    if (meet(y, out, x, m * k) || meet(y, out, x_scales, 4 * m) || meet(y, out, packed, (int64_t)zk_fp8_weight_bytes(n, k)) ||
        meet(y, out, w_scales, 4 * n))
        return bad("zk_linear_fp8: y overlaps an input");
    GemmArgs a{};
    a.x = (const uint8_t *)x;
    a.xs = x_scales;
    a.w = (const uint8_t *)packed;
    a.ws = w_scales;
    a.y = y;
    a.m = (int)m;
    a.n = (int)n;
    a.k = (int)k;
    a.chunks = (int)((k + kChunk - 1) / kChunk);
    a.tiles = (int)((n + 63) / 64 * 4);
    if ((int64_t)((m + 127) / 128) * ((a.tiles + 7) / 8) > (1 << 28)) return bad("zk_linear_fp8: too many rows and columns");
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("linear_fp8", s);
    if (out_dtype == ZK_F32) launch<true>(a, s);
    else launch<false>(a, s);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_linear_fp8: ") + hipGetErrorString(e));
    return ZK_OK;
}

}  // extern "C"
