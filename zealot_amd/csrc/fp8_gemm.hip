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
#include <type_traits>

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
    int splits, split_chunks;    // of k
    float *partial;
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
        for (int t = 0; t < MT; ++t)
#pragma unroll
            for (int f = 0; f < NT; ++f)
                acc[f][t] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w[f], x[t], acc[f][t], 0, 0, 0, 0, 0, 0);
    }
}

// The weight row of row i of tile T.
__device__ __forceinline__ int row_of(int T, int i) { return 64 * (T >> 2) + 16 * (i >> 2) + 4 * (T & 3) + (i & 3); }

// two values as bf16, to nearest even (one instruction)
__device__ __forceinline__ uint32_t two(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2_t));
}
// Column scales ws[n0 ..); behind the last one it again (nothing is stored there).
template <int N>
__device__ __forceinline__ void column_scales(const GemmArgs &a, int n0, float (&ws)[N]) {
    if (n0 + N <= a.n) {
#pragma unroll
        for (int i = 0; i < N; ++i) ws[i] = a.ws[n0 + i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) ws[i] = a.ws[min(n0 + i, a.n - 1)];
    }
}
// pieces of y's rows, which lie at their elements' alignment only where n is no multiple of 8
typedef u32x4 __attribute__((aligned(2))) u32x4_any;
typedef u32x2 __attribute__((aligned(2))) u32x2_any;
typedef f32x4 __attribute__((aligned(4))) f32x4_any;
// y[row, n0 .. n0 + N) = v * xs * ws, N a multiple of 4
template <bool F32, int N>
__device__ __forceinline__ void store_row(const GemmArgs &a, int row, int n0, const float (&v)[N], const float (&ws)[N], float xs) {
    float o[N];
#pragma unroll
    for (int i = 0; i < N; ++i) o[i] = v[i] * xs * ws[i];
    const size_t at = (size_t)row * a.n + n0;
    if (n0 + N <= a.n) {
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<f32x4_any *>((float *)a.y + at + i) = f32x4{o[i], o[i + 1], o[i + 2], o[i + 3]};
        } else if constexpr (N % 8 == 0) {
#pragma unroll
            for (int i = 0; i < N; i += 8)
                *reinterpret_cast<u32x4_any *>((uint16_t *)a.y + at + i) =
                    u32x4{two(o[i], o[i + 1]), two(o[i + 2], o[i + 3]), two(o[i + 4], o[i + 5]),
                          two(o[i + 6], o[i + 7])};
        } else {
#pragma unroll
            for (int i = 0; i < N; i += 4)
                *reinterpret_cast<u32x2_any *>((uint16_t *)a.y + at + i) = u32x2{two(o[i], o[i + 1]), two(o[i + 2], o[i + 3])};
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (n0 + i < a.n) {
                if constexpr (F32) ((float *)a.y)[at + i] = o[i];
                else ((uint16_t *)a.y)[at + i] = (uint16_t)two(o[i], 0.0f);
            }
    }
}
template <bool F32>
__device__ __forceinline__ void store4(const GemmArgs &a, int row, int n0, const f32x4 &v, float xs) {
    if (n0 >= a.n) return;
    float ws[4], u[4] = {v[0], v[1], v[2], v[3]};
    column_scales(a, n0, ws);
    store_row<F32>(a, row, n0, u, ws, xs);
}

// ------------------------------------------------------------ few rows of x
// (At most 16.)  A workgroup owns NT tiles of 16 weight rows and all of k, its KW
// waves every KW-th chunk of it: weights and x come from memory straight into the
// registers of the instruction, U chunks at a time, and the waves' sums meet in
// LDS, in the order of the waves.
template <int NT, int KW, int U, bool F32>
__global__ void __launch_bounds__(64 * KW) fp8_stream_kernel(GemmArgs a) {
    __shared__ f32x4 sums[KW][NT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    const int T0 = blockIdx.x * NT;
    const uint8_t *wp = a.w + (size_t)T0 * a.chunks * kTile + lane * 16;
    const uint8_t *xp = a.x + (size_t)min(r16, a.m - 1) * a.k + 16 * g;
    f32x4 acc[NT][1];
#pragma unroll
    for (int f = 0; f < NT; ++f) acc[f][0] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c0 = wave; c0 < a.chunks; c0 += KW * U) {
        u32x4 wv[U][NT][2], xv[U][2];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            // (behind the last chunk: its weights again, times zeros, and no branch around a load)
            const int c = c0 + u * KW, cw = min(c, a.chunks - 1);
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int f = 0; f < NT; ++f)
                    wv[u][f][h] = __builtin_nontemporal_load(
                        reinterpret_cast<const u32x4 *>(wp + ((size_t)f * a.chunks + cw) * kTile + 1024 * h));
                const bool in = c * kChunk + 64 * h + 16 * g < a.k;
                xv[u][h] = *reinterpret_cast<const u32x4 *>(in ? xp + c * kChunk + 64 * h : kZeros);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (every load before the first product)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            i32x8 w[NT], x[1];
#pragma unroll
            for (int f = 0; f < NT; ++f) w[f] = join(wv[u][f][0], wv[u][f][1]);
            x[0] = join(xv[u][0], xv[u][1]);
            multiply<F32>(w, x, acc);
        }
    }
#pragma unroll
    for (int f = 0; f < NT; ++f) sums[wave][f][lane] = acc[f][0];
    __syncthreads();
#pragma unroll
    for (int f = wave; f < NT; f += KW) {
        f32x4 v = sums[0][f][lane];
#pragma unroll
        for (int k = 1; k < KW; ++k) v += sums[k][f][lane];
        if (r16 < a.m) store4<F32>(a, r16, row_of(T0 + f, 4 * g), v, a.xs[r16]);
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
__device__ __forceinline__ void wait_lgkm0() { __builtin_amdgcn_s_waitcnt(0xc07f); }
// workgroup barrier without the fences of __syncthreads (those would wait for
// every load in flight); the memory clobber keeps LDS accesses on their side
__device__ __forceinline__ void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

// A workgroup owns 16 MT WM rows of x, 16 NT WN weight rows and a stretch of k;
// chunks of both come to LDS by DMA in a ring of D stages, D - 1 of them ahead.
// Weights stay in their packed order; a row of x has its eight units at u ^ (row
// % 8), so the eight rows of a DMA are whole 128-byte lines and the reads of a
// unit of 16 rows hit every bank alike.  With splits of k the sums go to `partial`
// ([splits][m][16 tiles] f32) and fp8_sum_kernel adds them in order.
template <int MT, int NT, int WM, int WN, int D, int KS, bool F32>
__global__ void __launch_bounds__(64 * WM * WN) fp8_gemm_kernel(GemmArgs a) {
    constexpr int kWaves = WM * WN;
    constexpr int BM = 16 * MT * WM, BT = NT * WN;  // rows of x, weight tiles
    constexpr int WQ = BT * 2, XQ = BM / 8;         // DMA instructions a chunk
    constexpr int WL = WQ / kWaves, XL = XQ / kWaves, L = WL + XL;
    static_assert(WQ % kWaves == 0 && XQ % kWaves == 0, "split over the waves");
    static_assert(4 % NT == 0, "a wave's tiles lie in one group of 64 rows");
    __shared__ u32x4 lds[D][KS][(BT * kTile + BM * kChunk) / 16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    // An XCD takes a run of tiles, eight m-tiles side by side: workgroups that
    // run at once share their rows and weights in its L2.
    const int all = a.tiles_m * a.tiles_n * a.splits, per = (all + 7) / 8;
    int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || tile >= all) return;
    const int split = tile / (a.tiles_m * a.tiles_n);
    tile -= split * a.tiles_m * a.tiles_n;
    const int band = tile / (8 * a.tiles_n), high = min(8, a.tiles_m - 8 * band), in = tile - band * 8 * a.tiles_n;
    const int tm = 8 * band + in % high, tn = in / high;
    const int m0 = tm * BM, T0 = tn * BT;
    const int c_begin = split * a.split_chunks, c_end = min(c_begin + a.split_chunks, a.chunks);

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
    auto issue = [&](int c0, int slot) {
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            u32x4 *st = lds[slot][u];
            const int c = min(c0 + u, c_end - 1);  // (what is behind the last chunk is not used)
#pragma unroll
            for (int j = 0; j < WL; ++j) g2l16(wsrc[j] + (size_t)c * kTile, (lds_void *)(st + 64 * (wave * WL + j)));
#pragma unroll
            for (int j = 0; j < XL; ++j)
                g2l16(c * kChunk + xcol[j] < a.k ? xsrc[j] + c * kChunk : kZeros,
                      (lds_void *)(st + BT * kTile / 16 + 64 * (wave * XL + j)));
        }
    };
    f32x4 acc[NT][MT];
#pragma unroll
    for (int f = 0; f < NT; ++f)
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[f][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int wm = wave % WM, wn = wave / WM;
#pragma unroll
    for (int d = 0; d < D - 1; ++d)
        if (c_begin + d * KS < c_end) issue(c_begin + d * KS, d);
    int slot = 0;
    for (int c = c_begin; c < c_end; c += KS) {
        // the stage is in once only those issued after it fly; the barrier says so
        // of every wave's part, and that every wave has left the stage before it
        // (near the end there is no more to issue: everything)
        if (c + (D - 2) * KS < c_end) wait_vmcnt<(D - 2) * KS * L>();
        else wait_vmcnt<0>();
        wg_barrier();
        i32x8 wv[KS][NT], xv[KS][MT];
#pragma unroll
        for (int u = 0; u < KS; ++u) {
            const u32x4 *wl = lds[slot][u] + wn * NT * (kTile / 16) + lane;
            const u32x4 *xl = lds[slot][u] + BT * kTile / 16 + (wm * MT * 16 + r16) * 8;
#pragma unroll
            for (int f = 0; f < NT; ++f) wv[u][f] = join(wl[f * (kTile / 16)], wl[f * (kTile / 16) + 64]);
#pragma unroll
            for (int t = 0; t < MT; ++t)
                xv[u][t] = join(xl[t * 128 + (g ^ (r16 & 7))], xl[t * 128 + ((g + 4) ^ (r16 & 7))]);
        }
        if (c + (D - 1) * KS < c_end) issue(c + (D - 1) * KS, slot == 0 ? D - 1 : slot - 1);
#pragma unroll
        for (int u = 0; u < KS; ++u)
            if (KS == 1 || c + u < c_end) multiply<F32>(wv[u], xv[u], acc);
        slot = slot == D - 1 ? 0 : slot + 1;
    }
    // (a lane's columns follow one another over the tiles: 4 NT from here on)
    const int T1 = T0 + wn * NT, n0 = row_of(T1, 4 * g);
    if (n0 >= a.n) return;
    if (a.splits > 1) {
        if (T1 >= a.tiles) return;
#pragma unroll
        for (int t = 0; t < MT; ++t) {
            const int row = m0 + (wm * MT + t) * 16 + r16;
            float *to = a.partial + ((size_t)split * a.m + row) * (16 * a.tiles) + n0;
            if (row < a.m)
#pragma unroll
                for (int f = 0; f < NT; ++f) *reinterpret_cast<f32x4 *>(to + 4 * f) = acc[f][t];
        }
        return;
    }
    float ws[4 * NT], xs[MT];  // (every scale before the first is used: one latency)
    column_scales(a, n0, ws);
#pragma unroll
    for (int t = 0; t < MT; ++t) xs[t] = a.xs[min(m0 + (wm * MT + t) * 16 + r16, a.m - 1)];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
        const int row = m0 + (wm * MT + t) * 16 + r16;
        if (row >= a.m) continue;
        float v[4 * NT];
#pragma unroll
        for (int i = 0; i < 4 * NT; ++i) v[i] = acc[i / 4][t][i % 4];
        store_row<F32>(a, row, n0, v, ws, xs[t]);
    }
}

// Many rows: 256 rows of x by 256 weight rows a workgroup, eight waves of 128 by
// 64 (two a SIMD), k in steps of 64.  A step's 32 KiB come to LDS by DMA in a ring
// of four.  The matrix instruction is 32x32x64, so that a step of a wave's
// operands is 48 registers: the next step's come from LDS while this one
// multiplies.  Lane l has row l % 32 of either operand (of weights packed tile l %
// 32 / 16) and units 2 (l / 32), 2 (l / 32) + 1 of the step's four, and ends with
// columns 16 (l / 32) + 32 (j % 2) + 8 a + 4 (j / 2) + i of its 64 in element 4 j + i
// of tile a: two runs of 16.  x lies in rows of 64 bytes, unit u at u ^ (row / 4 %
// 4): the reads of a unit of 16 rows hit every bank once.  8192 x 28672 x 4096: 790
// us, 658 without y's stores; the card's clock is 1.7 GHz under it and the matrix
// cores are busy 68 % of that.  (Workgroups that stay for several tiles, with the next
// tile's first stages ahead of the stores, took as long.)
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;
__device__ __forceinline__ rsrc_t buffer_of(const uint8_t *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, (int)bytes, 0x00027000);
}
__device__ __forceinline__ void b2l16(rsrc_t b, lds_void *l, uint32_t lane_at, uint32_t at) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(b, l, 16, (int)lane_at, (int)at, 0, 0);
}
template <bool EARLY>
__global__ void __launch_bounds__(512, 2) fp8_gemm_big_kernel(GemmArgs a) {
    constexpr int BM = 256, BT = 16, D = 4, kAhead = EARLY ? 3 : 0, kStage = 2048;  // (16-byte units of a stage)
    __shared__ u32x4 lds[D * kStage + (kAhead ? 8 * 16 : 0)];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r32 = lane & 31, h = lane >> 5;
    const int all = a.tiles_m * a.tiles_n, per = (all + 7) / 8;
    const int tile = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if ((int)(blockIdx.x >> 3) >= per || tile >= all) return;
    const int band = tile / (8 * a.tiles_n), high = min(8, a.tiles_m - 8 * band), in = tile - band * 8 * a.tiles_n;
    const int tm = 8 * band + in % high, tn = in / high, m0 = tm * BM, T0 = tn * BT;
    const int wm = wave & 1, wn = wave >> 1;

    // rows and tiles behind the last are behind the buffers' ends: nothing is read there
    const int tiles = min(BT, a.tiles - T0), rows = min(BM, a.m - m0);
    const rsrc_t wb = buffer_of(a.w + (size_t)T0 * a.chunks * kTile, (uint32_t)(tiles * a.chunks * kTile));
    const rsrc_t xb = buffer_of(a.x + (size_t)m0 * a.k, (uint32_t)rows * (uint32_t)a.k);
    // a wave's DMA: two tiles' weights (1 KiB each) and 32 rows of x (16 at a time)
    // (what tells a lane from its buffer's end lies in its own offset: a scalar offset behind the end is not checked)
    uint32_t woff[2], xoff[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
        woff[j] = (uint32_t)((wave * 2 + j) * a.chunks) * kTile + lane * 16;
        const int r = (wave * 2 + j) * 16 + (lane >> 2);
        xoff[j] = (uint32_t)r * a.k + 16 * ((lane & 3) ^ ((r >> 2) & 3));
    }
    // early lines: 64 rows of x, 32 lines of weights, twelve a wave
    const uint8_t *early;
    uint32_t early_step;
    {
        const int i = min(wave * 12 + lane, 95);
        if (i < 64) {
            early = a.x + (size_t)(m0 + min(4 * i + (tn & 3), rows - 1)) * a.k;
            early_step = kChunk;
        } else {
            const int line = (i - 64) * 8 + (tm & 7);
            early = a.w + (size_t)(T0 + min(line >> 4, tiles - 1)) * a.chunks * kTile + (line & 15) * 128;
            early_step = kTile;
        }
    }
    auto fetch_early = [&](int s) {
        if (kAhead && !(s & 1) && lane < 12) {
            const uint8_t *e = early + (size_t)(uint32_t)min(s / 2 + kAhead, a.chunks - 1) * early_step;
            __builtin_amdgcn_global_load_lds(e, (lds_void *)(lds + D * kStage + wave * 16), 4, 0, 0);
        }
    };
    // the j-th of a wave's four DMA instructions of step s
    auto issue = [&](int s, int slot, int j) {
        u32x4 *st = lds + slot * kStage;
        if (j < 2) b2l16(wb, (lds_void *)(st + 64 * (wave * 2 + j)), woff[j], 1024u * s);
        else b2l16(xb, (lds_void *)(st + 1024 + 64 * (wave * 2 + j - 2)), xoff[j - 2] + 64u * s, 0);
    };
    f32x16 acc[2][4];
#pragma unroll
    for (int f = 0; f < 2; ++f)
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) acc[f][t][i] = 0.0f;
    const int wl = (wn * 4 + (r32 >> 4)) * 64 + 2 * h * 16 + (r32 & 15);
    const int xr = 1024 + (wm * 128 + r32) * 4, xs = (r32 >> 2) & 3;
    const int xl0 = xr + ((2 * h) ^ xs), xl1 = xr + ((2 * h + 1) ^ xs);
    auto read_w = [&](int slot, int f, i32x8 (&w)[2]) {
        const u32x4 *st = lds + slot * kStage;
        w[f] = join(st[wl + f * 128], st[wl + f * 128 + 16]);
    };
    auto read_x = [&](int slot, int t, i32x8 (&x)[4]) {
        const u32x4 *st = lds + slot * kStage;
        x[t] = join(st[xl0 + t * 128], st[xl1 + t * 128]);
    };
    auto product = [&](int t, int f, const i32x8 (&w)[2], const i32x8 (&x)[4]) {
        acc[f][t] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(w[f], x[t], acc[f][t], 0, 0, 0, 0, 0, 0);
    };
    i32x8 w0[2], x0[4], w1[2], x1[4];
    const int steps = 2 * a.chunks;
    auto next = [](int slot) { return slot == D - 1 ? 0 : slot + 1; };
    // columns from k on (k is a multiple of 16) are other rows': in the last chunk they become zeros, like the weights there
    auto clear = [&](int s, int slot) {
        const int first = max(0, (a.k - 64 * s) / 16);
        u32x4 *st = lds + slot * kStage + 1024;
        for (int i = threadIdx.x; i < BM * 4; i += 512)
            if ((i & 3) >= first) st[(i & ~3) + ((i & 3) ^ ((i >> 4) & 3))] = u32x4{0, 0, 0, 0};
        wait_lgkm0();
        wg_barrier();
    };
    // Step s, whose operands are in w and x; the next step's go to wn and xn.  A quarter of its products come first, so that
    // the matrix cores have work at the barrier, which says: step s + 1 is in, everywhere, and step s is in every wave's
    // registers, so its slot takes step s + D.  Reads and DMA go between the other products, a few at a time: together they
    // would hold up the wave for hundreds of cycles (a CU takes a DMA instruction every 16).
#define PIN __builtin_amdgcn_sched_barrier(0)
    auto step = [&](auto last, int s, int slot, const i32x8 (&w)[2], const i32x8 (&x)[4], i32x8 (&wn)[2], i32x8 (&xn)[4]) {
        constexpr bool kLast = decltype(last)::value;  // one of the last D steps
        const bool more = !kLast || s + D < steps;
        const int to = next(slot);
        product(0, 0, w, x);
        product(0, 1, w, x);
        PIN;
        wait_lgkm0();
        if (!kLast || s + D - 1 < steps) wait_vmcnt<(D - 2) * 4 + (kAhead ? 1 : 0)>();
        else wait_vmcnt<0>();
        wg_barrier();
        if (kLast && 64 * (s + 2) > a.k) clear(s + 1, to);
        PIN;
        product(1, 0, w, x);
        PIN;
        if (more) {
            fetch_early(s + D);
            issue(s + D, slot, 0);
        }
        read_w(to, 0, wn);
        PIN;
        product(1, 1, w, x);
        PIN;
        if (more) issue(s + D, slot, 1);
        read_w(to, 1, wn);
        PIN;
        product(2, 0, w, x);
        PIN;
        if (more) issue(s + D, slot, 2);
        read_x(to, 0, xn);
        PIN;
        product(2, 1, w, x);
        PIN;
        if (more) issue(s + D, slot, 3);
        read_x(to, 1, xn);
        PIN;
        product(3, 0, w, x);
        PIN;
        read_x(to, 2, xn);
        PIN;
        product(3, 1, w, x);
        PIN;
        read_x(to, 3, xn);
        PIN;
    };
#pragma unroll
    for (int d = 0; d < D; ++d) {  // (there are at least as many steps: kBigChunks)
        fetch_early(d);
#pragma unroll
        for (int j = 0; j < 4; ++j) issue(d, d, j);
    }
    wait_vmcnt<(D - 1) * 4 + (kAhead ? 1 : 0)>();
    wg_barrier();
#pragma unroll
    for (int f = 0; f < 2; ++f) read_w(0, f, w0);
#pragma unroll
    for (int t = 0; t < 4; ++t) read_x(0, t, x0);
    int s = 0, slot = 0;
    for (; s + D + 1 < steps; s += 2) {
        step(std::false_type{}, s, slot, w0, x0, w1, x1);
        slot = next(slot);
        step(std::false_type{}, s + 1, slot, w1, x1, w0, x0);
        slot = next(slot);
    }
    for (; s + 2 < steps; s += 2) {
        step(std::true_type{}, s, slot, w0, x0, w1, x1);
        slot = next(slot);
        step(std::true_type{}, s + 1, slot, w1, x1, w0, x0);
        slot = next(slot);
    }
    step(std::true_type{}, s, slot, w0, x0, w1, x1);
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        product(t, 0, w1, x1);
        product(t, 1, w1, x1);
    }
#undef PIN
    // columns n0 .. + 15 and n0 + 32 .. + 47; every scale before the first is used: one latency
    const int n0 = 16 * (T0 + 4 * wn) + 16 * h;
    float ws[2][16], xs4[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) column_scales(a, n0 + 32 * q, ws[q]);
#pragma unroll
    for (int t = 0; t < 4; ++t) xs4[t] = a.xs[min(m0 + wm * 128 + 32 * t + r32, a.m - 1)];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
        const int row = m0 + wm * 128 + 32 * t + r32;
        if (row >= a.m) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            float v[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = acc[i >> 3][t][4 * (q + 2 * ((i >> 2) & 1)) + (i & 3)];
            if (n0 + 32 * q < a.n) store_row<false>(a, row, n0 + 32 * q, v, ws[q], xs4[t]);
        }
    }
}

// y from the sums of the splits, four columns a thread.
template <bool F32>
__global__ void __launch_bounds__(256) fp8_sum_kernel(GemmArgs a) {
    const int quads = 4 * a.tiles;
    const size_t q = (size_t)blockIdx.x * 256 + threadIdx.x;
    if (q >= (size_t)a.m * quads) return;
    const int row = (int)(q / quads), n0 = (int)(q - (size_t)row * quads) * 4;
    f32x4 v[1];
    sum_ranges(reinterpret_cast<const f32x4 *>(a.partial) + q, (size_t)a.m * quads, a.splits, v);
    store4<F32>(a, row, n0, v[0], a.xs[row]);
}

// ----------------------------------------------------------------- packing
// One workgroup a tile of 16 rows, 16 threads a row: the rows' largest values, then
// their values in order, a unit of 16 a thread (28672 x 4096 from e4m3 values 46 us, byte by byte 112;
// from bf16 111 us, 323; from f32 186).
template <typename T>
__global__ void __launch_bounds__(256) fp8_pack_kernel(const T *w, uint8_t *out, float *scales, int n, int k, int chunks, bool vec) {
    constexpr bool kReady = sizeof(T) == 1;  // values and scales are there
    __shared__ uint32_t red[4][16];
    const int tile = blockIdx.x, i = threadIdx.x & 15, row = row_of(tile, i), units = chunks * (kChunk / 16);
    const bool real = row < n;
    const T *from = w + (size_t)min(row, n - 1) * k;
    // the 16 values of a unit, zeros from column k on
    auto unit = [&](int u, T (&v)[16]) {
        if (vec && 16 * u + 16 <= k) {
#pragma unroll
            for (int j = 0; j < (int)sizeof(T); ++j) {
                const u32x4 piece = reinterpret_cast<const u32x4 *>(from + 16 * u)[j];
                __builtin_memcpy(reinterpret_cast<char *>(v) + 16 * j, &piece, 16);
            }
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = 16 * u + j < k ? from[16 * u + j] : T(0);
        }
    };
    auto f32_of = [](T v) {
        if constexpr (sizeof(T) == 4) return v;
        else return __uint_as_float((uint32_t)v << 16);
    };
    float s = 1.0f, r = 1.0f;
    if constexpr (!kReady) {
        uint32_t top = 0;  // as bits: NaN above infinity above the numbers
        for (int u = threadIdx.x >> 4; u < units; u += 16) {
            alignas(16) T v[16];
            unit(u, v);
#pragma unroll
            for (int j = 0; j < 16; ++j) top = max(top, __float_as_uint(f32_of(v[j])) & 0x7fffffffu);
        }
        top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        if ((threadIdx.x & 63) < 16) red[threadIdx.x >> 6][i] = top;
        __syncthreads();
        top = max(max(red[0][i], red[1][i]), max(red[2][i], red[3][i]));
        const float most = __uint_as_float(top) / 448.0f;
        s = most < 0x1p-126f ? 0x1p-126f : most;  // (NaN stays)
        if (threadIdx.x < 16 && real) scales[row] = s;
        r = 1.0f / s;
    }
    u32x4 *to = reinterpret_cast<u32x4 *>(out + (size_t)tile * chunks * kTile) + i;
    for (int u = threadIdx.x >> 4; u < units; u += 16) {
        alignas(16) T v[16];
        unit(u, v);
        u32x4 q;
        if constexpr (kReady) {
            __builtin_memcpy(&q, v, 16);
        } else if (s < __builtin_inff()) {
            auto over = [&](T y) { return quotient(f32_of(y), s, r); };
#pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = e4m3x4_in_range(over(v[4 * j]), over(v[4 * j + 1]), over(v[4 * j + 2]), over(v[4 * j + 3]));
        } else {  // no quotients: NaN, and zeros beside an infinity
#pragma unroll
            for (int j = 0; j < 4; ++j)
                q[j] = e4m3x4(f32_of(v[4 * j]) * r, f32_of(v[4 * j + 1]) * r, f32_of(v[4 * j + 2]) * r, f32_of(v[4 * j + 3]) * r);
        }
        to[u * 16] = real ? q : u32x4{0, 0, 0, 0};
    }
}

bool meet(const void *p, int64_t pb, const void *q, int64_t qb) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return pb > 0 && qb > 0 && a < b + qb && b < a + pb;
}
int bad(const char *what) { return set_error(ZK_ERR_INVALID_ARGUMENT, std::string("Internal error: ") + what); }
bool aligned16(const void *p) { return ((uintptr_t)p & 15u) == 0; }
bool shape_ok(int64_t m, int64_t n, int64_t k) {
    return m >= 0 && m <= (1 << 24) && n > 0 && n <= (1 << 22) && k > 0 && k <= (1 << 22) && k % 16 == 0;
}

// ------------------------------------------------------------------- choice
// What a product runs on.  Up to 16 rows of x the weights' stream is all that
// counts (1 row, 4096 x 14336: 11.1 us, 8.9 of them the weights at a copy's rate).
// Above, a call is taken to last
//   launch + rounds of 256 workgroups x (start + chunks x a chunk's time)
// and, with splits of k, their sums' launch and traffic: of the tiles and splits
// the one that this says ends first.  A chunk's time is what the tile was measured
// at with weights from memory and one workgroup a CU (4096 columns of 4096 and
// 14336): it grows with the tile's bytes, not its products, up to the largest.
struct Tile {
    int bm, bt;           // rows of x, 16-row weight tiles
    float start, chunk;   // us
};
enum { k32x32, k32x64, k64x32, k64x64, k64x128, k128x64, k128x128, k256x128, k256x256, kTiles };
constexpr Tile kTileCosts[kTiles] = {{32, 2, 0.6f, 0.155f}, {32, 4, 0.7f, 0.23f},  {64, 2, 0.9f, 0.20f},
                                     {64, 4, 0.6f, 0.275f}, {64, 8, 0.9f, 0.40f},  {128, 4, 0.9f, 0.405f},
                                     {128, 8, 1.6f, 0.60f}, {256, 8, 2.9f, 0.86f}, {256, 16, 6.7f, 1.44f}};
constexpr int kStreamRows = 16;
constexpr int kBigChunks = 4;  // of the largest tile at least (below, starting it costs more than it gains)
constexpr int kMaxSplits = 8;

struct Choice {
    int tile, splits, split_chunks;
};
Choice choose(int64_t m, int64_t n, int64_t k, bool f32) {
    const int64_t tiles = (n + 63) / 64 * 4, chunks = (k + kChunk - 1) / kChunk;
    Choice best{0, 1, (int)chunks};
    float least = 1e30f;
    for (int t = 0; t < (f32 ? k256x128 : kTiles); ++t) {  // (f32 results: their conversions fill the larger tiles' registers)
        const Tile &c = kTileCosts[t];
        const int64_t groups = ((m + c.bm - 1) / c.bm) * ((tiles + c.bt - 1) / c.bt);
        if (t == k256x256 && chunks < kBigChunks) continue;
        for (int s = 1; s <= (t == k256x256 ? 1 : kMaxSplits); s *= 2) {
            const int64_t each = (chunks + s - 1) / s;
            if (s > 1 && (each < 8 || groups * s > 512)) break;
            float us = (float)((groups * s + 255) / 256) * (c.start + each * c.chunk);
            if (s > 1) us += 2.5f + (float)s * m * tiles * 16 * 8 / 4e6f;
            if (us < least) {
                least = us;
                best = {t, (int)((chunks + each - 1) / each), (int)each};
            }
        }
    }
    return best;
}

template <bool F32>
void launch(GemmArgs a, const Choice &c, hipStream_t s) {
    if (a.m <= kStreamRows) {
        // few tiles: all the waves on one; many: four waves each, and from 9 rows on several tiles to a
        // load of x (16 rows, 28672 columns: 20.3 us with four, 24.3 with one)
        if (a.tiles <= 256) fp8_stream_kernel<1, 8, 4, F32><<<a.tiles, 512, 0, s>>>(a);
        else if (a.m <= 8) fp8_stream_kernel<1, 4, 8, F32><<<a.tiles, 256, 0, s>>>(a);
        else if (a.tiles < 1024) fp8_stream_kernel<2, 4, 4, F32><<<a.tiles / 2, 256, 0, s>>>(a);
        else fp8_stream_kernel<4, 4, 2, F32><<<a.tiles / 4, 256, 0, s>>>(a);
        return;
    }
    a.splits = c.splits;
    a.split_chunks = c.split_chunks;
    auto go = [&](auto kernel, int threads) {
        a.tiles_m = (a.m + kTileCosts[c.tile].bm - 1) / kTileCosts[c.tile].bm;
        a.tiles_n = (a.tiles + kTileCosts[c.tile].bt - 1) / kTileCosts[c.tile].bt;
        const int64_t all = (int64_t)a.tiles_m * a.tiles_n * a.splits;
        kernel<<<(unsigned)(8 * ((all + 7) / 8)), threads, 0, s>>>(a);
    };
    switch (c.tile) {
        case k32x32: go(fp8_gemm_kernel<2, 1, 1, 2, 4, 2, F32>, 128); break;
        case k32x64: go(fp8_gemm_kernel<2, 1, 1, 4, 4, 1, F32>, 256); break;
        case k64x32: go(fp8_gemm_kernel<2, 1, 2, 2, 4, 2, F32>, 256); break;
        case k64x64: go(fp8_gemm_kernel<2, 2, 2, 2, 4, 2, F32>, 256); break;
        case k64x128: go(fp8_gemm_kernel<2, 2, 2, 4, 6, 1, F32>, 512); break;
        case k128x64: go(fp8_gemm_kernel<2, 2, 4, 2, 6, 1, F32>, 512); break;
        case k128x128: go(fp8_gemm_kernel<2, 4, 4, 2, 4, 1, F32>, 512); break;
        default:
            if constexpr (!F32) {
                if (c.tile == k256x128) go(fp8_gemm_kernel<4, 4, 4, 2, 3, 1, false>, 512);
                // (early lines pay where eight m-tiles share them: 2048 x 4096 x 14336 156 -> 127 us, 512 rows 157 -> 176)
                else if (a.m > 7 * 256) go(fp8_gemm_big_kernel<true>, 512);
                else go(fp8_gemm_big_kernel<false>, 512);
            }
    }
    if (a.splits > 1) fp8_sum_kernel<F32><<<(unsigned)(((size_t)a.m * 4 * a.tiles + 255) / 256), 256, 0, s>>>(a);
}
size_t partial_bytes(int64_t m, int64_t n, const Choice &c) {
    return m <= kStreamRows || c.splits == 1 ? 0 : (size_t)c.splits * m * ((n + 63) / 64 * 64) * 4;
}

}  // namespace

extern "C" {

size_t zk_fp8_weight_bytes(int64_t n, int64_t k) {
    if (n <= 0 || k <= 0 || n > (1 << 22) || k > (1 << 22)) return 0;
    return (size_t)((n + 63) / 64) * 4 * ((k + kChunk - 1) / kChunk) * kTile;
}

int zk_fp8_weight(const void *w, zk_dtype dtype, void *packed, float *scales, int64_t n, int64_t k, void *stream) {
    if (!valid_dtype(dtype)) return bad("zk_fp8_weight: unknown dtype");
    if (n <= 0 || k <= 0 || n > (1 << 22) || k > (1 << 22)) return bad("zk_fp8_weight: bad shape");
    if (!w || !packed || (!scales && dtype != ZK_FP8_E4M3)) return bad("zk_fp8_weight: NULL pointer");
    if (!aligned16(packed)) return bad("zk_fp8_weight: the packed weight must be 16-byte aligned");
    const int64_t bytes = (int64_t)zk_fp8_weight_bytes(n, k), in = n * k * elt_size(dtype);
    const int64_t out = dtype == ZK_FP8_E4M3 ? 0 : 4 * n;  // (its scales are the caller's)
    if (meet(packed, bytes, w, in) || meet(scales, out, w, in) || meet(scales, out, packed, bytes))
        return bad("zk_fp8_weight: operands overlap");
    hipStream_t s = (hipStream_t)stream;
    const int chunks = (int)((k + kChunk - 1) / kChunk);
    const unsigned grid = (unsigned)((n + 63) / 64 * 4);
    const bool vec = k % 16 == 0 && aligned16(w);
    auto go = [&](auto *from) { fp8_pack_kernel<<<grid, 256, 0, s>>>(from, (uint8_t *)packed, scales, (int)n, (int)k, chunks, vec); };
    if (dtype == ZK_F32) go((const float *)w);
    else if (dtype == ZK_BF16) go((const uint16_t *)w);
    else go((const uint8_t *)w);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_fp8_weight: ") + hipGetErrorString(e));
    return ZK_OK;
}

size_t zk_linear_fp8_workspace_size(int64_t m, int64_t n, int64_t k, zk_dtype out_dtype) {
    if (!shape_ok(m, n, k) || m == 0) return 0;
    return partial_bytes(m, n, choose(m, n, k, out_dtype == ZK_F32));
}

int zk_linear_fp8(const void *x, const float *x_scales, const void *packed, const float *w_scales, void *y, int64_t m,
                  int64_t n, int64_t k, zk_dtype out_dtype, void *workspace, size_t workspace_bytes, void *stream) {
    if (out_dtype != ZK_F32 && out_dtype != ZK_BF16) return bad("zk_linear_fp8: the output must be f32 or bf16");
    if (!shape_ok(m, n, k)) return bad("zk_linear_fp8: bad shape (k a multiple of 16; at most 2^24 rows, 2^22 columns and k)");
    if (m == 0) return ZK_OK;
    if (!x || !x_scales || !packed || !w_scales || !y) return bad("zk_linear_fp8: NULL pointer");
    if (!aligned16(x) || !aligned16(packed) || !aligned16(y)) return bad("zk_linear_fp8: x, the weight and y must be 16-byte aligned");
    const Choice choice = choose(m, n, k, out_dtype == ZK_F32);
    const int64_t need = (int64_t)partial_bytes(m, n, choice);
    if (need && (!workspace || workspace_bytes < (size_t)need))
        return bad("zk_linear_fp8: workspace too small (zk_linear_fp8_workspace_size)");
    if (need && !aligned16(workspace)) return bad("zk_linear_fp8: the workspace must be 16-byte aligned");
    const int64_t out = m * n * elt_size(out_dtype);
    const struct {
        const void *p;
        int64_t bytes;
    } in[] = {{x, m * k}, {x_scales, 4 * m}, {packed, (int64_t)zk_fp8_weight_bytes(n, k)}, {w_scales, 4 * n}};
    for (const auto &i : in)
        if (meet(y, out, i.p, i.bytes) || meet(workspace, need, i.p, i.bytes)) return bad("zk_linear_fp8: y or the workspace overlaps an input");
    if (meet(y, out, workspace, need)) return bad("zk_linear_fp8: y overlaps the workspace");
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
    a.partial = (float *)workspace;
    if ((int64_t)((m + 31) / 32) * ((a.tiles + 1) / 2) > (1 << 28)) return bad("zk_linear_fp8: too many rows and columns");
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("linear_fp8", s);
    if (out_dtype == ZK_F32) launch<true>(a, choice, s);
    else launch<false>(a, choice, s);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_linear_fp8: ") + hipGetErrorString(e));
    return ZK_OK;
}

}  // extern "C"
