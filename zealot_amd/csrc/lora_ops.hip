// lora_ops.hip -- low-rank adapters of many requests beside a shared
// projection: y[t] += c_a B_a (A_a x[t]) for every row t whose request brings
// an adapter a = ids[t].  No counterpart in the reference (one model, one set
// of weights, src/model_loader.rs:241).
//
// A step's plan groups its rows by adapter, once for all layers' projections:
//   order    the rows, sorted by adapter, in order within one; then -1
//   offsets  where each adapter's rows begin in it
//   tiles    (adapter + 2^16 rows, first position) of runs of at most tile_rows
//            rows of one adapter; (-1, 0) behind the last
// A product is two launches over the tiles.  The shrink forms
// v[p] = c_a A_a x[order[p]] (f32, parts * rank values a row) with A as the first
// operand of the matrix instruction and the tile's rows as the second, k split
// over the waves of a workgroup and, where there are few tiles, over workgroups,
// whose sums the second launch adds in their order.  The expand takes 64 columns
// of y a wave: B's rows as the first operand, v as the second, straight from
// memory into registers; a lane ends with two runs of eight columns of a row and
// adds them in place.
// Columns of y may come in parts that have an A of their own each (query, key
// and value columns of a fused projection): part p meets v[p rank ..] alone.
//
// Every tile reads all of its adapter's A and B, from L2 after the first, and x
// once for every 64 ranks of all parts; y is read and written once.  A few rows are
// bound by the launches' latency, prompts of ranks above 32 by A and B (8192 rows of 4096
// columns: rank 32 53 us, 64 71, 128 112; the last asks L2 for 1 GB, x and y are 0.2).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>
#include <type_traits>

#include "zk_common.h"

using namespace zk;

namespace {

constexpr int kMaxAdapters = 2048;
constexpr int kMaxParts = 4;
constexpr int kMaxRank = 256, kMaxRanks = 512;  // of one part, of all

// Rows of a tile: 16 (one matrix instruction) for a decode step, where most
// tiles have few rows; 32 for prompts, whose rows of one adapter are many: A and
// B are read once per 32 rows, and 8192 rows are a workgroup a CU.  (64 rows of 32
// adapters 11.9 us with 16, 13.1 with 32; 1024 rows of 64, mixed, 14.1 and 15.5, in runs
// 16.3 and 15.4; 2048, mixed, 24.3 and 23.2; 8192 in runs 60.2 and 53.4.)
int tile_rows_for(int64_t rows) { return rows <= 1024 ? 16 : 32; }
int64_t max_tiles(int64_t rows, int64_t adapters) {
    return rows / tile_rows_for(rows) + std::min(rows, adapters);
}

// ---------------------------------------------------------------------- plan
struct PlanArgs {
    const int32_t *ids;
    int32_t *order, *offsets;
    int2 *tiles;
    int rows, adapters, bits, tile_shift, max_tiles;  // tiles of 2^tile_shift rows
};

// One workgroup: each wave counts the adapters of a stretch of rows, the counts of
// (adapter, wave) become positions, and each wave goes through its stretch again, 64
// rows at a time: lanes of the same adapter find each other bit by bit, or at once
// where all have one, as in a prompt.  The waves' counts are their own, so the order
// does not depend on scheduling.  What bounds it is the latency of a decode step (64
// rows 4.2 us) and the one CU of a long one; ids and positions are asked for kBatch
// groups of 64 at a time (32768 rows in runs 27 us, one at a time 53; mixed, of 2000
// adapters, 44, 68 where lanes find each other for the counts too).
constexpr int kBatch = 8;
__global__ void __launch_bounds__(1024) lora_plan_kernel(PlanArgs a) {
    __shared__ int at[16 * kMaxAdapters];
    __shared__ int first[kMaxAdapters], tile0[kMaxAdapters], count[kMaxAdapters];
    __shared__ int scan_rows[16], scan_tiles[16];
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6), A = a.adapters;
    const int tile_rows = 1 << a.tile_shift, stretch = ((a.rows + 1023) / 1024) * 64;
    const int r0 = min(wave * stretch, a.rows), r1 = min(r0 + stretch, a.rows);
    auto ids_of = [&](int r, int (&id)[kBatch]) {
#pragma unroll
        for (int i = 0; i < kBatch; ++i) id[i] = a.ids[min(r + 64 * i + lane, a.rows - 1)];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) id[i] = r + 64 * i + lane < r1 ? id[i] : -1;
    };
    // the lanes whose row has this lane's adapter (0: no row, no adapter)
    auto peers = [&](int id) -> uint64_t {
        const bool has = (unsigned)id < (unsigned)A;
        uint64_t same = __ballot(has);
        if (same == 0 || __ballot(id == __builtin_amdgcn_readfirstlane(id)) == ~0ull) return same;
        for (int b = 0; b < a.bits; ++b) {
            const uint64_t set = __ballot((id >> b) & 1);
            same &= (id >> b) & 1 ? set : ~set;
        }
        return has ? same : 0;
    };
    auto rank_of = [](uint64_t same) {   // how many of them come before this lane
        return __builtin_amdgcn_mbcnt_hi((unsigned)(same >> 32), __builtin_amdgcn_mbcnt_lo((unsigned)same, 0));
    };
    int id[kBatch];
    if (r0 < r1) ids_of(r0, id);
    for (int i = t; i < 16 * A; i += 1024) at[i] = 0;
    __syncthreads();
    for (int r = r0; r < r1; r += 64 * kBatch) {
        if (r > r0) ids_of(r, id);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            if (r + 64 * i >= r1) break;
            // (counts need no order: a lane adds its own, one lane for all where they are alike)
            const bool has = (unsigned)id[i] < (unsigned)A;
            if (__ballot(id[i] == __builtin_amdgcn_readfirstlane(id[i])) == ~0ull) {
                if (has && lane == 0) atomicAdd(&at[wave * A + id[i]], 64);
            } else if (has) {
                atomicAdd(&at[wave * A + id[i]], 1);
            }
        }
    }
    __syncthreads();
    const int per = (A + 1023) / 1024, a0 = min(t * per, A), a1 = min(a0 + per, A);
    int mine = 0, my_tiles = 0;
    for (int x = a0; x < a1; ++x) {
        int n = 0;
#pragma unroll
        for (int w = 0; w < 16; ++w) n += at[w * A + x];
        count[x] = n;
        mine += n;
        my_tiles += (n + tile_rows - 1) >> a.tile_shift;
    }
    int total, tiles;
    int pos = block_exclusive_scan_1024(mine, scan_rows, &total);
    int tile = block_exclusive_scan_1024(my_tiles, scan_tiles, &tiles);
    for (int x = a0; x < a1; ++x) {
        int c[16], n = pos;
#pragma unroll
        for (int w = 0; w < 16; ++w) c[w] = at[w * A + x];
        a.offsets[x] = pos;
        first[x] = pos;
        tile0[x] = tile;
#pragma unroll
        for (int w = 0; w < 16; ++w) {
            at[w * A + x] = n;
            n += c[w];
        }
        tile += (n - pos + tile_rows - 1) >> a.tile_shift;
        pos = n;
    }
    if (t == 0) a.offsets[A] = total;
    for (int i = total + t; i < a.rows; i += 1024) a.order[i] = -1;
    for (int i = tiles + t; i < a.max_tiles; i += 1024) a.tiles[i] = make_int2(-1, 0);
    __syncthreads();
    const bool again = r1 - r0 > 64 * kBatch;
    for (int r = r0; r < r1; r += 64 * kBatch) {
        if (again) ids_of(r, id);
        uint64_t same[kBatch];
        int base[kBatch];   // asked for all groups first: the answers come in order
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            same[i] = r + 64 * i < r1 ? peers(id[i]) : 0;
            base[i] = 0;
            if (same[i] && rank_of(same[i]) == 0)
                base[i] = atomicAdd(&at[wave * A + id[i]], __popcll(same[i]));
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            const int from = __shfl(base[i], same[i] ? __ffsll((unsigned long long)same[i]) - 1 : lane);
            if (same[i] == 0) continue;
            const int p = from + (int)rank_of(same[i]), j = p - first[id[i]];
            a.order[p] = r + 64 * i + lane;
            if ((j & (tile_rows - 1)) == 0)
                a.tiles[tile0[id[i]] + (j >> a.tile_shift)] = make_int2(id[i] | min(tile_rows, count[id[i]] - j) << 16, p);
        }
    }
}

// ------------------------------------------------------------------- products
struct LoraArgs {
    const void *x;
    const float *x_scales;  // fp8 rows
    int64_t x_stride;
    const void *a, *b;
    const float *scales;  // [adapters] or null
    const int32_t *order;
    const int2 *tiles;
    float *v;  // [splits][rows][v_stride]: part p from p * part_stride on
    void *y;
    int64_t y_stride;
    int rows, adapters, k, n, rank, parts, part_stride, v_stride, splits, blocks, groups;  // blocks: of 64 columns a wave; groups: of workgroups' columns
    int part_end[kMaxParts], part_block;
};

// E values of a row from column c on, as the matrix instruction's operand (16
// bytes of T), zeros from `cols` on: one by one (`take`), or whole (`piece`) where
// E divides the row's length.  No branch around a load (it would
// be waited for before the next): what lies behind the row is read at its end and
// not used.
template <typename T> struct Operand;
template <> struct Operand<uint16_t> {
    static constexpr int E = 8;  // values a lane, 32 a step
    static __device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    }
};
template <> struct Operand<float> {
    static constexpr int E = 4;  // values a lane, 16 a step
    static __device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, f32x4 c) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[i]), __uint_as_float(b[i]), c, 0, 0, 0);
        return c;
    }
};
__device__ __forceinline__ u32x4 take(const uint16_t *row, int c, int cols) {
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i / 2] |= (c + i < cols ? (uint32_t)row[min(c + i, cols - 1)] : 0u) << (16 * (i & 1));
    return w;
}
__device__ __forceinline__ u32x4 take(const float *row, int c, int cols) {
    u32x4 w = {0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = c + i < cols ? __float_as_uint(row[min(c + i, cols - 1)]) : 0u;
    return w;
}
// eight e4m3 values as bf16 (exact)
__device__ __forceinline__ u32x4 operand(const u32x4 &v) { return v; }
__device__ __forceinline__ u32x4 operand(const u32x2 &v) {
    const u32x2 lo = e4m3x4_to_bf16x4(v[0]), hi = e4m3x4_to_bf16x4(v[1]);
    return u32x4{lo[0], lo[1], hi[0], hi[1]};
}
__device__ __forceinline__ u32x4 take(const uint8_t *row, int c, int cols) {
    u32x2 q = {0, 0};
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i / 4] |= (c + i < cols ? (uint32_t)row[min(c + i, cols - 1)] : 0u) << (8 * (i & 3));
    return operand(q);
}
// As they are in memory, for `operand`.  Four lanes of a row ask for 64 bytes of it, half a line, and an
// instruction for halves of 16 lines; so two steps are loaded together, lanes r and r +
// 8 taking the line's pieces of row r in the first and of row r + 8 in the second, and
// change places after (swap8).  Any order of k does as long as A and x share it.
// (8192 x 4096 of rank 32: 21.5 us, 26 with half lines; 32768 rows 79, 93.)
// (Any: at the elements' own alignment, in one instruction all the same.)
template <typename X> struct RawOf;
template <> struct RawOf<uint16_t> {
    typedef u32x4 type;
    typedef u32x4 __attribute__((aligned(2))) Any;
};
template <> struct RawOf<float> {
    typedef u32x4 type;
    typedef u32x4 __attribute__((aligned(4))) Any;
};
template <> struct RawOf<uint8_t> {
    typedef u32x2 type;
    typedef u32x2 __attribute__((aligned(1))) Any;
};
template <typename X>
__device__ __forceinline__ typename RawOf<X>::type piece(const X *row, int c, int cols) {
    typedef typename RawOf<X>::type Raw;
    constexpr int E = sizeof(Raw) / sizeof(X), N = sizeof(Raw) / 4;
    Raw v = *reinterpret_cast<const typename RawOf<X>::Any *>(row + min(c, cols - E));
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = c < cols ? v[i] : 0;
    return v;
}
// Lanes 8 .. 15 of u change places with lanes 0 .. 7 of v, in every row of 16 lanes.
template <typename V>
__device__ __forceinline__ void swap8(V &u, V &v) {
    constexpr int kRotate8 = 0x128;  // row_ror:8
#pragma unroll
    for (int i = 0; i < (int)(sizeof(V) / 4); ++i) {
        const uint32_t a = u[i], b = v[i];
        u[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)a, (int)b, kRotate8, 0xf, 0xc, false);
        v[i] = (uint32_t)__builtin_amdgcn_update_dpp((int)b, (int)a, kRotate8, 0xf, 0x3, false);
    }
}

// Rows of tile `i`: its adapter, first position and count (0: none).
__device__ __forceinline__ int tile_at(const LoraArgs &a, int i, int rows, int &adapter, int &p0) {
    const int2 t = a.tiles[i];
    adapter = t.x & 0xffff;
    p0 = t.y;
    if (t.x < 0 || adapter >= a.adapters || (unsigned)p0 >= (unsigned)a.rows) return 0;
    return min(min(t.x >> 16, rows), a.rows - p0);
}

// v of a tile: MT groups of 16 rows by RT groups of 16 ranks, each wave of the
// workgroup every W-th step of four matrix instructions of its stretch of k.
template <typename X, typename T, int MT, int RT, int W, bool WHOLE>
__global__ void __launch_bounds__(64 * W) lora_shrink_kernel(LoraArgs a) {
    constexpr int E = Operand<T>::E, U = WHOLE ? 4 : 2, kStep = 4 * E * U;
    __shared__ f32x4 sums[W][RT * MT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    int adapter, p0;
    const int count = tile_at(a, blockIdx.x, 16 * MT, adapter, p0);
    if (count == 0) return;
    const int i0 = blockIdx.y * RT * 16, split = blockIdx.z;
    // rows of x and of A: two for a lane's pieces of two steps, or its own
    constexpr int P = WHOLE ? 2 : 1;
    const int r8 = WHOLE ? r16 & 7 : r16;
    const X *xr[MT][P];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int h = 0; h < P; ++h) {
            const int row = a.order[p0 + min(16 * m + 8 * h + r8, count - 1)];
            xr[m][h] = (const X *)a.x + (size_t)min((unsigned)row, (unsigned)a.rows - 1) * a.x_stride;
        }
    // row i of v's values: rank i % part_stride of part i / part_stride (what is behind a part's ranks is not kept)
    const T *ar[RT][P];
#pragma unroll
    for (int f = 0; f < RT; ++f)
#pragma unroll
        for (int h = 0; h < P; ++h) {
            const int i = min(i0 + 16 * f + 8 * h + r8, a.parts * a.part_stride - 1);
            const int part = (i >= a.part_stride) + (i >= 2 * a.part_stride) + (i >= 3 * a.part_stride);  // (of at most 4)
            ar[f][h] = (const T *)a.a + ((size_t)adapter * a.parts * a.rank + part * a.rank + min(i - part * a.part_stride, a.rank - 1)) * a.k;
        }
    f32x4 acc[RT][MT];
#pragma unroll
    for (int f = 0; f < RT; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[f][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int c = (split * W + wave) * kStep; c < a.k; c += a.splits * W * kStep) {
        typedef typename RawOf<X>::type Raw;
        u32x4 av[U][RT];
        std::conditional_t<WHOLE, Raw, u32x4> xv[U][MT];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if constexpr (WHOLE) {
                const int at = c + 4 * E * (u & ~1) + E * (2 * g + (r16 >> 3));
#pragma unroll
                for (int f = 0; f < RT; ++f) av[u][f] = piece(ar[f][u & 1], at, a.k);
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[u][m] = piece(xr[m][u & 1], at, a.k);
            } else {
                const int at = c + 4 * E * u + E * g;
#pragma unroll
                for (int f = 0; f < RT; ++f) av[u][f] = take(ar[f][0], at, a.k);
#pragma unroll
                for (int m = 0; m < MT; ++m) xv[u][m] = take(xr[m][0], at, a.k);
            }
        }
        __builtin_amdgcn_sched_barrier(0);  // (every load before the first product)
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (WHOLE && u % 2 == 0) {
#pragma unroll
                for (int f = 0; f < RT; ++f) swap8(av[u][f], av[u + 1][f]);
#pragma unroll
                for (int m = 0; m < MT; ++m) swap8(xv[u][m], xv[u + 1][m]);
            }
#pragma unroll
            for (int f = 0; f < RT; ++f)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[f][m] = Operand<T>::mfma(av[u][f], operand(xv[u][m]), acc[f][m]);
        }
    }
#pragma unroll
    for (int f = 0; f < RT; ++f)
#pragma unroll
        for (int m = 0; m < MT; ++m) sums[wave][f * MT + m][lane] = acc[f][m];
    __syncthreads();
    const float scale = a.scales ? a.scales[adapter] : 1.0f;
    for (int j = wave; j < RT * MT; j += W) {
        const int f = j / MT, row = 16 * (j % MT) + r16, i = i0 + 16 * f + 4 * g;
        if (row >= count || i >= a.v_stride) continue;
        f32x4 v = sums[0][j][lane];
#pragma unroll
        for (int w = 1; w < W; ++w) v += sums[w][j][lane];
        float s = scale;
        if (sizeof(X) == 1) s *= a.x_scales[min((unsigned)a.order[p0 + row], (unsigned)a.rows - 1)];
        v *= s;
        *reinterpret_cast<f32x4 *>(a.v + ((size_t)split * a.rows + p0 + row) * a.v_stride + i) = v;
    }
}

__device__ __forceinline__ int part_of(const LoraArgs &a, int col) {
    if (a.part_block) return (col / a.part_block) % a.parts;
    int p = 0;
#pragma unroll
    for (int i = 0; i < kMaxParts - 1; ++i) p += i < a.parts - 1 && col >= a.part_end[i];
    return p;
}

// two values as bf16, to nearest even (one instruction)
__device__ __forceinline__ uint32_t two(float lo, float hi) {
    typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{lo, hi}, bf16x2_t));
}

// E values of v's row from rank r on, as operands: f32 as they are; for bf16 each
// as two, which together hold 16 bits of it, so that the sum keeps what f32 v has
// over one rounding to 8.
template <typename T> struct Values;
template <> struct Values<float> {
    static constexpr int H = 1;
    static __device__ __forceinline__ void split(const float (&v)[4], u32x4 (&o)[1]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[0][i] = __float_as_uint(v[i]);
    }
};
template <> struct Values<uint16_t> {
    static constexpr int H = 2;
    static __device__ __forceinline__ void split(const float (&v)[8], u32x4 (&o)[2]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t w = two(v[2 * i], v[2 * i + 1]);
            o[0][i] = w;
            // (nothing is left of a value that has no finite first half)
            const float a = bf16lo(w), b = bf16hi(w);
            o[1][i] = two((w & 0x7f80u) == 0x7f80u ? 0.0f : v[2 * i] - a, (w & 0x7f800000u) == 0x7f800000u ? 0.0f : v[2 * i + 1] - b);
        }
    }
};

// y of a tile and a workgroup's columns, 64 of every 256 a wave: workgroups that
// follow one another, and the waves of one, write the same rows side by side.  The
// values of the parts that these columns meet are summed over the splits into LDS
// first, then each wave works alone: a block of y is asked for before the product
// that is added to it.  ONE: no block of 64 columns meets two parts; else each gets the
// product of every part that it meets, and keeps its columns' (8192 x 28672 in two parts by
// 16 columns in turn, rank 16, 362 us for both launches, in two halves 198).  What bounds it
// is y's way there and back (8192 x 4096 of rank 32: 34 us, 3.9 TB/s; 28672 columns 4.6).
template <typename T, int MT, bool WHOLE, bool ONE>
__global__ void __launch_bounds__(256) lora_expand_kernel(LoraArgs a) {
    constexpr int E = Operand<T>::E, kStep = 4 * E, H = Values<T>::H;
    extern __shared__ f32x4 lds[];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r16 = lane & 15, g = lane >> 4;
    int adapter, p0;
    const int count = tile_at(a, blockIdx.x / a.groups, 16 * MT, adapter, p0);
    if (count == 0) return;
    const int steps = (a.rank + kStep - 1) / kStep;
    const int begin = blockIdx.x % a.groups * a.blocks * 256, end = min(begin + a.blocks * 256, a.n);
    // rows of y (from a.rows on: none), a lane's own and those whose lines it asks for
    unsigned row[MT], line_row[MT][2];
    const int r8 = r16 & 7, half = r16 >> 3;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        row[m] = 16 * m + r16 < count ? (unsigned)a.order[p0 + 16 * m + r16] : ~0u;
#pragma unroll
        for (int h = 0; h < 2; ++h) line_row[m][h] = 16 * m + 8 * h + r8 < count ? (unsigned)a.order[p0 + 16 * m + 8 * h + r8] : ~0u;
    }
    // values: rows of `line` 16-byte units, one spare against bank conflicts
    int part0 = 0, part1 = a.parts - 1;
    if (!a.part_block) {
        part0 = part_of(a, begin);
        part1 = part_of(a, end - 1);
    }
    const int units = (part1 + 1 - part0) * (a.part_stride / 4), line = units + 1;
    {
        const float *src = a.v + (size_t)p0 * a.v_stride + part0 * a.part_stride;
        const size_t plane = (size_t)a.rows * a.v_stride;
        for (int i = threadIdx.x; i < 16 * MT * units; i += 256) {
            const int r = i / units, u = i - r * units;
            if (r >= count) break;
            const float *at = src + (size_t)r * a.v_stride + 4 * u;
            f32x4 v = *reinterpret_cast<const f32x4 *>(at);
#pragma unroll 4
            for (int q = 1; q < a.splits; ++q) v += *reinterpret_cast<const f32x4 *>(at + q * plane);
            lds[r * line + u] = v;
        }
    }
    __syncthreads();
    auto values = [&](int part, int s, u32x4 (&o)[MT][H]) {
        const int r = s * kStep + E * g;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            float v[E];
            const f32x4 *src = lds + min(16 * m + r16, count - 1) * line + (part - part0) * (a.part_stride / 4);
#pragma unroll
            for (int i = 0; i < E; i += 4) {
                const f32x4 w = src[min(r + i, a.part_stride - 4) / 4];
#pragma unroll
                for (int e = 0; e < 4; ++e) v[i + e] = r + i + e < a.rank ? w[e] : 0.0f;
            }
            Values<T>::split(v, o[m]);
        }
    };
    // Columns n1 = n0 + 32 q + 8 g .. + 7 of row r16 of each group, whole pieces.  (No branch around a load: lanes that have
    // none read another.)  bf16: of 64 columns that y has, eight lanes ask for a row's line and give it back, as the shrink's
    // do; between, a lane has its row's pieces (32768 x 4096 of rank 32: 102 us, 110 with half lines).
    typedef u32x4 Pieces[MT][2][H == 2 ? 1 : 2];
    typedef typename RawOf<T>::Any Any;
    const bool pieces = a.n >= 8;
    const unsigned any = (unsigned)min((unsigned)a.order[p0], (unsigned)a.rows - 1);
    auto lines = [&](int n0) { return H == 2 && pieces && n0 + 64 <= a.n; };
    auto ask = [&](int n0, Pieces &had) {
        if (!pieces) return;
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const unsigned r = lines(n0) ? line_row[m][q] : row[m];
                const int n1 = lines(n0) ? n0 + 8 * g + 32 * half : min(n0 + 32 * q + 8 * g, (a.n - 8) & ~7);
                const T *y = (const T *)a.y + (size_t)(r < (unsigned)a.rows ? r : any) * a.y_stride + n1;
#pragma unroll
                for (int i = 0; i < (H == 2 ? 1 : 2); ++i) had[m][q][i] = reinterpret_cast<const Any *>(y)[i];
            }
    };
    auto give = [&](int n0, Pieces &had, const f32x4 (&acc)[4][MT]) {
        auto d = [&](int m, int q, int i) { return acc[2 * q + i / 4][m][i % 4]; };
        auto add = [&](u32x4 &w, int m, int q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = two(bf16lo(w[i]) + d(m, q, 2 * i), bf16hi(w[i]) + d(m, q, 2 * i + 1));
        };
        if (lines(n0)) {
#pragma unroll
            for (int m = 0; m < MT; ++m) {
                swap8(had[m][0][0], had[m][1][0]);
                add(had[m][0][0], m, 0);
                add(had[m][1][0], m, 1);
                swap8(had[m][0][0], had[m][1][0]);
#pragma unroll
                for (int h = 0; h < 2; ++h)
                    if (line_row[m][h] < (unsigned)a.rows)
                        *reinterpret_cast<Any *>((T *)a.y + (size_t)line_row[m][h] * a.y_stride + n0 + 8 * g + 32 * half) = had[m][h][0];
            }
            return;
        }
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            if (row[m] >= (unsigned)a.rows) continue;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int n1 = n0 + 32 * q + 8 * g;
                T *y = (T *)a.y + (size_t)row[m] * a.y_stride + n1;
                if (n1 + 8 <= a.n && pieces) {
                    Any *yw = reinterpret_cast<Any *>(y);
                    if constexpr (H == 2) {
                        add(had[m][q][0], m, q);
                        yw[0] = had[m][q][0];
                    } else {
#pragma unroll
                        for (int i = 0; i < 2; ++i) {
                            u32x4 w = had[m][q][i];
#pragma unroll
                            for (int e = 0; e < 4; ++e) w[e] = __float_as_uint(__uint_as_float(w[e]) + d(m, q, 4 * i + e));
                            yw[i] = w;
                        }
                    }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (n1 + i < a.n) {
                            if constexpr (H == 2) y[i] = (T)two(__uint_as_float((uint32_t)y[i] << 16) + d(m, q, i), 0.0f);
                            else y[i] += d(m, q, i);
                        }
                }
            }
        }
    };
    u32x4 kept[MT][H];  // of one step's ranks, over the blocks of a part
    int kept_part = -1;
    for (int n0 = begin + wave * 64; n0 < end; n0 += 256) {
        Pieces had;
        ask(n0, had);
        // row r16 of B tile t: column n0 + 32 (t / 2) + 8 (r16 / 4) + 4 (t % 2) + r16 % 4
        const T *bb[4];
#pragma unroll
        for (int t = 0; t < 4; ++t)
            bb[t] = (const T *)a.b + ((size_t)adapter * a.n + min(n0 + 32 * (t >> 1) + 8 * (r16 >> 2) + 4 * (t & 1) + (r16 & 3), a.n - 1)) * a.rank;
        // the product of these columns with part p's values
        auto product = [&](int p, f32x4 (&acc)[4][MT]) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
#pragma unroll
                for (int m = 0; m < MT; ++m) acc[t][m] = f32x4{0.f, 0.f, 0.f, 0.f};
            for (int s = 0; s < steps; ++s) {
                u32x4 bv[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    if constexpr (WHOLE) bv[t] = piece(bb[t], s * kStep + E * g, a.rank);
                    else bv[t] = take(bb[t], s * kStep + E * g, a.rank);
                }
                if (steps > 1 || kept_part != p) {
                    values(p, s, kept);
                    kept_part = p;
                }
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int h = 0; h < H; ++h)
#pragma unroll
                        for (int t = 0; t < 4; ++t) acc[t][m] = Operand<T>::mfma(bv[t], kept[m][h], acc[t][m]);
            }
        };
        f32x4 acc[4][MT];
        if (ONE) {
            product(part_of(a, n0), acc);
        } else {  // columns of several parts: each takes its own part's product
            const int lo = a.part_block ? 0 : part_of(a, n0), hi = a.part_block ? a.parts - 1 : part_of(a, min(n0 + 63, a.n - 1));
            product(lo, acc);
            f32x4 one[4][MT];
            for (int p = lo + 1; p <= hi; ++p) {
                product(p, one);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool mine = part_of(a, min(n0 + 32 * (t >> 1) + 8 * g + 4 * (t & 1) + e, a.n - 1)) == p;
#pragma unroll
                        for (int m = 0; m < MT; ++m) acc[t][m][e] = mine ? one[t][m][e] : acc[t][m][e];
                    }
            }
        }
        give(n0, had, acc);
    }
}

int part_stride_of(int rank) { return (rank + 3) / 4 * 4; }
int v_stride_of(int rank, int parts) { return (part_stride_of(rank) * parts + 15) / 16 * 16; }
int rank_groups(int v_stride) { return v_stride <= 64 ? v_stride / 16 : 4; }  // of 16, a workgroup
// Workgroups of k of one tile and rank group: enough of them for two a CU (prompts:
// one, of twice the waves), a wave at least one step.  (64 rows of k 14336 11.2 us, for
// one a CU 11.9, for four 11.3; 8192 rows 57.7, for two a CU 58.7, for four 62.)
int splits_of(int64_t rows, int64_t adapters, int64_t k, int rank, int parts, zk_dtype dtype) {
    const int vs = v_stride_of(rank, parts), rt = rank_groups(vs), waves = tile_rows_for(rows) == 16 ? 4 : 8;
    const int64_t tiles = std::max<int64_t>(1, max_tiles(rows, adapters)) * ((vs / 16 + rt - 1) / rt);
    const int64_t most = std::max<int64_t>(1, k / (waves * (dtype == ZK_F32 ? 64 : 128)));
    const int64_t want = ((waves == 4 ? 512 : 256) + tiles - 1) / tiles;
    return (int)std::min<int64_t>({most, want, 16});
}

bool meet(const void *p, int64_t pb, const void *q, int64_t qb) {
    const uintptr_t a = (uintptr_t)p, b = (uintptr_t)q;
    return p && q && pb > 0 && qb > 0 && a < b + qb && b < a + pb;
}
int bad(const char *what) { return set_error(ZK_ERR_INVALID_ARGUMENT, std::string("Internal error: ") + what); }
bool aligned(const void *p, int b) { return ((uintptr_t)p & (uintptr_t)(b - 1)) == 0; }

bool shape_ok(int64_t rows, int64_t adapters, int64_t k, int rank, int parts) {
    return rows >= 0 && rows <= (1 << 24) && adapters >= 1 && adapters <= kMaxAdapters && k >= 1 && k <= (1 << 23) && rank >= 1 &&
           rank <= kMaxRank && parts >= 1 && parts <= kMaxParts && rank * parts <= kMaxRanks;
}

template <typename X, typename T, int MT>
void shrink(const LoraArgs &a, int tiles, bool whole, hipStream_t s) {
    constexpr int W = MT == 1 ? 4 : 8;
    const int rt = rank_groups(a.v_stride), groups = (a.v_stride / 16 + rt - 1) / rt;
    const dim3 grid((unsigned)tiles, (unsigned)groups, (unsigned)a.splits);
    auto go = [&](auto kernel) { kernel<<<grid, 64 * W, 0, s>>>(a); };
    if (rt == 1) whole ? go(lora_shrink_kernel<X, T, MT, 1, W, true>) : go(lora_shrink_kernel<X, T, MT, 1, W, false>);
    else if (rt == 2) whole ? go(lora_shrink_kernel<X, T, MT, 2, W, true>) : go(lora_shrink_kernel<X, T, MT, 2, W, false>);
    else if (rt == 3) whole ? go(lora_shrink_kernel<X, T, MT, 3, W, true>) : go(lora_shrink_kernel<X, T, MT, 3, W, false>);
    else whole ? go(lora_shrink_kernel<X, T, MT, 4, W, true>) : go(lora_shrink_kernel<X, T, MT, 4, W, false>);
}

template <typename T, int MT>
void expand(LoraArgs a, int tiles, hipStream_t s) {
    constexpr int E = Operand<T>::E;
    const bool whole = a.rank % E == 0;
    bool one = a.part_block % 64 == 0;
    for (int i = 0; i < a.parts - 1 && !a.part_block; ++i) one = one && a.part_end[i] % 64 == 0;
    // Blocks of 64 columns a wave: values are summed and split once for them, as long as
    // 16384 waves are left (with 4096: 32768 rows x 4096 223 us for 199, 8192 x 28672 262 for 235).
    const int all = (a.n + 63) / 64;
    a.blocks = (int)std::max<int64_t>(1, std::min<int64_t>(4, (int64_t)tiles * all / 16384));
    a.groups = (all + 4 * a.blocks - 1) / (4 * a.blocks);
    const dim3 grid((unsigned)tiles * (unsigned)a.groups);
    const size_t bytes = (size_t)16 * MT * (a.parts * (a.part_stride / 4) + 1) * 16;
    auto go = [&](auto kernel) {
        if (bytes > 65536) (void)hipFuncSetAttribute((const void *)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
        kernel<<<grid, 256, bytes, s>>>(a);
    };
    if (one) whole ? go(lora_expand_kernel<T, MT, true, true>) : go(lora_expand_kernel<T, MT, false, true>);
    else whole ? go(lora_expand_kernel<T, MT, true, false>) : go(lora_expand_kernel<T, MT, false, false>);
}

template <typename X, typename T>
void both(const LoraArgs &a, int tiles, hipStream_t s) {
    constexpr int E = Operand<T>::E;
    const bool whole = a.k % E == 0;
    if (tile_rows_for(a.rows) == 16) {
        shrink<X, T, 1>(a, tiles, whole, s);
        expand<T, 1>(a, tiles, s);
    } else {
        shrink<X, T, 2>(a, tiles, whole, s);
        expand<T, 2>(a, tiles, s);
    }
}

}  // namespace

extern "C" {

int64_t zk_lora_max_tiles(int64_t num_rows, int64_t num_adapters) {
    if (num_rows <= 0 || num_rows > (1 << 24) || num_adapters <= 0 || num_adapters > kMaxAdapters) return 0;
    return max_tiles(num_rows, num_adapters);
}

int zk_lora_plan(const int32_t *adapter_ids, int64_t num_rows, int64_t num_adapters, int32_t *order, int32_t *offsets,
                 int32_t *tiles, void *stream) {
    if (num_rows < 0 || num_rows > (1 << 24) || num_adapters <= 0 || num_adapters > kMaxAdapters)
        return bad("zk_lora_plan: bad shape (at most 2^24 rows and 2048 adapters)");
    if (!offsets || (num_rows > 0 && (!adapter_ids || !order || !tiles))) return bad("zk_lora_plan: NULL pointer");
    if (!aligned(tiles, 8)) return bad("zk_lora_plan: tiles must be 8-byte aligned");
    const int64_t nt = num_rows ? max_tiles(num_rows, num_adapters) : 0;
    const struct {
        const void *p;
        int64_t bytes;
    } all[] = {{order, 4 * num_rows}, {offsets, 4 * (num_adapters + 1)}, {tiles, 8 * nt}, {adapter_ids, 4 * num_rows}};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 4; ++j)
            if (meet(all[i].p, all[i].bytes, all[j].p, all[j].bytes)) return bad("zk_lora_plan: operands overlap");
    PlanArgs a{};
    a.ids = adapter_ids;
    a.order = order;
    a.offsets = offsets;
    a.tiles = (int2 *)tiles;
    a.rows = (int)num_rows;
    a.adapters = (int)num_adapters;
    while ((1 << a.bits) < num_adapters) ++a.bits;
    a.tile_shift = tile_rows_for(num_rows) == 16 ? 4 : 5;
    a.max_tiles = (int)nt;
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("lora_plan", s);
    lora_plan_kernel<<<1, 1024, 0, s>>>(a);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_lora_plan: ") + hipGetErrorString(e));
    return ZK_OK;
}

size_t zk_lora_workspace_size(int64_t num_rows, int64_t num_adapters, int64_t k, int rank, int num_parts, zk_dtype dtype) {
    if (!shape_ok(num_rows, num_adapters, k, rank, num_parts) || num_rows == 0) return 0;
    return (size_t)splits_of(num_rows, num_adapters, k, rank, num_parts, dtype) * num_rows * v_stride_of(rank, num_parts) * 4;
}

int zk_lora(const void *x, const float *x_scales, int64_t x_stride, zk_dtype x_dtype, const void *a_weights,
            const void *b_weights, const float *scales, zk_dtype dtype, const int32_t *order,
            const int32_t *tiles, int64_t num_rows, int64_t num_adapters, int64_t k, int64_t n, int rank, int num_parts,
            const int64_t *part_cols, int part_block, void *y, int64_t y_stride, void *workspace, size_t workspace_bytes,
            void *stream) {
    if (dtype != ZK_F32 && dtype != ZK_BF16) return bad("zk_lora: the weights and y must be f32 or bf16");
    if (x_dtype != dtype && !(x_dtype == ZK_FP8_E4M3 && dtype == ZK_BF16))
        return bad("zk_lora: x must have the weights' type, or be fp8 beside bf16 weights");
    if ((x_dtype == ZK_FP8_E4M3) != (x_scales != nullptr)) return bad("zk_lora: x_scales go with fp8 rows");
    if (!shape_ok(num_rows, num_adapters, k, rank, num_parts) || n <= 0 || n > (1 << 23) || part_block < 0)
        return bad("zk_lora: bad shape (ranks of a part at most 256, of all parts 512, at most 4 parts and 2048 adapters)");
    if (x_stride == 0) x_stride = k;
    if (y_stride == 0) y_stride = n;
    if (x_stride < k || y_stride < n || x_stride > (1ll << 31) || y_stride > (1ll << 31)) return bad("zk_lora: bad row stride");
    LoraArgs a{};
    if (part_block) {
        if (n % ((int64_t)part_block * num_parts)) return bad("zk_lora: the columns must be whole rounds of the parts' blocks");
    } else if (num_parts > 1) {
        if (!part_cols) return bad("zk_lora: part_cols missing");
        int64_t end = 0;
        for (int i = 0; i < num_parts; ++i) {
            if (part_cols[i] <= 0 || part_cols[i] > n) return bad("zk_lora: parts must hold the columns of y");
            end += part_cols[i];
            a.part_end[i] = (int)std::min(end, n);
        }
        if (end != n) return bad("zk_lora: parts must hold the columns of y");
    }
    if (num_rows == 0) return ZK_OK;
    if (!x || !a_weights || !b_weights || !order || !tiles || !y) return bad("zk_lora: NULL pointer");
    const size_t need = zk_lora_workspace_size(num_rows, num_adapters, k, rank, num_parts, dtype);
    if (!workspace || workspace_bytes < need) return bad("zk_lora: workspace too small (zk_lora_workspace_size)");
    if (!aligned(workspace, 16) || !aligned(tiles, 8)) return bad("zk_lora: the workspace must be 16-byte, tiles 8-byte aligned");
    const int e = elt_size(dtype), ranks = rank * num_parts;
    const int64_t nt = max_tiles(num_rows, num_adapters);
    if (nt * ((n + 1023) / 1024) > 0x7fffffff) return bad("zk_lora: more rows of y than a launch takes");
    const int64_t xb = ((num_rows - 1) * x_stride + k) * elt_size(x_dtype), yb = ((num_rows - 1) * y_stride + n) * e;
    const struct {
        const void *p;
        int64_t bytes;
    } in[] = {{x, xb}, {x_scales, 4 * num_rows}, {a_weights, num_adapters * ranks * k * e}, {b_weights, num_adapters * n * rank * e},
              {scales, 4 * num_adapters}, {order, 4 * num_rows}, {tiles, 8 * nt}};
    for (const auto &i : in)
        if (meet(i.p, i.bytes, y, yb) || meet(i.p, i.bytes, workspace, (int64_t)need)) return bad("zk_lora: y or the workspace overlaps an input");
    if (meet(y, yb, workspace, (int64_t)need)) return bad("zk_lora: y overlaps the workspace");
    a.x = x;
    a.x_scales = x_scales;
    a.x_stride = x_stride;
    a.a = a_weights;
    a.b = b_weights;
    a.scales = scales;
    a.order = order;
    a.tiles = (const int2 *)tiles;
    a.v = (float *)workspace;
    a.y = y;
    a.y_stride = y_stride;
    a.rows = (int)num_rows;
    a.adapters = (int)num_adapters;
    a.k = (int)k;
    a.n = (int)n;
    a.rank = rank;
    a.parts = num_parts;
    a.part_stride = part_stride_of(rank);
    a.v_stride = v_stride_of(rank, num_parts);
    a.splits = splits_of(num_rows, num_adapters, k, rank, num_parts, dtype);
    a.part_block = part_block;
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("lora", s);
    if (dtype == ZK_F32) both<float, float>(a, (int)nt, s);
    else if (x_dtype == ZK_BF16) both<uint16_t, uint16_t>(a, (int)nt, s);
    else both<uint8_t, uint16_t>(a, (int)nt, s);
    if (hipError_t er = hipGetLastError(); er != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_lora: ") + hipGetErrorString(er));
    return ZK_OK;
}

}  // extern "C"
