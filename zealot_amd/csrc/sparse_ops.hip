// sparse_ops.hip -- the selection side of sparse decode attention over pages:
// bounds of each page's keys, an upper bound of a page's logits from them, and
// the best pages of each (sequence, kv-head).  paged_sparse.hip attends them.
// No reference counterpart (its decode reads every page,
// src/attention/kernels/paged_attention.cu:65-131).
//
// bounds[b][h][0][d] = min, [1][d] = max over the page's tokens of K[.., d], in
// the pool's type (exact: a bound is one of the keys' values).
// For any key k of page p and query q:
//   q . k = sum_d q_d k_d <= sum_d max(q_d lo_d, q_d hi_d)
//         = sum_d min(q_d, 0) lo_d + max(q_d, 0) hi_d,
// the last form a product of 2 D terms, which runs on the matrix cores.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "attn_device.h"
#include "zk_common.h"

using namespace zk;

namespace {

constexpr int kThreads = 256;

int check_launch(const char *what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: ") + what + ": " + hipGetErrorString(e));
    return ZK_OK;
}

// ------------------------------------------------------------ page bounds
// One 16-byte piece of a row as f32 values (VEC), or one element.
template <int KV, bool VEC> struct Piece;
template <bool VEC> struct Piece<ZK_F32, VEC> {
    static constexpr int N = VEC ? 4 : 1;
    typedef typename std::conditional<VEC, u32x4, uint32_t>::type raw_t;
    static __device__ __forceinline__ void unpack(raw_t v, float *x) {
        if constexpr (VEC) {
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = __uint_as_float(v[e]);
        } else {
            x[0] = __uint_as_float(v);
        }
    }
    static __device__ __forceinline__ raw_t pack(const float *x) {
        if constexpr (VEC) return u32x4{__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3])};
        else return __float_as_uint(x[0]);
    }
};
template <bool VEC> struct Piece<ZK_BF16, VEC> {
    static constexpr int N = VEC ? 8 : 1;
    typedef typename std::conditional<VEC, u32x4, uint16_t>::type raw_t;
    static __device__ __forceinline__ void unpack(raw_t v, float *x) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                x[2 * i] = bf16lo(v[i]);
                x[2 * i + 1] = bf16hi(v[i]);
            }
        } else {
            x[0] = __uint_as_float((uint32_t)v << 16);
        }
    }
    static __device__ __forceinline__ raw_t pack(const float *x) {  // (bf16 values: the high halves)
        if constexpr (VEC) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                v[i] = __builtin_amdgcn_perm(__float_as_uint(x[2 * i + 1]), __float_as_uint(x[2 * i]), 0x07060302u);
            return v;
        } else {
            return (uint16_t)(__float_as_uint(x[0]) >> 16);
        }
    }
};
template <bool VEC> struct Piece<ZK_FP8_E4M3, VEC> {
    static constexpr int N = VEC ? 16 : 1;
    typedef typename std::conditional<VEC, u32x4, uint8_t>::type raw_t;
    static __device__ __forceinline__ void unpack(raw_t v, float *x) {
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < 4; ++i) e4m3x4_to_f32(v[i], x + 4 * i);
        } else {
            float t[4];
            e4m3x4_to_f32(v, t);
            x[0] = t[0];
        }
    }
    static __device__ __forceinline__ raw_t pack(const float *x) {
        if constexpr (VEC) {
            u32x4 v;
#pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = e4m3x4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
            return v;
        } else {
            return (uint8_t)e4m3x4(x[0], 0.f, 0.f, 0.f);
        }
    }
};
template <int KV, bool VEC>
struct Rows : Piece<KV, VEC> {
    typedef Piece<KV, VEC> B;
    static __device__ __forceinline__ typename B::raw_t fetch(const char *p) { return *(const typename B::raw_t *)p; }
    static __device__ __forceinline__ void load(const char *p, float *x) { B::unpack(fetch(p), x); }
    static __device__ __forceinline__ void store(char *p, const float *x) { *(typename B::raw_t *)p = B::pack(x); }
};

// NaN once seen stays: a page with such a key has NaN bounds (v_minimum3_f32).
__device__ __forceinline__ float min_nan(float a, float b) { return __builtin_elementwise_minimum(a, b); }
__device__ __forceinline__ float max_nan(float a, float b) { return __builtin_elementwise_maximum(a, b); }

// A workgroup looks at `rows` rows of the slot map (one wave's load of 64 slots
// tells where runs begin and how far they go).  The row that is the first of its
// page's run (consecutive rows with consecutive slots of one block) folds the
// run's keys, and the page's bounds from before unless the run begins the page.
// A thread holds a 16-byte piece of a token's heads, 16 tokens of it in flight.
// Bound by HBM for prompts (26000 tokens, 8 heads of 128 bf16, 63 MB: 12.8 us, 4.9 TB/s; with one
// row after the other 23.6), by
// latency for a decode step's single tokens.
template <int KV, bool VEC>
__global__ void __launch_bounds__(kThreads)
page_bounds_kernel(const char *__restrict__ k_pool, const int64_t *__restrict__ slots, int64_t num_tokens, int rows,
                   int hkv, int head_dim, int block_size, int64_t num_slots, char *__restrict__ bounds) {
    typedef Rows<KV, VEC> P;
    constexpr int N = P::N, ES = KV == ZK_F32 ? 4 : KV == ZK_BF16 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int ppr = head_dim / N, pieces = hkv * ppr;
    // Workgroups go to the 8 XCDs in turn, and of a prompt's only those work where a page
    // begins: an XCD takes the rows of 16 tokens in a row (2000 rows of one prompt 7.5 us
    // in order, which one XCD has alone, 6.2)
    const int bx = blockIdx.x, per = 16 / rows, span = 8 * per;
    const int group = (bx | (span - 1)) < (int)gridDim.x ? (bx & ~(span - 1)) | (bx & 7) * per | (bx >> 3 & (per - 1)) : bx;
    const int64_t t0 = (int64_t)group * rows;
    // lane i: row t0 - 1 + i
    const int64_t t = t0 - 1 + lane;
    const int64_t slot = t >= 0 && t < num_tokens ? slots[t] : -2;
    const int64_t prev = __shfl_up(slot, 1);
    const bool valid = slot >= 0 && slot < num_slots;
    const int64_t blk = valid ? slot / block_size : 0;
    const int tib = valid ? (int)(slot - blk * block_size) : 0;
    const uint64_t inside = __builtin_amdgcn_ballot_w64(lane > 0 && valid && tib > 0 && slot == prev + 1);
    uint64_t heads = __builtin_amdgcn_ballot_w64(lane > 0 && lane <= rows && valid) & ~inside;
    for (; heads; heads &= heads - 1) {
        const int i = __builtin_ctzll(heads);
        const int64_t s0 = __shfl(slot, i), b = __shfl(blk, i);
        const int first = __shfl(tib, i);
        int run = 1;
        const uint64_t after = i == 63 ? 0 : inside >> (i + 1);
        run += __builtin_ctzll(~after);  // (a run's rows after its first; `after` has a clear top bit)
        while (i + run >= 64 && run < block_size - first) {  // past the rows that the wave holds
            const int j = run + lane;
            const int64_t r = t0 - 1 + i + j;
            const bool on = j < block_size - first && r < num_tokens && slots[r] == s0 + j;
            const uint64_t off = ~__builtin_amdgcn_ballot_w64(on);
            run += off ? (int)__builtin_ctzll(off) : 64;
            if (off) break;
        }
        for (int x = threadIdx.x; x < pieces; x += blockDim.x) {
            const int h = x / ppr, c = x - h * ppr;
            const size_t row_bytes = (size_t)head_dim * ES;
            const char *src = k_pool + (((size_t)b * hkv + h) * block_size + first) * row_bytes + (size_t)c * N * ES;
            char *dst = bounds + ((size_t)b * hkv + h) * 2 * row_bytes + (size_t)c * N * ES;
            float lo[N], hi[N];
            if (first) {
                P::load(dst, lo);
                P::load(dst + row_bytes, hi);
            } else {
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    lo[e] = INFINITY;
                    hi[e] = -INFINITY;
                }
            }
            auto fold = [&]<int F>(int j0) {  // F rows, the run's last again past its end
                typename P::raw_t raw[F];
#pragma unroll
                for (int j = 0; j < F; ++j) raw[j] = P::fetch(src + (size_t)min(j0 + j, run - 1) * row_bytes);
#pragma unroll
                for (int j = 0; j < F; ++j) {
                    float v[N];
                    P::unpack(raw[j], v);
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        lo[e] = min_nan(lo[e], v[e]);
                        hi[e] = max_nan(hi[e], v[e]);
                    }
                }
            };
            if (run == 1) fold.template operator()<1>(0);
            else if (run <= 4) fold.template operator()<4>(0);
            else
                for (int j0 = 0; j0 < run; j0 += 16) fold.template operator()<16>(j0);
            P::store(dst, lo);
            P::store(dst + row_bytes, hi);
        }
    }
}

// ------------------------------------------------------------ page scores
struct ScoreArgs {
    const void *q;
    const char *bounds;
    const int32_t *tables, *seq_lens;
    float *scores;  // [N][Hkv][max_blocks]
    int64_t num_blocks;
    int num_heads, num_kv_heads, head_dim, block_size, max_blocks, grouped, q_f32;
    int tiles;  // of 16 pages a wave (at most kScoreTiles)
};
constexpr int kScoreTiles = 24, kScoreHeads = 2;  // most tiles a wave, waves (kv-heads) a workgroup
constexpr int kMostPages = 65535 * 16 * kScoreTiles;  // of a context, by the grid

// Pages that a length holds, at most `most`.
__device__ __forceinline__ int held_pages(int len, int block_size, int most) {
    return len <= 0 ? 0 : (int)min((uint32_t)(len - 1) / (uint32_t)block_size + 1u, (uint32_t)most);
}
__device__ __forceinline__ int qhead(const ScoreArgs &a, int kvh, int j, int G) {
    return a.grouped ? kvh * G + j : kvh + j * a.num_kv_heads;
}

// A = 16 pages' [lo | hi] rows, B = the query heads' [min(q, 0) | max(q, 0)], on
// v_mfma_f32_16x16x32_bf16 (bf16 queries on bf16 or fp8 bounds: both exact in bf16,
// the sums in f32) or v_mfma_f32_16x16x4_f32 (f32 bounds).  One wave per (16 *
// tiles pages, kv-head, sequence).  A page's row of 2 D values is contiguous, the
// rows of a tile lie anywhere: the wave loads whole rows, one tile ahead where its
// registers allow, and turns them into fragments through LDS, rows 16 bytes
// longer than they are so that 16 of them do not meet in a bank.  Columns past
// the G heads repeat them, which leaves the maximum over the heads as it is.
//
// 256 contexts of 512 to 8192 tokens, 32 / 8 heads of 128 bf16 (271 MB): 54 us, 5.0
// TB/s; on contexts of one length 5.7 TB/s (a plain read of such rows: 6.6).  Loaded by
// the lanes that need them, 64 bytes of 16 rows an instruction, the lines were
// fetched twice: 83 us.
template <int KV, int D>
__global__ void __launch_bounds__(64 * kScoreHeads) page_scores_mfma_kernel(ScoreArgs a) {
    constexpr bool F32 = KV == ZK_F32;
    constexpr int ES = F32 ? 4 : KV == ZK_BF16 ? 2 : 1, RB = 2 * D * ES;
    constexpr int CPR = RB / 16, LDR = RB + 16;     // 16-byte chunks of a row, its bytes in LDS
    constexpr int LPT = 16 * RB / 1024;             // loads a tile
    constexpr int QN = F32 ? CPR / 4 : 2 * D / 32;  // query pieces: 4 f32, 8 bf16 dims
    static_assert(16 * RB % 1024 == 0 && CPR % 4 == 0, "row shape");
    extern __shared__ __attribute__((aligned(16))) char dyn[];  // a tile a wave
    __shared__ int32_t ids[16 * kScoreTiles];
    __shared__ float found[kScoreHeads][16 * kScoreTiles];
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4, wave = threadIdx.x >> 6;
    // Consecutive workgroups go to the XCDs in turn: the kv-heads first, so that a block's
    // rows are not asked for by one XCD at a time (256 contexts 56 us with the sequences
    // first, 54; 64 of f32 39, 34), chunks last, as a sequence's later ones are often
    // behind its context, and a sequence's chunks in other places of their turns, so that a
    // long context has all XCDs
    const int kvh = blockIdx.x * (blockDim.x >> 6) + wave;
    const int n = (int)(gridDim.y & 1 ? blockIdx.y : (blockIdx.y + blockIdx.z) % gridDim.y);
    const int held = held_pages(a.seq_lens[n], a.block_size, a.max_blocks);
    const int32_t *row = a.tables + (size_t)n * a.max_blocks;
    const int p0 = blockIdx.z * 16 * a.tiles, p1 = min(p0 + 16 * a.tiles, a.max_blocks);
    const int live = min(p1, held) - p0;  // pages here that the sequence holds
    for (int i = threadIdx.x; i < 16 * a.tiles; i += blockDim.x) {
        const int id = i < live ? row[p0 + i] : -1;
        ids[i] = id < a.num_blocks ? id : -1;
    }
    __syncthreads();
    if (kvh >= a.num_kv_heads) return;
    float *out = a.scores + ((size_t)n * a.num_kv_heads + kvh) * a.max_blocks + p0;
    for (int p = max(live, 0) + lane; p < p1 - p0; p += 64) out[p] = -INFINITY;  // behind the context
    if (live <= 0) return;
    // The query's piece i meets dims d .. of the row [lo | hi]: the negative
    // values (by sign bit; a NaN goes into the half of its sign) of dims d .. below D,
    // the others of d - D .. from there.
    const int G = a.num_heads / a.num_kv_heads;
    const size_t q0 = ((size_t)n * a.num_heads + qhead(a, kvh, col % G, G)) * D;
    u32x4 qf[QN];
#pragma unroll
    for (int i = 0; i < QN; ++i) {
        const int d = F32 ? 16 * i + 4 * grp : KV == ZK_BF16 ? 32 * i + 8 * grp : 64 * (i / 2) + 16 * grp + 8 * (i % 2);
        const bool hi = d >= D;
        const size_t at = q0 + (hi ? d - D : d);
        u32x4 w;
        if constexpr (F32) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                w[e] = a.q_f32 ? __float_as_uint(((const float *)a.q)[at + e]) : (uint32_t)((const uint16_t *)a.q)[at + e] << 16;
                w[e] = (w[e] >> 31 != 0) == hi ? 0u : w[e];
            }
        } else {
            w = *reinterpret_cast<const u32x4 *>((const uint16_t *)a.q + at);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t m = ((w[e] >> 15) & 0x10001u) * 0xffffu;  // 0xffff in negative halves
                w[e] &= hi ? ~m : m;
            }
        }
        qf[i] = w;
    }
    char *lds = dyn + wave * 16 * LDR;
    const size_t block_bytes = (size_t)RB * a.num_kv_heads;
    const char *base = a.bounds + (size_t)kvh * RB;
    auto load = [&](int tile, u32x4 (&in)[LPT]) {
#pragma unroll
        for (int j = 0; j < LPT; ++j) {
            const int slot = 64 * j + lane, r = slot / CPR, c = slot % CPR;
            const size_t blk = (size_t)max(ids[16 * tile + r], 0);
            in[j] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(base + blk * block_bytes + c * 16));
        }
    };
    auto tile = [&](int t, const u32x4 (&in)[LPT]) {
#pragma unroll
        for (int j = 0; j < LPT; ++j) {
            const int slot = 64 * j + lane, r = slot / CPR, c = slot % CPR;
            *reinterpret_cast<u32x4 *>(lds + r * LDR + c * 16) = in[j];
        }
        wave_sync();  // rows go to other lanes than loaded them
        f32x4 acc[2] = {f32x4{0.f, 0.f, 0.f, 0.f}, f32x4{0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int c = 0; c < CPR / 4; ++c) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(lds + col * LDR + (4 * c + grp) * 16);
            if constexpr (F32) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    acc[e & 1] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(w[e]), __uint_as_float(qf[c][e]), acc[e & 1], 0, 0, 0);
            } else if constexpr (KV == ZK_BF16) {
                acc[c & 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), __builtin_bit_cast(bf16x8, qf[c]),
                                                                     acc[c & 1], 0, 0, 0);
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const u32x2 lo = e4m3x4_to_bf16x4(w[2 * h]), hi = e4m3x4_to_bf16x4(w[2 * h + 1]);
                    acc[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, u32x4{lo[0], lo[1], hi[0], hi[1]}),
                                                                     __builtin_bit_cast(bf16x8, qf[2 * c + h]), acc[h], 0, 0, 0);
                }
            }
        }
        wave_sync();  // the next tile's rows come behind these reads
        f32x4 s = acc[0] + acc[1];  // column col's scores of the tile's pages 4 grp + i
#pragma unroll
        for (int i = 0; i < 4; ++i) {  // maximum over the 16 columns
            s[i] = max_nan(s[i], dpp<0x121>(s[i]));
            s[i] = max_nan(s[i], dpp<0x122>(s[i]));
            s[i] = max_nan(s[i], dpp<0x124>(s[i]));
            s[i] = max_nan(s[i], dpp<0x128>(s[i]));
        }
        // lane col < 4 of each group writes page 4 grp + col
        float v = s[0];
        v = col == 1 ? s[1] : v;
        v = col == 2 ? s[2] : v;
        v = col == 3 ? s[3] : v;
        const int p = 16 * t + 4 * grp + col;
        if (col < 4) found[wave][p] = ids[p] >= 0 ? v : -INFINITY;
    };
    const int tiles = (live + 15) / 16;
    u32x4 in0[LPT];
    load(0, in0);
    if constexpr (LPT <= 8) {
        u32x4 in1[LPT];
        int t = 0;
        for (; t + 1 < tiles; t += 2) {
            load(t + 1, in1);
            tile(t, in0);
            load(min(t + 2, tiles - 1), in0);
            tile(t + 1, in1);
        }
        if (t < tiles) tile(t, in0);
    } else {
        for (int t = 0; t < tiles; ++t) {
            tile(t, in0);
            if (t + 1 < tiles) load(t + 1, in0);
        }
    }
    // in whole lines at the end: 64 bytes a tile as they come cost 2 us of 256 contexts' 54
    wave_sync();
    for (int p = lane; p < live; p += 64) out[p] = found[wave][p];
}

// Any shape and type: one wave per (page, kv-head, sequence), lanes over the
// dimensions.
template <int KV>
__global__ void __launch_bounds__(kThreads) page_scores_generic_kernel(ScoreArgs a) {
    typedef Rows<KV, false> P;
    constexpr int ES = KV == ZK_F32 ? 4 : KV == ZK_BF16 ? 2 : 1;
    const int lane = threadIdx.x & 63;
    const int page = blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6), kvh = blockIdx.y, n = blockIdx.z;
    if (page >= a.max_blocks) return;
    const int D = a.head_dim, G = a.num_heads / a.num_kv_heads;
    float best = -INFINITY;
    const int blk = page < held_pages(a.seq_lens[n], a.block_size, a.max_blocks) ? a.tables[(size_t)n * a.max_blocks + page] : -1;
    if (blk >= 0 && blk < a.num_blocks) {
        const char *lo = a.bounds + ((size_t)blk * a.num_kv_heads + kvh) * 2 * D * ES, *hi = lo + (size_t)D * ES;
        for (int j = 0; j < G; ++j) {
            const size_t qo = ((size_t)n * a.num_heads + qhead(a, kvh, j, G)) * D;
            float s = 0.0f;
            for (int d = lane; d < D; d += 64) {
                const float q = a.q_f32 ? ((const float *)a.q)[qo + d]
                                        : __uint_as_float((uint32_t)((const uint16_t *)a.q)[qo + d] << 16);
                float l, u;
                P::load(lo + (size_t)d * ES, &l);
                P::load(hi + (size_t)d * ES, &u);
                const bool neg = __float_as_uint(q) >> 31;
                s = fmaf(neg ? q : 0.0f, l, s);
                s = fmaf(neg ? 0.0f : q, u, s);
            }
            for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o);
            best = j == 0 ? s : max_nan(best, s);
        }
    }
    if (lane == 0) a.scores[((size_t)n * a.num_kv_heads + kvh) * a.max_blocks + page] = best;
}

// ------------------------------------------------------------ selection
// Order of the scores as unsigned numbers: greater score, greater key; -0 as
// +0, every NaN above +inf, pages taken in any case (kGiven) above those.
constexpr uint32_t kGiven = 0xffffffffu;
__device__ __forceinline__ uint32_t score_key(float x) {
    const uint32_t u = __float_as_uint(x + 0.0f);
    if (x != x) return 0xfffffffeu;
    return u >> 31 ? ~u : u | 0x80000000u;
}

// One workgroup of W waves per (sequence, kv-head); a lane keeps the keys of R
// pages: page (w R + r) 64 + lane.  The k-th largest key is found bit by bit from
// the top, over the bits in which keys differ at all (a count of keys not below the
// candidate, a ballot a register; ended when a candidate has exactly k), then pages
// above it and, in page order, as many equal to it as are wanted are written at
// their rank: no sort, and the list ascends by itself.  Waves add their counts in
// LDS (whole numbers: the order does not matter), a counter and a barrier a round.
// Bound by the rounds' instructions after the loads' latency; two bits a round
// with three candidates take more of them (9.6 us instead of 8.5 over all 32 bits
// for 2048 rows of 512 pages, 19.4 instead of 16.0 for 16 of 8192).
template <int W, int R>
__global__ void __launch_bounds__(64 * W)
select_pages_kernel(const float *__restrict__ scores, const int32_t *__restrict__ seq_lens, int width, int block_size,
                    int k, int sink, int recent, int32_t *__restrict__ pages) {
    __shared__ int count_s[32];
    __shared__ uint32_t diff_s;
    __shared__ int part[2][W];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int hkv = gridDim.x, n = blockIdx.y;
    const size_t rowi = (size_t)n * hkv + blockIdx.x;
    const float *row = scores + rowi * (size_t)width;
    const int len = seq_lens[n];
    uint32_t key[R];  // first the scores' bits: all loads before any use
    if constexpr (W == 1) {  // (narrow rows: not behind the length's load, though it may leave few of them)
#pragma unroll
        for (int r = 0; r < R; ++r) key[r] = __float_as_uint(row[min(r * 64 + lane, width - 1)]);
    }
    const float first = row[min(sink, width - 1)];
    const int held = held_pages(len, block_size, width);
    int32_t *out = pages + rowi * (size_t)k;
    if (held <= k) {  // all of them
        for (int i = threadIdx.x; i < k; i += 64 * W) out[i] = i < held ? i : -1;
        return;
    }
    const int free0 = sink, free1 = held - recent;  // pages that compete (at least one: held > k >= sink + recent)
    if constexpr (W > 1) {
        if (threadIdx.x < 32) count_s[threadIdx.x] = 0;
        if (threadIdx.x == 0) diff_s = 0;
    }
    const uint32_t base = score_key(first);
    if constexpr (W > 1) {
#pragma unroll
        for (int r = 0; r < R; ++r) key[r] = __float_as_uint(row[min((w * R + r) * 64 + lane, held - 1)]);
    }
    // What follows goes through a lane's keys four times.  With many of them the compiler
    // must not keep the page numbers and masks of one pass for the next, nor a pass's
    // masks to its end: they are more registers than there are, and keys spilt to memory
    // (64 keys a lane: 92 bytes of them; 32 rows of 62000 pages 64 us, 48)
    constexpr bool kMany = R > 16;
    int page = w * R * 64 + lane;  // of key[0]
    auto again = [&] {
        if constexpr (kMany) asm volatile("" : "+v"(page));
    };
    auto settle = [](int r, int &sum) {  // the sum so far, every 8 keys
        if constexpr (kMany)
            if (r % 8 == 7) asm volatile("" : "+s"(sum));
    };
    again();
    uint32_t diff = 0;  // bits in which competing keys differ from the first one
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int p = page + r * 64;
        const bool competes = p >= free0 && p < free1;
        const uint32_t x = score_key(__uint_as_float(key[r]));
        diff |= competes ? x ^ base : 0u;
        key[r] = competes ? x : p < held ? kGiven : 0u;
        if constexpr (kMany) asm volatile("" : "+v"(key[r]));  // here, not behind the barriers
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) diff |= (uint32_t)__shfl_xor((int)diff, o);
    if constexpr (W > 1) {
        __syncthreads();
        if (lane == 0) atomicOr(&diff_s, diff);
        __syncthreads();
        diff = diff_s;
    }
    // the greatest value with at least k keys not below it
    uint32_t t = base & ~diff, left = __builtin_amdgcn_readfirstlane(diff);
    if (sink + recent == k) {
        t = kGiven;
        left = 0;
    }
#pragma unroll 1
    while (left) {
        const int bit = 31 - __builtin_clz(left);
        left &= ~(1u << bit);
        const uint32_t cand = t | 1u << bit;
        int c = 0;
#pragma unroll
        for (int r = 0; r < R; ++r) {
            c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] >= cand));
            settle(r, c);
        }
        if constexpr (W > 1) {
            if (lane == 0) atomicAdd(&count_s[bit], c);
            __syncthreads();
            c = count_s[bit];
        }
        c = __builtin_amdgcn_readfirstlane(c);
        if (c >= k) t = cand;
        if (c == k) break;
    }
    // counts of this wave's keys above t and equal to it
    int above = 0, equal = 0;
#pragma unroll
    for (int r = 0; r < R; ++r) {
        above += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] > t));
        equal += __builtin_popcountll(__builtin_amdgcn_ballot_w64(key[r] == t));
        settle(r, above);
        settle(r, equal);
    }
    int above_at = 0, equal_at = 0, all_above = above;
    if constexpr (W > 1) {
        if (lane == 0) {
            part[0][w] = above;
            part[1][w] = equal;
        }
        __syncthreads();
        all_above = 0;
#pragma unroll
        for (int j = 0; j < W; ++j) {
            const int pa = part[0][j], pb = part[1][j];
            above_at += j < w ? pa : 0;
            equal_at += j < w ? pb : 0;
            all_above += pa;
        }
    }
    const int want = k - all_above;  // of the equal ones, the first (after a count of exactly k: all)
    const uint64_t below = (1ull << lane) - 1;
    again();
    if constexpr (kMany) asm volatile("" : "+v"(t));
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const uint64_t gt = __builtin_amdgcn_ballot_w64(key[r] > t), eq = __builtin_amdgcn_ballot_w64(key[r] == t);
        const int ga = above_at + __builtin_popcountll(gt & below), ea = equal_at + __builtin_popcountll(eq & below);
        if (key[r] > t || (key[r] == t && ea < want)) out[ga + min(ea, want)] = page + r * 64;
        above_at += __builtin_popcountll(gt);
        equal_at += __builtin_popcountll(eq);
    }
}

constexpr int kSelectMost = 16 * 64 * 64;  // pages of the widest variant

template <int KV, int D>
void launch_scores_d(const ScoreArgs &a, dim3 grid, hipStream_t s) {
    const int waves = std::min(a.num_kv_heads, kScoreHeads);
    const int lds = waves * 16 * (2 * D * (KV == ZK_F32 ? 4 : KV == ZK_BF16 ? 2 : 1) + 16);
    page_scores_mfma_kernel<KV, D><<<grid, 64 * waves, lds, s>>>(a);
}
template <int KV>
void launch_scores(const ScoreArgs &a, dim3 grid, hipStream_t s) {
    if (a.head_dim == 64) launch_scores_d<KV, 64>(a, grid, s);
    else if (a.head_dim == 96) launch_scores_d<KV, 96>(a, grid, s);
    else if (a.head_dim == 128) launch_scores_d<KV, 128>(a, grid, s);
    else if constexpr (KV != ZK_F32) launch_scores_d<KV, 256>(a, grid, s);
}
bool scores_mfma(int q_dtype, int kv_dtype, int head_dim, int G) {
    if (G > 16 || (q_dtype == ZK_F32 && kv_dtype != ZK_F32)) return false;  // (f32 queries are not rounded)
    return head_dim == 64 || head_dim == 96 || head_dim == 128 || (head_dim == 256 && kv_dtype != ZK_F32);
}

}  // namespace

extern "C" {

int zk_page_bounds(const void *k_pool, zk_dtype kv_dtype, const int64_t *slot_mapping, int64_t num_tokens,
                   int num_kv_heads, int head_dim, int block_size, int64_t num_blocks, void *bounds, void *stream) {
    if (!valid_dtype(kv_dtype))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_bounds: unsupported dtype");
    if (num_tokens < 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 || num_blocks <= 0 ||
        (int64_t)num_kv_heads * head_dim > 0x7fffffff)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_bounds: bad shape");
    if (num_tokens == 0) return ZK_OK;
    if (!k_pool || !slot_mapping || !bounds)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_bounds: NULL pointer");
    const bool vec = ((size_t)head_dim * elt_size(kv_dtype)) % 16 == 0 && (((uintptr_t)k_pool | (uintptr_t)bounds) & 15u) == 0;
    // a row a workgroup while that fills the chip no more than a few times, then two and
    // four: us with 1, 2, 4 and 8, 26000 rows of prompts 19.4, 14.2, 12.9 and 13.1; 2000
    // of one prompt 6.3, 4.7, 4.5; 1000 and 3000 single tokens 4.2, 5.0, 6.1 and 8.7, 8.0, 9.1
    const int64_t rows = num_tokens <= 512 ? 1 : num_tokens <= 4096 ? 2 : 4;
    const int64_t groups = (num_tokens + rows - 1) / rows;
    if (groups > 0xffffff)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_bounds: too many tokens for one launch");
    const unsigned grid = (unsigned)groups;
    const int pieces = num_kv_heads * (vec ? head_dim * elt_size(kv_dtype) / 16 : head_dim);
    const int threads = std::min(kThreads, (pieces + 63) / 64 * 64);
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("page_bounds", s);
    auto go = [&](auto kernel) {
        kernel<<<grid, threads, 0, s>>>((const char *)k_pool, slot_mapping, num_tokens, (int)rows, num_kv_heads, head_dim,
                                         block_size, num_blocks * block_size, (char *)bounds);
    };
    if (kv_dtype == ZK_F32) vec ? go(page_bounds_kernel<ZK_F32, true>) : go(page_bounds_kernel<ZK_F32, false>);
    else if (kv_dtype == ZK_BF16) vec ? go(page_bounds_kernel<ZK_BF16, true>) : go(page_bounds_kernel<ZK_BF16, false>);
    else vec ? go(page_bounds_kernel<ZK_FP8_E4M3, true>) : go(page_bounds_kernel<ZK_FP8_E4M3, false>);
    return check_launch("zk_page_bounds");
}

int zk_page_scores(const void *q, zk_dtype q_dtype, const void *bounds, zk_dtype kv_dtype, const int32_t *block_tables,
                   const int32_t *seq_lens, float *scores, int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                   int block_size, int max_blocks_per_seq, int64_t num_blocks, zk_gqa_mapping mapping, void *stream) {
    if ((q_dtype != ZK_F32 && q_dtype != ZK_BF16) || !valid_dtype(kv_dtype))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_scores: unsupported dtype");
    if (num_seqs < 0 || num_seqs > 65535 || num_heads <= 0 || num_kv_heads <= 0 || num_kv_heads > 65535 || head_dim <= 0 ||
        block_size <= 0 || max_blocks_per_seq <= 0 || max_blocks_per_seq > kMostPages || num_blocks <= 0 ||
        num_heads % num_kv_heads != 0)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_scores: bad shape");
    if (mapping != ZK_GQA_GROUPED && mapping != ZK_GQA_MODULO)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_scores: bad gqa mapping");
    if (num_seqs == 0) return ZK_OK;
    if (!q || !bounds || !block_tables || !seq_lens || !scores)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_page_scores: NULL pointer");
    ScoreArgs a{};
    a.q = q;
    a.bounds = (const char *)bounds;
    a.tables = block_tables;
    a.seq_lens = seq_lens;
    a.scores = scores;
    a.num_blocks = num_blocks;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.grouped = mapping == ZK_GQA_GROUPED;
    a.q_f32 = q_dtype == ZK_F32;
    const int G = num_heads / num_kv_heads;
    hipStream_t s = (hipStream_t)stream;
    KernelTimer timer("page_scores", s);
    const bool mfma = scores_mfma(q_dtype, kv_dtype, head_dim, G) && (((uintptr_t)q | (uintptr_t)bounds) & 15u) == 0;
    if (mfma) {
        // Long stretches a wave as long as there are enough of them; us with 8, 12 and 16
        // tiles to begin with: 256 contexts of 512 to 8192 tokens 53.4, 53.8, 58.6; 256 of
        // 8192 98.0, 96.1, 92.1; 2 of 100000 and more (fp8) 8.6, 7.7, 8.6; 64 of f32 38.2,
        // 34.4, 38.1
        a.tiles = 12;
        auto groups = [&](int tiles) {
            return (int64_t)num_seqs * num_kv_heads * ((max_blocks_per_seq + 16 * tiles - 1) / (16 * tiles));  // of a wave
        };
        while (a.tiles > 1 && groups(a.tiles) < 2048) a.tiles /= 2;
        while ((max_blocks_per_seq + 16 * a.tiles - 1) / (16 * a.tiles) > 65535 && a.tiles < kScoreTiles) a.tiles *= 2;
        const dim3 grid((num_kv_heads + kScoreHeads - 1) / kScoreHeads, num_seqs,
                        (max_blocks_per_seq + 16 * a.tiles - 1) / (16 * a.tiles));
        if (kv_dtype == ZK_F32) launch_scores<ZK_F32>(a, grid, s);
        else if (kv_dtype == ZK_BF16) launch_scores<ZK_BF16>(a, grid, s);
        else launch_scores<ZK_FP8_E4M3>(a, grid, s);
    } else {
        const dim3 grid((max_blocks_per_seq + kThreads / 64 - 1) / (kThreads / 64), num_kv_heads, num_seqs);
        if (kv_dtype == ZK_F32) page_scores_generic_kernel<ZK_F32><<<grid, kThreads, 0, s>>>(a);
        else if (kv_dtype == ZK_BF16) page_scores_generic_kernel<ZK_BF16><<<grid, kThreads, 0, s>>>(a);
        else page_scores_generic_kernel<ZK_FP8_E4M3><<<grid, kThreads, 0, s>>>(a);
    }
    return check_launch("zk_page_scores");
}

int zk_select_pages(const float *scores, const int32_t *seq_lens, int num_seqs, int num_kv_heads,
                    int max_blocks_per_seq, int block_size, int num_pages, int sink, int recent, int32_t *pages,
                    void *stream) {
    if (num_seqs < 0 || num_seqs > 65535 || num_kv_heads <= 0 || max_blocks_per_seq <= 0 || block_size <= 0 ||
        num_pages <= 0 || num_pages > kMostPages || (int64_t)max_blocks_per_seq * block_size > 0x7fffffff)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_select_pages: bad shape");
    if (sink < 0 || recent < 0 || (int64_t)sink + recent > num_pages)
        return set_error(ZK_ERR_INVALID_ARGUMENT,
                         "Internal error: zk_select_pages: sink + recent must not exceed num_pages");
    if (max_blocks_per_seq > kSelectMost)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_select_pages: at most 65536 pages a sequence");
    if (num_seqs == 0) return ZK_OK;
    if (!scores || !seq_lens || !pages)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_select_pages: NULL pointer");
    const dim3 grid(num_kv_heads, num_seqs);
    hipStream_t s = (hipStream_t)stream;
    const int width = max_blocks_per_seq;
    KernelTimer timer("select_pages", s);
    auto go = [&](auto kernel, int waves) {
        kernel<<<grid, 64 * waves, 0, s>>>(scores, seq_lens, width, block_size, num_pages, sink, recent, pages);
    };
    // the fewest waves that hold a row in a few registers a lane (2048 rows of up to 8192
    // pages with 16 waves of 8 registers 55 us, 8 of 16 43; 32 rows of 16250 with 16 of 32
    // 24.5, 8 of 32 16.8, 16 of 16 15.1; 32 of 62000 with 16 of 64 48)
    if (width <= 64 * 8) go(select_pages_kernel<1, 8>, 1);
    else if (width <= 64 * 4 * 8) go(select_pages_kernel<4, 8>, 4);
    else if (width <= 64 * 8 * 16) go(select_pages_kernel<8, 16>, 8);
    else if (width <= 64 * 16 * 16) go(select_pages_kernel<16, 16>, 16);
    else if (width <= 64 * 16 * 32) go(select_pages_kernel<16, 32>, 16);
    else go(select_pages_kernel<16, 64>, 16);
    return check_launch("zk_select_pages");
}

}  // extern "C"
