// paged_sparse.hip -- decode attention of one query row per sequence over a
// list of its pages per kv-head (sparse_ops.hip selects them), for gfx950.
// No reference counterpart (its decode walks every page,
// src/attention/kernels/paged_attention.cu:65-131).
//
//   o[n, h] = softmax over tokens t of the listed pages, t < len[n], of
//             (q[n, h] . k_t * scale) times v_t
// An entry that is negative, past the table or the length, or whose block lies
// outside the pool adds nothing; a page listed twice counts twice; a row
// without tokens is zero.
//
// Bound by HBM: every listed page's K and V are read once for the G = H / Hkv
// heads that share them.  Softmax in the log2 domain, statistics and sums in
// f32; f32 queries keep their 24 bits on every pool.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>

#include "attn_device.h"
#include "zk_common.h"

using namespace zk;

namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxList = 1024;  // list entries of a workgroup
constexpr int kMaxG = 16;

struct SparseArgs {
    const void *q;
    const char *k_pool, *v_pool;
    void *out;
    const int32_t *tables, *seq_lens, *pages;
    const float *k_scales, *v_scales;
    float2 *ml;  // [N][H][splits] (m, l)
    float *po;   // [N][H][splits][D]
    int64_t num_blocks;
    int num_seqs, num_heads, num_kv_heads, head_dim, block_size, max_blocks, num_pages, splits, per_split;
    float scale_log2;
    int grouped, q_f32;
};

__device__ __forceinline__ int qhead_of(const SparseArgs &a, int kvh, int j, int G) {
    return a.grouped ? kvh * G + j : kvh + j * a.num_kv_heads;
}
__device__ __forceinline__ float load_q(const SparseArgs &a, size_t i) {
    return a.q_f32 ? ((const float *)a.q)[i] : __uint_as_float((uint32_t)((const uint16_t *)a.q)[i] << 16);
}

__device__ __forceinline__ void store_out(const SparseArgs &a, size_t i, float x) {
    if (a.q_f32) ((float *)a.out)[i] = x;
    else ((uint16_t *)a.out)[i] = (uint16_t)f32_to_bf16_bits(x);
}

// The entries of this workgroup's part of list (n, kvh) that add something, in
// list order: their blocks and how many of a page's tokens lie below the
// length.  Returns their number.  All threads of the workgroup.
template <int WAVES>
__device__ __forceinline__ int stage_list(const SparseArgs &a, int n, int kvh, int split, int32_t *blk, int32_t *cnt,
                                          int *wave_sum) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t len = min((int64_t)max(a.seq_lens[n], 0), (int64_t)a.max_blocks * a.block_size);
    const int32_t *list = a.pages + ((size_t)n * a.num_kv_heads + kvh) * a.num_pages;
    const int32_t *row = a.tables + (size_t)n * a.max_blocks;
    const int e0 = split * a.per_split, e1 = min(e0 + a.per_split, a.num_pages);
    int total = 0;
    for (int e = e0; e < e1; e += 64 * WAVES) {
        const int i = e + (int)threadIdx.x;
        const int pg = i < e1 ? list[i] : -1;
        int b = -1, c = 0;
        if (pg >= 0 && pg < a.max_blocks) {
            b = row[pg];
            c = (int)max(min(len - (int64_t)pg * a.block_size, (int64_t)a.block_size), (int64_t)0);
        }
        const bool ok = c > 0 && b >= 0 && b < a.num_blocks;
        const uint64_t mask = __builtin_amdgcn_ballot_w64(ok);
        int at = total + __builtin_popcountll(mask & ((1ull << lane) - 1));
        if constexpr (WAVES > 1) {
            if (lane == 0) wave_sum[wave] = __builtin_popcountll(mask);
            __syncthreads();
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                const int s = wave_sum[w];
                at += w < wave ? s : 0;
                total += s;
            }
            __syncthreads();
        } else {
            total += __builtin_popcountll(mask);
        }
        if (ok) {
            blk[at] = b;
            cnt[at] = c;
        }
    }
    __syncthreads();
    return total;
}

// ------------------------------------------------------------ MFMA kernel
// 16-token pages, D in {64, 96, 128, 256}, up to 16 heads a kv-head: one workgroup
// of four waves per (kv-head, sequence, split).  A wave takes every fourth step of the
// staged pages (a step is a pair of bf16 or fp8 pages, one f32 page); K and V go
// from memory straight into the lanes that feed the matrix cores, no LDS in the
// loop:
//   QK^T  v_mfma_f32_16x16x32_bf16, A = 16 K rows, B = the query heads; lane
//         (grp, col) reads 16 bytes of row col a k-step (any order of the dims
//         will do as long as the query's is the same) and gets tokens
//         4 grp + i of head col;
//   PV    v_mfma_f32_16x16x32_bf16 over the pair's 32 tokens: the scores'
//         fragment of both pages is the B operand as it is (slots 8 grp + e:
//         token 4 grp + e % 4 of page e / 4), and lane (grp, col) reads D / 16
//         consecutive dims of tokens 4 grp + i, whole rows by 16 lanes, which
//         v_perm transposes into the D / 16 A operands.
// f32 pools: v_mfma_f32_16x16x4_f32, four k-steps a 16-byte chunk of K, one a
// token of PV.
// The reference maximum of a head is moved only when a score exceeds it by
// kSlack.  The waves' results are merged in LDS.
//
// 256 contexts, 64 pages of each, 32 / 8 heads of 128 bf16 (1048 MB): 166 us, 6.3
// TB/s (a read of one piece reaches 7.5, one of shuffled 4 KB pieces 7 % less).
// Three workgroups run on a CU, by LDS (42.5 KB at a head size of 128: the lists' and the
// merge's) as by registers (bf16 pools: 134 to 162).  One step ahead in registers needs 208 of them,
// two waves a SIMD, and took 179; held to 128 registers the kernel spills, 215.
constexpr int kWaves = 4;
constexpr float kSlack = 8.0f;

// The `BYTES` bytes at p (nontemporal), in the widest pieces that their number allows.
template <int BYTES>
__device__ __forceinline__ void load_words(const char *p, uint32_t *w) {
    if constexpr (BYTES % 16 == 0) {
#pragma unroll
        for (int j = 0; j < BYTES / 16; ++j) {
            const u32x4 v = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(p + 16 * j));
#pragma unroll
            for (int e = 0; e < 4; ++e) w[4 * j + e] = v[e];
        }
    } else if constexpr (BYTES % 8 == 0) {
#pragma unroll
        for (int j = 0; j < BYTES / 8; ++j) {
            const u32x2 v = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(p + 8 * j));
            w[2 * j] = v[0];
            w[2 * j + 1] = v[1];
        }
    } else if constexpr (BYTES % 4 == 0) {
#pragma unroll
        for (int j = 0; j < BYTES / 4; ++j) w[j] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(p + 4 * j));
    } else {
        static_assert(BYTES == 6, "6 bytes: fp8 rows of 96");
        const uint16_t *h = reinterpret_cast<const uint16_t *>(p);
        w[0] = (uint32_t)__builtin_nontemporal_load(h) | (uint32_t)__builtin_nontemporal_load(h + 1) << 16;
        w[1] = __builtin_nontemporal_load(h + 2);
    }
}

// A value as three bf16 of its sign that add up to it: the leading 8 bits, the next 8
// and the last.  A part that would be zero is 2^-30 of the value instead (an infinite
// key times 0 would be NaN), and an infinity or NaN is all three.
__device__ __forceinline__ void three_parts(float x, float (&part)[3]) {
    const bool finite = fabsf(x) < INFINITY;
    const float tiny = x * 0x1p-30f;
    part[0] = finite ? __uint_as_float(__float_as_uint(x) & 0xffff0000u) : x;
    const float rest = x - part[0];
    part[1] = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
    part[2] = rest - part[1];
#pragma unroll
    for (int i = 1; i < 3; ++i) part[i] = !finite ? x : part[i] == 0.0f ? tiny : part[i];
}

// PARTS: bf16 values that a query value is held in: 1, or 3 for f32 queries on bf16
// and fp8 pools (exact: 24 bits).  256 lists of 64 pages with one part of 8 bits and with
// three: bf16 pools 176 and 184 us, fp8 100 and 112; 128 of heads of 256 192 and 227.
template <int KV, int D, int PARTS>
__global__ void __launch_bounds__(64 * kWaves) sparse_mfma_kernel(SparseArgs a) {
    constexpr bool F32 = KV == ZK_F32;
    static_assert(!F32 || PARTS == 1, "f32 products take f32 values");
    constexpr int BS = 16, ELT = F32 ? 4 : KV == ZK_BF16 ? 2 : 1, RB = D * ELT;
    constexpr int PG = F32 ? 1 : 2;            // pages a step
    constexpr int CB = RB % 64 ? 8 : 16;       // bytes of a K row that a lane reads at once
    constexpr int KC = RB / (4 * CB);          // ... and how often
    constexpr int KK = F32 ? KC : D / 32;      // query pieces: 4 f32, 8 bf16 dims
    constexpr int DT = D / 16, VB = DT * ELT;  // dims and bytes of a V row a lane
    constexpr int VW = (VB + 3) / 4;
    static_assert(DT % 2 == 0 && (CB == 16 || KV == ZK_FP8_E4M3), "row shape");
    constexpr size_t PAGE = (size_t)BS * RB;
    __shared__ int32_t blk[kMaxList], cnt[kMaxList];
    __shared__ int wave_sum[kWaves];
    __shared__ float mo[kWaves][kMaxG * (D + 4)], mm[kWaves][kMaxG], mlsum[kWaves][kMaxG];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int kvh = blockIdx.x, split = blockIdx.y, n = blockIdx.z;
    const int np = stage_list<kWaves>(a, n, kvh, split, blk, cnt, wave_sum);
    const int H = a.num_heads, G = H / a.num_kv_heads;
    // query pieces, as the lanes read K: bf16 rows (and fp8 ones read 8 bytes at
    // once): dims 32 kk + 8 grp .. + 7; fp8 rows (16 dims in 16 bytes): 64 (kk / 2) +
    // 16 grp + 8 (kk % 2) .. + 7; f32 rows: 16 kk + 4 grp .. + 3
    u32x4 qf[PARTS][KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        const int d0 = F32 ? 16 * kk + 4 * grp : KV == ZK_BF16 || CB == 8 ? 32 * kk + 8 * grp : 64 * (kk / 2) + 16 * grp + 8 * (kk % 2);
        u32x4 w[PARTS];
#pragma unroll
        for (int i = 0; i < PARTS; ++i) w[i] = u32x4{0u, 0u, 0u, 0u};
        if (col < G) {
            const size_t at = ((size_t)n * H + qhead_of(a, kvh, col, G)) * D + d0;
            if constexpr (F32) {
#pragma unroll
                for (int j = 0; j < 4; ++j) w[0][j] = __float_as_uint(load_q(a, at + j));
            } else if constexpr (PARTS == 3) {
                const float *p = (const float *)a.q + at;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float lo[3], hi[3];
                    three_parts(p[2 * j], lo);
                    three_parts(p[2 * j + 1], hi);
#pragma unroll
                    for (int i = 0; i < 3; ++i) w[i][j] = bf16x2_rne(lo[i], hi[i]);
                }
            } else {
                w[0] = *reinterpret_cast<const u32x4 *>((const uint16_t *)a.q + at);
            }
        }
#pragma unroll
        for (int i = 0; i < PARTS; ++i) qf[i][kk] = w[i];
    }
    float sl2 = a.scale_log2, vscale = 1.0f;
    if constexpr (KV == ZK_FP8_E4M3) {
        sl2 *= a.k_scales[(size_t)n * a.num_kv_heads + kvh];
        vscale = a.v_scales[(size_t)n * a.num_kv_heads + kvh];
    }
    const char *kbase = a.k_pool + (size_t)kvh * PAGE + (size_t)col * RB + grp * CB;
    const char *vbase = a.v_pool + (size_t)kvh * PAGE + (size_t)(4 * grp) * RB + col * VB;
    const size_t block_bytes = PAGE * a.num_kv_heads;

    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -FLT_MAX, l = 0.0f;
    const int steps = (np + PG - 1) / PG;
    for (int step = wave; step < steps; step += kWaves) {
        uint32_t kw[PG][KC][CB / 4];
        uint32_t vw[PG][4][VW];
        int tokens[PG];
#pragma unroll
        for (int h = 0; h < PG; ++h) {  // (an odd list's last page again, without tokens)
            const int i = min(PG * step + h, np - 1);
            const int b = __builtin_amdgcn_readfirstlane(blk[i]);
            tokens[h] = PG * step + h < np ? __builtin_amdgcn_readfirstlane(cnt[i]) : 0;
            const char *kp = kbase + (size_t)b * block_bytes, *vp = vbase + (size_t)b * block_bytes;
#pragma unroll
            for (int c = 0; c < KC; ++c) load_words<CB>(kp + 4 * CB * c, kw[h][c]);
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) load_words<VB>(vp + i2 * RB, vw[h][i2]);
        }
        float sc[PG][4];
#pragma unroll
        for (int h = 0; h < PG; ++h) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
            if constexpr (F32) {
                f32x4 s2 = s;  // two chains
#pragma unroll
                for (int c = 0; c < KC; ++c)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        f32x4 &t = e & 1 ? s2 : s;
                        t = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kw[h][c][e]), __uint_as_float(qf[0][c][e]), t, 0, 0, 0);
                    }
                s += s2;
            } else {
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    u32x4 w;
                    if constexpr (KV == ZK_BF16) {
                        w = u32x4{kw[h][kk][0], kw[h][kk][1], kw[h][kk][2], kw[h][kk][3]};
                    } else {
                        const uint32_t *c8 = CB == 8 ? kw[h][kk] : kw[h][kk / 2] + 2 * (kk % 2);
                        const u32x2 lo = e4m3x4_to_bf16x4(c8[0]), hi = e4m3x4_to_bf16x4(c8[1]);
                        w = u32x4{lo[0], lo[1], hi[0], hi[1]};
                    }
#pragma unroll
                    for (int i = PARTS - 1; i >= 0; --i)
                        s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w),
                                                                    __builtin_bit_cast(bf16x8, qf[i][kk]), s, 0, 0, 0);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h][i] = 4 * grp + i < tokens[h] ? s[i] * sl2 : -INFINITY;
        }
        float mx = -INFINITY;
#pragma unroll
        for (int h = 0; h < PG; ++h) mx = fmaxf(mx, fmaxf(fmaxf(sc[h][0], sc[h][1]), fmaxf(sc[h][2], sc[h][3])));
        if (__builtin_amdgcn_ballot_w64(mx > m + kSlack)) {
            float cm = fmaxf(mx, xor16(mx));
            cm = fmaxf(cm, xor32(cm));
            const float m_new = fmaxf(m, cm);
            const float alpha = exp2_fast(m - m_new);
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
            m = m_new;
        }
        float pr[PG][4];
#pragma unroll
        for (int h = 0; h < PG; ++h) {
#pragma unroll
            for (int i = 0; i < 4; ++i) pr[h][i] = exp2_fast(sc[h][i] - m);
            l += (pr[h][0] + pr[h][1]) + (pr[h][2] + pr[h][3]);
            if (tokens[h] < BS) {  // what lies behind the length must not reach O
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * grp + i >= tokens[h])
#pragma unroll
                        for (int j = 0; j < VW; ++j) vw[h][i][j] = 0u;
            }
        }
        if constexpr (F32) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    o[dt] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(vw[0][i][dt]), pr[0][i], o[dt], 0, 0, 0);
        } else {
            // V rows as bf16 pairs: vb[h][i][j] = dims (2 j, 2 j + 1) of token 4 grp + i
            uint32_t vb[PG][4][DT / 2];
#pragma unroll
            for (int h = 0; h < PG; ++h)
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < VW; ++j) {
                        if constexpr (KV == ZK_BF16) {
                            vb[h][i][j] = vw[h][i][j];
                        } else {
                            const u32x2 c2 = e4m3x4_to_bf16x4(vw[h][i][j]);
                            vb[h][i][2 * j] = c2[0];
                            if (2 * j + 1 < DT / 2) vb[h][i][2 * j + 1] = c2[1];
                        }
                    }
            // weights as two bf16 each, the leading 8 bits and what they leave (16 bits in
            // all): the matrix cores wait for memory anyway.  2^-20 of the weight is added
            // to the second, which is then never zero nor of the other sign: an infinity
            // in V stays one.  In f32 results (queries of three parts) the weights are three
            // parts as well, their 24 bits (184 us as with two).
            constexpr int WP = PARTS == 3 ? 3 : 2;
            u32x4 pw[WP];
#pragma unroll
            for (int h = 0; h < PG; ++h)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    if constexpr (WP == 3) {
                        float lo[3], hi[3];
                        three_parts(pr[h][i], lo);
                        three_parts(pr[h][i + 1], hi);
#pragma unroll
                        for (int j = 0; j < 3; ++j) pw[j][2 * h + i / 2] = bf16x2_rne(lo[j], hi[j]);
                    } else {
                        const uint32_t w = __builtin_amdgcn_perm(__float_as_uint(pr[h][i + 1]), __float_as_uint(pr[h][i]), 0x07060302u);
                        constexpr float kAll = 1.0f + 0x1p-20f;
                        pw[0][2 * h + i / 2] = w;
                        pw[1][2 * h + i / 2] = bf16x2_rne(fmaf(pr[h][i], kAll, -bf16lo(w)), fmaf(pr[h][i + 1], kAll, -bf16hi(w)));
                    }
                }
#pragma unroll
            for (int j = 0; j < DT / 2; ++j) {
                u32x4 ev, od;
#pragma unroll
                for (int h = 0; h < PG; ++h) {
                    ev[2 * h] = __builtin_amdgcn_perm(vb[h][1][j], vb[h][0][j], 0x05040100u);
                    ev[2 * h + 1] = __builtin_amdgcn_perm(vb[h][3][j], vb[h][2][j], 0x05040100u);
                    od[2 * h] = __builtin_amdgcn_perm(vb[h][1][j], vb[h][0][j], 0x07060302u);
                    od[2 * h + 1] = __builtin_amdgcn_perm(vb[h][3][j], vb[h][2][j], 0x07060302u);
                }
                const bf16x8 e8 = __builtin_bit_cast(bf16x8, ev), o8 = __builtin_bit_cast(bf16x8, od);
#pragma unroll
                for (int i = 0; i < WP; ++i) {
                    const bf16x8 w8 = __builtin_bit_cast(bf16x8, pw[i]);
                    o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(e8, w8, o[2 * j], 0, 0, 0);
                    o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(o8, w8, o[2 * j + 1], 0, 0, 0);
                }
            }
        }
    }
    if (wave < steps) {
        l += xor16(l);
        l += xor32(l);
    } else {
        m = -INFINITY;  // saw nothing
    }
    if (col < G) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                mo[wave][col * (D + 4) + DT * (4 * grp + i) + dt] = o[dt][i];
        if (grp == 0) {
            mm[wave][col] = m;
            mlsum[wave][col] = l;
        }
    }
    __syncthreads();
    for (int i = threadIdx.x; i < G * D; i += 64 * kWaves) {
        const int j = i / D, d = i % D;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) M = fmaxf(M, mm[w][j]);
        float L = 0.0f, v = 0.0f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = mm[w][j] == -INFINITY ? 0.0f : exp2_fast(mm[w][j] - M);
            L += mlsum[w][j] * f;
            v += mm[w][j] == -INFINITY ? 0.0f : mo[w][j * (D + 4) + d] * f;
        }
        const size_t row = (size_t)n * H + qhead_of(a, kvh, j, G);
        if (a.splits == 1) {
            store_out(a, row * D + d, v * inverse_sum(L, M, vscale));
        } else {
            const size_t slot = row * a.splits + split;
            a.po[slot * D + d] = v * vscale;
            if (d == 0) a.ml[slot] = make_float2(M, L);
        }
    }
}

// ------------------------------------------------------------ generic kernel
// Any pool type and block size, D <= 256, G <= 16: one wave per (kv-head,
// sequence, split), a token a lane for the scores, a dimension a lane for the
// sums; GM: the kv-head's heads rounded up to 4, 8 or 16.
constexpr int kDimSlots = 4;

template <int KV>
__device__ __forceinline__ float load_kv(const char *pool, size_t i) {
    if constexpr (KV == ZK_F32) return ((const float *)pool)[i];
    else if constexpr (KV == ZK_BF16) return __uint_as_float((uint32_t)((const uint16_t *)pool)[i] << 16);
    else {
        const f32x2 r = __builtin_amdgcn_cvt_pk_f32_fp8((int)((const uint8_t *)pool)[i], false);
        return r[0];
    }
}

template <int KV, int GM>
__global__ void __launch_bounds__(64) sparse_generic_kernel(SparseArgs a) {
    __shared__ int32_t blk[kMaxList], cnt[kMaxList];
    __shared__ float q_s[256][GM], p_s[64][GM];  // a dimension's (token's) heads side by side
    const int lane = threadIdx.x;
    const int kvh = blockIdx.x, split = blockIdx.y, n = blockIdx.z;
    const int D = a.head_dim, G = a.num_heads / a.num_kv_heads, H = a.num_heads;
    for (int i = lane; i < GM * D; i += 64) {  // (heads past G: zeros)
        const int j = i / D, d = i - j * D;
        q_s[d][j] = j < G ? load_q(a, ((size_t)n * H + qhead_of(a, kvh, j, G)) * D + d) : 0.0f;
    }
    const int np = stage_list<1>(a, n, kvh, split, blk, cnt, nullptr);
    float sl2 = a.scale_log2, vs = 1.0f;
    if constexpr (KV == ZK_FP8_E4M3) {
        sl2 *= a.k_scales[(size_t)n * a.num_kv_heads + kvh];
        vs = a.v_scales[(size_t)n * a.num_kv_heads + kvh];
    }
    float m[GM], l[GM], o[GM][kDimSlots];
#pragma unroll
    for (int j = 0; j < GM; ++j) {
        m[j] = np ? -FLT_MAX : -INFINITY;
        l[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < kDimSlots; ++c) o[j][c] = 0.0f;
    }
    const size_t head_rows = (size_t)kvh * a.block_size, block_rows = (size_t)a.num_kv_heads * a.block_size;
    for (int e = 0; e < np; ++e) {
        const size_t row0 = (size_t)blk[e] * block_rows + head_rows;
        const int tokens = cnt[e];
        for (int t0 = 0; t0 < tokens; t0 += 64) {
            const int here = min(64, tokens - t0);
            const bool valid = lane < here;
            const size_t row = (row0 + t0 + (valid ? lane : 0)) * D;
            float s[GM];
#pragma unroll
            for (int j = 0; j < GM; ++j) s[j] = 0.0f;
            for (int d = 0; d < D; ++d) {
                const float kd = load_kv<KV>(a.k_pool, row + d);
#pragma unroll
                for (int j = 0; j < GM; ++j) s[j] = fmaf(q_s[d][j], kd, s[j]);
            }
#pragma unroll
            for (int j = 0; j < GM; ++j) {
                const float sj = valid ? s[j] * sl2 : -INFINITY;
                float mx = sj;
                for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off));
                const float m_new = fmaxf(m[j], mx), alpha = exp2f(m[j] - m_new);
                const float p = valid ? exp2f(sj - m_new) : 0.0f;
                float ps = p;
                for (int off = 32; off > 0; off >>= 1) ps += __shfl_xor(ps, off);
                l[j] = l[j] * alpha + ps;
                m[j] = m_new;
#pragma unroll
                for (int c = 0; c < kDimSlots; ++c) o[j][c] *= alpha;
                p_s[lane][j] = p;
            }
            __syncthreads();
            for (int i = 0; i < here; ++i) {
#pragma unroll
                for (int c = 0; c < kDimSlots; ++c) {
                    const int d = lane + c * 64;
                    const float v = d < D ? load_kv<KV>(a.v_pool, (row0 + t0 + i) * D + d) : 0.0f;
#pragma unroll
                    for (int j = 0; j < GM; ++j) o[j][c] = fmaf(p_s[i][j], v, o[j][c]);
                }
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int j = 0; j < GM; ++j) {
        if (j < G) {
            const size_t row = (size_t)n * H + qhead_of(a, kvh, j, G);
            const float inv = inverse_sum(l[j], m[j], vs);
#pragma unroll
            for (int c = 0; c < kDimSlots; ++c) {
                const int d = lane + c * 64;
                if (d < D) {
                    if (a.splits == 1) store_out(a, row * D + d, o[j][c] * inv);
                    else a.po[(row * a.splits + split) * D + d] = o[j][c] * vs;
                }
            }
            if (a.splits > 1 && lane == 0) a.ml[row * a.splits + split] = make_float2(m[j], l[j]);
        }
    }
}

// o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s: one workgroup per (head,
// sequence).  A lane holds a split's statistics (chunks of 64 splits); a thread
// four dimensions of every (256 / (D / 4))-th split, whose values are loaded
// before the statistics are used; the parts are added in order.
constexpr int kReduceThreads = 256;
__global__ void __launch_bounds__(kReduceThreads) sparse_reduce_kernel(SparseArgs a) {
    constexpr int U = 4;
    __shared__ float part[kReduceThreads][5];
    const int h = blockIdx.x, n = blockIdx.y, D = a.head_dim, S = a.splits, lane = threadIdx.x & 63;
    const size_t row = (size_t)n * a.num_heads + h;
    const float2 *ml = a.ml + row * S;
    const int quads = (D + 3) / 4, every = kReduceThreads / quads;  // D <= 256
    const int quad = threadIdx.x % quads, first = threadIdx.x / quads;
    const bool on = first < every, whole = D % 4 == 0;
    float M = -INFINITY, L = 0.0f;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = 0; s0 < S; s0 += 64) {
        const int here = min(64, S - s0);
        const float2 x = lane < here ? ml[s0 + lane] : make_float2(-INFINITY, 0.0f);
        f32x4 p[U];
        auto load = [&](int s) -> f32x4 {
            const float *src = a.po + (row * S + s0 + s) * D + 4 * quad;
            if (whole) return *reinterpret_cast<const f32x4 *>(src);
            f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < 4; ++e)
                if (4 * quad + e < D) r[e] = src[e];
            return r;
        };
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (on && first + u * every < here) p[u] = load(first + u * every);
        float c = x.x;
        for (int o = 32; o > 0; o >>= 1) c = fmaxf(c, __shfl_xor(c, o));
        const float m_new = fmaxf(M, c), alpha = M == -INFINITY ? 0.0f : exp2_fast(M - m_new);
        const float w = x.x == -INFINITY ? 0.0f : exp2_fast(x.x - m_new);
        float ls = x.y * w;
        for (int o = 32; o > 0; o >>= 1) ls += __shfl_xor(ls, o);
        L = L * alpha + (c == -INFINITY ? 0.0f : ls);
        M = m_new;
        v *= alpha;
        for (int u = 0; u * every < here; ++u) {  // (the same for the workgroup: the shuffle needs every lane)
            const int s = first + u * every;
            const float ws = __shfl(w, min(s, 63));
            if (!on || s >= here || ws == 0.0f) continue;
            v += ws * (u == 0 ? p[0] : u == 1 ? p[1] : u == 2 ? p[2] : u == 3 ? p[3] : load(s));
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) part[threadIdx.x][e] = v[e];
    __syncthreads();
    if (first == 0) {
        for (int f = 1; f < every; ++f)
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += part[f * quads + quad][e];
        const float inv = inverse_sum(L, M);
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (4 * quad + e < D) store_out(a, row * D + 4 * quad + e, v[e] * inv);
    }
}

bool mfma_dim(int head_dim) { return head_dim == 64 || head_dim == 96 || head_dim == 128 || head_dim == 256; }

// Parts of a list, by its capacity (what it holds is known on the device only): enough
// workgroups to fill the CUs twice (one-wave ones of the generic kernel at head sizes
// that are not the matrix cores': four waves a SIMD), of at least 8 (4) pages each and,
// from 16 parts on, 16, at most kMaxList.  us with parts of 8, 16 and 32 pages: 8 lists of
// 64 bf16 pages 9.6, 10.8, 13.3; 16 of 256 fp8 pages 13.3 (32 parts), 12.0, 13.7.
int splits_for(int num_seqs, int num_kv_heads, int head_dim, int num_pages) {
    const int64_t rows = (int64_t)num_seqs * num_kv_heads;
    const bool mfma = mfma_dim(head_dim);
    const int64_t want = ((mfma ? 512 : 4096) + rows - 1) / rows;
    int64_t s = std::min<int64_t>(want, num_pages / (mfma ? 8 : 4));
    if (mfma) s = std::min<int64_t>(s, std::max(16, num_pages / 16));
    return (int)std::max<int64_t>(std::max<int64_t>(s, 1), (num_pages + kMaxList - 1) / kMaxList);
}

size_t align256(size_t x) { return (x + 255) & ~(size_t)255; }

int bad(const char *what) {
    return set_error(ZK_ERR_INVALID_ARGUMENT, std::string("Internal error: zk_paged_decode_sparse: ") + what);
}
int check_launch(const char *what) {
    hipError_t e = hipGetLastError();
    if (e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: ") + what + ": " + hipGetErrorString(e));
    return ZK_OK;
}

template <int KV, int PARTS>
void launch_mfma(const SparseArgs &a, dim3 grid, hipStream_t s) {
    if (a.head_dim == 64) sparse_mfma_kernel<KV, 64, PARTS><<<grid, 64 * kWaves, 0, s>>>(a);
    else if (a.head_dim == 96) sparse_mfma_kernel<KV, 96, PARTS><<<grid, 64 * kWaves, 0, s>>>(a);
    else if (a.head_dim == 128) sparse_mfma_kernel<KV, 128, PARTS><<<grid, 64 * kWaves, 0, s>>>(a);
    else sparse_mfma_kernel<KV, 256, PARTS><<<grid, 64 * kWaves, 0, s>>>(a);
}
template <int KV>
void launch(const SparseArgs &a, dim3 grid, int G, bool mfma, hipStream_t s) {
    if (mfma && a.q_f32 && KV != ZK_F32) launch_mfma<KV, KV == ZK_F32 ? 1 : 3>(a, grid, s);
    else if (mfma) launch_mfma<KV, 1>(a, grid, s);
    else if (G <= 4) sparse_generic_kernel<KV, 4><<<grid, 64, 0, s>>>(a);
    else if (G <= 8) sparse_generic_kernel<KV, 8><<<grid, 64, 0, s>>>(a);
    else sparse_generic_kernel<KV, 16><<<grid, 64, 0, s>>>(a);
}

}  // namespace

extern "C" {

size_t zk_paged_decode_sparse_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                             int num_pages) {
    if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_pages <= 0 ||
        num_pages > 65535 * kMaxList)
        return 0;
    const int splits = splits_for(num_seqs, num_kv_heads, head_dim, num_pages);
    if (splits == 1) return 0;
    const size_t slots = (size_t)num_seqs * num_heads * splits;
    return align256(sizeof(float2) * slots) + sizeof(float) * slots * head_dim;
}

int zk_paged_decode_sparse(const void *q, zk_dtype q_dtype, const void *k_pool, const void *v_pool, zk_dtype kv_dtype,
                           void *out, const int32_t *block_tables, const int32_t *seq_lens, const int32_t *pages,
                           int num_pages, int num_seqs, int num_heads, int num_kv_heads, int head_dim, int block_size,
                           int max_blocks_per_seq, int64_t num_blocks, float scale, zk_gqa_mapping mapping,
                           const float *k_scales, const float *v_scales, void *workspace, size_t workspace_bytes,
                           void *stream) {
    if (q_dtype != ZK_F32 && q_dtype != ZK_BF16) return bad("q dtype must be f32 or bf16");
    if (!valid_dtype(kv_dtype)) return bad("unsupported kv dtype");
    if (num_seqs < 0 || num_seqs > 65535 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
        block_size <= 0 || max_blocks_per_seq <= 0 || num_blocks <= 0 || num_pages <= 0)
        return bad("bad shape");
    if (num_heads % num_kv_heads != 0) return bad("num_heads must be a multiple of num_kv_heads");
    if (mapping != ZK_GQA_GROUPED && mapping != ZK_GQA_MODULO) return bad("bad gqa mapping");
    if (head_dim > 256 || num_heads / num_kv_heads > kMaxG) return bad("head_dim <= 256 and H/Hkv <= 16 required");
    if ((int64_t)max_blocks_per_seq * block_size > 0x7fffffff) return bad("context too long");
    if (num_pages > 65535 * kMaxList) return bad("too many pages a list");
    const int splits = num_seqs > 0 ? splits_for(num_seqs, num_kv_heads, head_dim, num_pages) : 1;
    if (num_seqs == 0) return ZK_OK;
    if (!q || !k_pool || !v_pool || !out || !block_tables || !seq_lens || !pages) return bad("NULL pointer");
    if ((kv_dtype == ZK_FP8_E4M3) != (k_scales != nullptr && v_scales != nullptr) || !k_scales != !v_scales)
        return bad("fp8 pools need k/v scales, other pools none");
    const size_t need = zk_paged_decode_sparse_workspace_size(num_seqs, num_heads, num_kv_heads, head_dim, num_pages);
    if (need && (!workspace || workspace_bytes < need || ((uintptr_t)workspace & 255u)))
        return set_error(ZK_ERR_INVALID_ARGUMENT,
                         "Internal error: zk_paged_decode_sparse: workspace too small or not 256-B aligned (need " +
                             std::to_string(need) + " bytes)");
    const int G = num_heads / num_kv_heads;
    SparseArgs a{};
    a.q = q;
    a.k_pool = (const char *)k_pool;
    a.v_pool = (const char *)v_pool;
    a.out = out;
    a.tables = block_tables;
    a.seq_lens = seq_lens;
    a.pages = pages;
    a.k_scales = k_scales;
    a.v_scales = v_scales;
    if (splits > 1) {
        a.ml = (float2 *)workspace;
        a.po = (float *)((char *)workspace + align256(sizeof(float2) * (size_t)num_seqs * num_heads * splits));
    }
    a.num_blocks = num_blocks;
    a.num_seqs = num_seqs;
    a.num_heads = num_heads;
    a.num_kv_heads = num_kv_heads;
    a.head_dim = head_dim;
    a.block_size = block_size;
    a.max_blocks = max_blocks_per_seq;
    a.num_pages = num_pages;
    a.splits = splits;
    a.per_split = (num_pages + splits - 1) / splits;
    a.scale_log2 = scale * kLog2e;
    a.grouped = mapping == ZK_GQA_GROUPED;
    a.q_f32 = q_dtype == ZK_F32;
    hipStream_t s = (hipStream_t)stream;
    // Workgroups go to the 8 XCDs in turn: a sequence's are on all of them this way (with the
    // sequences first, 1 % less time on 256 lists, a long one among 8 has one XCD alone)
    const dim3 grid(num_kv_heads, splits, num_seqs);
    const bool mfma = block_size == 16 && mfma_dim(head_dim) &&
                      (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15u) == 0;
    {
        KernelTimer timer("sparse_partials", s);
        if (kv_dtype == ZK_F32) launch<ZK_F32>(a, grid, G, mfma, s);
        else if (kv_dtype == ZK_BF16) launch<ZK_BF16>(a, grid, G, mfma, s);
        else launch<ZK_FP8_E4M3>(a, grid, G, mfma, s);
    }
    if (int rc = check_launch("zk_paged_decode_sparse")) return rc;
    if (splits == 1) return ZK_OK;
    KernelTimer timer("sparse_reduce", s);
    sparse_reduce_kernel<<<dim3(num_heads, num_seqs), kReduceThreads, 0, s>>>(a);
    return check_launch("zk_paged_decode_sparse reduce");
}

}  // extern "C"
