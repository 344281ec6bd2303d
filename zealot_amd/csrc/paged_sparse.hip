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
// f32; the weights are rounded to bf16 for PV on bf16 and fp8 pools, whose
// values have no more bits.
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
// bf16 and fp8 pools, 16-token pages, D in {64, 128}, G in {1, 2, 4, 8, 16}: one
// workgroup of four waves per (kv-head, sequence, split).  A wave takes every
// fourth pair of the staged pages; K and V go from memory straight into the
// lanes that feed the matrix cores, one pair ahead of the one being computed:
//   QK^T  v_mfma_f32_16x16x32_bf16, A = 16 K rows, B = the query heads; lane
//         (grp, col) reads 16 bytes of row col a k-step (any order of the dims
//         will do as long as the query's is the same) and gets tokens
//         4 grp + i of head col;
//   PV    v_mfma_f32_16x16x32_bf16 over the pair's 32 tokens: the scores'
//         fragment of both pages is the B operand as it is (slots 8 grp + e:
//         token 4 grp + e % 4 of page e / 4), and lane (grp, col) reads D / 16
//         consecutive dims of tokens 4 grp + i, whole rows by 16 lanes, which
//         v_perm transposes into the D / 16 A operands.
// No LDS in the loop.  The reference maximum of a head is moved only when a
// score exceeds it by kSlack.  The waves' results are merged in LDS.
constexpr int kWaves = 4;
constexpr float kSlack = 8.0f;

template <int KV, int D, int G>
__global__ void __launch_bounds__(64 * kWaves) sparse_mfma_kernel(SparseArgs a) {
    constexpr int BS = 16, ELT = KV == ZK_BF16 ? 2 : 1, RB = D * ELT;
    constexpr int KK = D / 32;                 // MFMA k-steps
    constexpr int KC = RB / 64;                // 16-byte chunks of a K row a lane
    constexpr int DT = D / 16, VB = DT * ELT;  // dims and bytes of a V row a lane
    constexpr int VW = VB / 4;
    constexpr size_t PAGE = (size_t)BS * RB;
    __shared__ int32_t blk[kMaxList], cnt[kMaxList];
    __shared__ int wave_sum[kWaves];
    __shared__ float mo[kWaves][G][D + 4], mm[kWaves][G], mlsum[kWaves][G];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, grp = lane >> 4;
    const int kvh = blockIdx.x, split = blockIdx.y, n = blockIdx.z;
    const int np = stage_list<kWaves>(a, n, kvh, split, blk, cnt, wave_sum);
    const int H = a.num_heads;
    // query fragments: k-step kk of bf16 rows holds dims 32 kk + 8 grp .. + 7,
    // of fp8 rows (16 dims in 16 bytes) dims 64 (kk / 2) + 16 grp + 8 (kk % 2) .. + 7
    bf16x8 qf[KK];
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
        const int d0 = KV == ZK_BF16 ? 32 * kk + 8 * grp : 64 * (kk / 2) + 16 * grp + 8 * (kk % 2);
        u32x4 w = {0u, 0u, 0u, 0u};
        if (col < G) {
            const size_t at = ((size_t)n * H + qhead_of(a, kvh, col, G)) * D + d0;
            if (a.q_f32) {
                const float *p = (const float *)a.q + at;
#pragma unroll
                for (int j = 0; j < 4; ++j) w[j] = bf16x2_rne(p[2 * j], p[2 * j + 1]);
            } else {
                w = *reinterpret_cast<const u32x4 *>((const uint16_t *)a.q + at);
            }
        }
        qf[kk] = __builtin_bit_cast(bf16x8, w);
    }
    float sl2 = a.scale_log2, vscale = 1.0f;
    if constexpr (KV == ZK_FP8_E4M3) {
        sl2 *= a.k_scales[(size_t)n * a.num_kv_heads + kvh];
        vscale = a.v_scales[(size_t)n * a.num_kv_heads + kvh];
    }
    const char *kbase = a.k_pool + (size_t)kvh * PAGE + (size_t)col * RB + grp * 16;
    const char *vbase = a.v_pool + (size_t)kvh * PAGE + (size_t)(4 * grp) * RB + col * VB;
    const size_t block_bytes = PAGE * a.num_kv_heads;

    struct Pair {
        u32x4 k[2][KC];
        uint32_t v[2][4][VW];
        int cnt[2];
    };
    auto load = [&](int pair, Pair &r) {  // pair: of this list; past its end the last page again, with no tokens
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int i = min(2 * pair + h, np - 1);
            const int b = __builtin_amdgcn_readfirstlane(blk[i]);
            r.cnt[h] = 2 * pair + h < np ? __builtin_amdgcn_readfirstlane(cnt[i]) : 0;
            const char *kp = kbase + (size_t)b * block_bytes, *vp = vbase + (size_t)b * block_bytes;
#pragma unroll
            for (int c = 0; c < KC; ++c)
                r.k[h][c] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kp + 64 * c));
#pragma unroll
            for (int i2 = 0; i2 < 4; ++i2) {
                if constexpr (VB == 16) {
                    const u32x4 w = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vp + i2 * RB));
#pragma unroll
                    for (int j = 0; j < 4; ++j) r.v[h][i2][j] = w[j];
                } else if constexpr (VB == 8) {
                    const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2 *>(vp + i2 * RB));
                    r.v[h][i2][0] = w[0];
                    r.v[h][i2][1] = w[1];
                } else {
                    r.v[h][i2][0] = __builtin_nontemporal_load(reinterpret_cast<const uint32_t *>(vp + i2 * RB));
                }
            }
        }
    };
    f32x4 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = -FLT_MAX, l = 0.0f;
    auto compute = [&](const Pair &r) {
        float sc[2][4];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                u32x4 w;
                if constexpr (KV == ZK_BF16) {
                    w = r.k[h][kk];
                } else {
                    const u32x2 lo = e4m3x4_to_bf16x4(r.k[h][kk / 2][2 * (kk % 2)]),
                                hi = e4m3x4_to_bf16x4(r.k[h][kk / 2][2 * (kk % 2) + 1]);
                    w = u32x4{lo[0], lo[1], hi[0], hi[1]};
                }
                s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, w), qf[kk], s, 0, 0, 0);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) sc[h][i] = 4 * grp + i < r.cnt[h] ? s[i] * sl2 : -INFINITY;
        }
        const float mx = fmaxf(fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[0][2], sc[0][3])),
                               fmaxf(fmaxf(sc[1][0], sc[1][1]), fmaxf(sc[1][2], sc[1][3])));
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
        u32x4 pw;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            float p[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) p[i] = exp2_fast(sc[h][i] - m);
            l += (p[0] + p[1]) + (p[2] + p[3]);
            pw[2 * h] = bf16x2_rne(p[0], p[1]);
            pw[2 * h + 1] = bf16x2_rne(p[2], p[3]);
        }
        // V rows as bf16 pairs: vw[h][i][j] = dims (2 j, 2 j + 1) of token 4 grp + i
        uint32_t vw[2][4][DT / 2];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if constexpr (KV == ZK_BF16) {
#pragma unroll
                    for (int j = 0; j < DT / 2; ++j) vw[h][i][j] = r.v[h][i][j];
                } else {
#pragma unroll
                    for (int j = 0; j < DT / 4; ++j) {
                        const u32x2 c2 = e4m3x4_to_bf16x4(r.v[h][i][j]);
                        vw[h][i][2 * j] = c2[0];
                        vw[h][i][2 * j + 1] = c2[1];
                    }
                }
            }
#pragma unroll
        for (int h = 0; h < 2; ++h)
            if (r.cnt[h] < BS) {  // what lies behind the length must not reach O
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (4 * grp + i >= r.cnt[h])
#pragma unroll
                        for (int j = 0; j < DT / 2; ++j) vw[h][i][j] = 0u;
            }
        const bf16x8 pb = __builtin_bit_cast(bf16x8, pw);
#pragma unroll
        for (int j = 0; j < DT / 2; ++j) {
            u32x4 ev, od;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                ev[2 * h] = __builtin_amdgcn_perm(vw[h][1][j], vw[h][0][j], 0x05040100u);
                ev[2 * h + 1] = __builtin_amdgcn_perm(vw[h][3][j], vw[h][2][j], 0x05040100u);
                od[2 * h] = __builtin_amdgcn_perm(vw[h][1][j], vw[h][0][j], 0x07060302u);
                od[2 * h + 1] = __builtin_amdgcn_perm(vw[h][3][j], vw[h][2][j], 0x07060302u);
            }
            o[2 * j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, ev), pb, o[2 * j], 0, 0, 0);
            o[2 * j + 1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, od), pb, o[2 * j + 1], 0, 0, 0);
        }
    };
    const int pairs = (np + 1) / 2;
    if (wave < pairs) {
        Pair r0, r1;
        load(wave, r0);
        int j = wave;
        for (; j + kWaves < pairs; j += 2 * kWaves) {
            load(j + kWaves, r1);
            compute(r0);
            load(min(j + 2 * kWaves, pairs), r0);  // (pair `pairs`: the last page again)
            compute(r1);
        }
        if (j < pairs) compute(r0);
        l += xor16(l);
        l += xor32(l);
    } else {
        m = -INFINITY;  // saw nothing
    }
    if (col < G) {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) mo[wave][col][DT * (4 * grp + i) + dt] = o[dt][i];
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
            v += mm[w][j] == -INFINITY ? 0.0f : mo[w][j][d] * f;
        }
        const size_t row = (size_t)n * H + qhead_of(a, kvh, j, G);
        if (a.splits == 1) {
            const float r = v * inverse_sum(L, M, vscale);
            if (a.q_f32) ((float *)a.out)[row * D + d] = r;
            else ((uint16_t *)a.out)[row * D + d] = (uint16_t)f32_to_bf16_bits(r);
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
// sums.
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

template <int KV>
__global__ void __launch_bounds__(64) sparse_generic_kernel(SparseArgs a) {
    __shared__ int32_t blk[kMaxList], cnt[kMaxList];
    __shared__ float q_s[kMaxG * 256], p_s[kMaxG][64];
    const int lane = threadIdx.x;
    const int kvh = blockIdx.x, split = blockIdx.y, n = blockIdx.z;
    const int D = a.head_dim, G = a.num_heads / a.num_kv_heads, H = a.num_heads;
    for (int i = lane; i < G * D; i += 64)
        q_s[i] = load_q(a, ((size_t)n * H + qhead_of(a, kvh, i / D, G)) * D + i % D);
    const int np = stage_list<1>(a, n, kvh, split, blk, cnt, nullptr);
    float sl2 = a.scale_log2, vs = 1.0f;
    if constexpr (KV == ZK_FP8_E4M3) {
        sl2 *= a.k_scales[(size_t)n * a.num_kv_heads + kvh];
        vs = a.v_scales[(size_t)n * a.num_kv_heads + kvh];
    }
    float m[kMaxG], l[kMaxG], o[kMaxG][kDimSlots];
#pragma unroll
    for (int j = 0; j < kMaxG; ++j) {
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
            float s[kMaxG];
#pragma unroll
            for (int j = 0; j < kMaxG; ++j) s[j] = 0.0f;
            if (valid)
                for (int d = 0; d < D; ++d) {
                    const float kd = load_kv<KV>(a.k_pool, (row0 + t0 + lane) * D + d);
#pragma unroll
                    for (int j = 0; j < kMaxG; ++j)
                        if (j < G) s[j] = fmaf(q_s[j * D + d], kd, s[j]);
                }
#pragma unroll
            for (int j = 0; j < kMaxG; ++j) {
                if (j >= G) break;
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
                p_s[j][lane] = p;
            }
            __syncthreads();
            for (int i = 0; i < here; ++i) {
                float vd[kDimSlots];
#pragma unroll
                for (int c = 0; c < kDimSlots; ++c) {
                    const int d = lane + c * 64;
                    vd[c] = d < D ? load_kv<KV>(a.v_pool, (row0 + t0 + i) * D + d) : 0.0f;
                }
#pragma unroll
                for (int j = 0; j < kMaxG; ++j) {
                    if (j >= G) break;
#pragma unroll
                    for (int c = 0; c < kDimSlots; ++c) o[j][c] = fmaf(p_s[j][i], vd[c], o[j][c]);
                }
            }
            __syncthreads();
        }
    }
#pragma unroll
    for (int j = 0; j < kMaxG; ++j) {
        if (j >= G) break;
        const size_t row = (size_t)n * H + qhead_of(a, kvh, j, G);
        const float inv = inverse_sum(l[j], m[j], vs);
#pragma unroll
        for (int c = 0; c < kDimSlots; ++c) {
            const int d = lane + c * 64;
            if (d >= D) break;
            if (a.splits == 1) {
                const float r = o[j][c] * inv;
                if (a.q_f32) ((float *)a.out)[row * D + d] = r;
                else ((uint16_t *)a.out)[row * D + d] = (uint16_t)f32_to_bf16_bits(r);
            } else {
                a.po[(row * a.splits + split) * D + d] = o[j][c] * vs;
            }
        }
        if (a.splits > 1 && lane == 0) a.ml[row * a.splits + split] = make_float2(m[j], l[j]);
    }
}

// o = sum_s 2^(m_s - M) o_s / sum_s 2^(m_s - M) l_s, in split order: a thread a
// dimension, the splits' statistics read by all.
__global__ void sparse_reduce_kernel(SparseArgs a) {
    const int h = blockIdx.x, n = blockIdx.y, d = threadIdx.x, D = a.head_dim;
    const size_t row = (size_t)n * a.num_heads + h;
    const float2 *ml = a.ml + row * a.splits;
    float M = -INFINITY;
    for (int s = 0; s < a.splits; ++s) M = fmaxf(M, ml[s].x);
    float L = 0.0f, v = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
        const float2 x = ml[s];
        if (x.x == -INFINITY) continue;
        const float f = exp2_fast(x.x - M);
        L += x.y * f;
        if (d < D) v += a.po[(row * a.splits + s) * D + d] * f;
    }
    if (d >= D) return;
    const float r = v * inverse_sum(L, M);
    if (a.q_f32) ((float *)a.out)[row * D + d] = r;
    else ((uint16_t *)a.out)[row * D + d] = (uint16_t)f32_to_bf16_bits(r);
}

// Parts of a list: enough workgroups to fill the CUs twice, of at least 16
// pages each (a wave then has two pairs), at most kMaxList.
int splits_for(int num_seqs, int num_kv_heads, int num_pages) {
    const int64_t rows = (int64_t)num_seqs * num_kv_heads;
    const int64_t want = (512 + rows - 1) / rows;
    int64_t s = std::max<int64_t>(1, std::min<int64_t>(want, num_pages / 16));
    s = std::max<int64_t>(s, (num_pages + kMaxList - 1) / kMaxList);
    return (int)s;
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

template <int KV, int D>
void launch_g(const SparseArgs &a, dim3 grid, int G, hipStream_t s) {
    switch (G) {
        case 1: sparse_mfma_kernel<KV, D, 1><<<grid, 64 * kWaves, 0, s>>>(a); break;
        case 2: sparse_mfma_kernel<KV, D, 2><<<grid, 64 * kWaves, 0, s>>>(a); break;
        case 4: sparse_mfma_kernel<KV, D, 4><<<grid, 64 * kWaves, 0, s>>>(a); break;
        case 8: sparse_mfma_kernel<KV, D, 8><<<grid, 64 * kWaves, 0, s>>>(a); break;
        default: sparse_mfma_kernel<KV, D, 16><<<grid, 64 * kWaves, 0, s>>>(a); break;
    }
}
template <int KV>
void launch_d(const SparseArgs &a, dim3 grid, int G, hipStream_t s) {
    if (a.head_dim == 128) launch_g<KV, 128>(a, grid, G, s);
    else launch_g<KV, 64>(a, grid, G, s);
}

}  // namespace

extern "C" {

size_t zk_paged_decode_sparse_workspace_size(int num_seqs, int num_heads, int num_kv_heads, int head_dim,
                                             int num_pages) {
    if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || num_pages <= 0) return 0;
    const int splits = splits_for(num_seqs, num_kv_heads, num_pages);
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
    if (num_seqs < 0 || num_seqs > 65535 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
        max_blocks_per_seq <= 0 || num_blocks <= 0 || num_pages <= 0)
        return bad("bad shape");
    if (num_heads % num_kv_heads != 0) return bad("num_heads must be a multiple of num_kv_heads");
    if (mapping != ZK_GQA_GROUPED && mapping != ZK_GQA_MODULO) return bad("bad gqa mapping");
    if (head_dim > 256 || num_heads / num_kv_heads > kMaxG) return bad("head_dim <= 256 and H/Hkv <= 16 required");
    if ((int64_t)max_blocks_per_seq * block_size > 0x7fffffff) return bad("context too long");
    const int splits = num_seqs > 0 ? splits_for(num_seqs, num_kv_heads, num_pages) : 1;
    if (splits > 65535) return bad("too many pages a list");
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
    const dim3 grid(num_kv_heads, splits, num_seqs);
    const bool mfma = kv_dtype != ZK_F32 && block_size == 16 && (head_dim == 64 || head_dim == 128) &&
                      (G == 1 || G == 2 || G == 4 || G == 8 || G == 16) &&
                      (((uintptr_t)q | (uintptr_t)k_pool | (uintptr_t)v_pool) & 15u) == 0;
    {
        KernelTimer timer("sparse_partials", s);
        if (mfma) {
            if (kv_dtype == ZK_BF16) launch_d<ZK_BF16>(a, grid, G, s);
            else launch_d<ZK_FP8_E4M3>(a, grid, G, s);
        } else if (kv_dtype == ZK_F32) {
            sparse_generic_kernel<ZK_F32><<<grid, 64, 0, s>>>(a);
        } else if (kv_dtype == ZK_BF16) {
            sparse_generic_kernel<ZK_BF16><<<grid, 64, 0, s>>>(a);
        } else {
            sparse_generic_kernel<ZK_FP8_E4M3><<<grid, 64, 0, s>>>(a);
        }
    }
    if (int rc = check_launch("zk_paged_decode_sparse")) return rc;
    if (splits == 1) return ZK_OK;
    KernelTimer timer("sparse_reduce", s);
    sparse_reduce_kernel<<<dim3(num_heads, num_seqs), (head_dim + 63) / 64 * 64, 0, s>>>(a);
    return check_launch("zk_paged_decode_sparse reduce");
}

}  // extern "C"
