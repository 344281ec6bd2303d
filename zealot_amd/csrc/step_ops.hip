// step_ops.hip -- the tables of a serving step from its request lengths, on
// the GPU: which blocks its new tokens take, the slot, position and sequence
// of every token row, the offsets and the lengths afterwards.
//
// Sequence i holds s_i tokens and receives n_i; with B tokens a block,
//   p_i = ceil(s_i / B), e_i = ceil((s_i + n_i) / B)    (blocks before, after)
//   base_i = cursor + sum over j < i of (e_j - p_j)
//   table[i][p_i + k] = granted[base_i + k]             (k < e_i - p_i)
//   row cu_i + j: position s_i + j, slot table[i][pos / B] * B + pos % B
// The reference computes slots and tables on the host, token by token
// (src/kv_cache.rs:127-161, :229-256).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <string>

#include "zk_common.h"

using namespace zk;

namespace {

struct StepArgs {
    int32_t *tables;
    const int32_t *seq_lens, *new_lens, *granted;
    const int64_t *cursor;
    int64_t *cursor_out, *slots, *cu;
    int32_t *positions, *rows, *kv_lens;
    int64_t num_granted, num_rows, cap;  // cap: tokens a table holds
    int num_seqs, max_blocks, block_size;
};

__device__ __forceinline__ int64_t before_of(const StepArgs &a, int i) { return max(a.seq_lens[i], 0); }
__device__ __forceinline__ int64_t new_of(const StepArgs &a, int i) { return max(a.new_lens[i], 0); }
// Blocks that sequence i's step takes: those of its tokens that the table has room for.
__device__ __forceinline__ int64_t blocks_of(int64_t tokens, const StepArgs &a) {
    return (uint64_t)(min(tokens, a.cap) + a.block_size - 1) / (uint32_t)a.block_size;
}

// Every workgroup scans all lengths (thread t the t-th run of `per`
// sequences), then finds the sequence of each of its token rows: a binary
// search of the runs' offsets in LDS and a walk inside the run.  Nothing is
// handed between workgroups, so the call is one launch; what it costs is the
// latency of three dependent reads.  A row that begins a block enters it in
// the table: rows in begun blocks only read entries below p_i, so no entry is
// both read and written.
template <int kThreads>
__global__ void __launch_bounds__(kThreads) step_tables_kernel(StepArgs a) {
    __shared__ int64_t tok_at[kThreads], blk_at[kThreads];
    __shared__ int64_t wave_tok[kThreads / 64], wave_blk[kThreads / 64];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int per = (a.num_seqs + kThreads - 1) / kThreads;
    const int i0 = min(t * per, a.num_seqs), i1 = min(i0 + per, a.num_seqs);
    int64_t tok = 0, blk = 0;
    for (int i = i0; i < i1; ++i) {
        const int64_t s = before_of(a, i), n = new_of(a, i);
        tok += n;
        blk += blocks_of(s + n, a) - blocks_of(s, a);
    }
    int64_t tok_in = tok, blk_in = blk;  // inclusive over the wave
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int64_t u = __shfl_up(tok_in, o), v = __shfl_up(blk_in, o);
        if (lane >= o) {
            tok_in += u;
            blk_in += v;
        }
    }
    if (lane == 63) {
        wave_tok[wave] = tok_in;
        wave_blk[wave] = blk_in;
    }
    __syncthreads();
    int64_t total = 0, blocks = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        if (w < wave) {
            tok_in += wave_tok[w];
            blk_in += wave_blk[w];
        }
        total += wave_tok[w];
        blocks += wave_blk[w];
    }
    tok_at[t] = tok_in - tok;
    blk_at[t] = blk_in - blk;
    const int64_t cursor = a.cursor ? max(*a.cursor, (int64_t)0) : 0;
    if (blockIdx.x == 0) {
        int64_t at = tok_in - tok;
        for (int i = i0; i < i1; ++i) {
            const int64_t s = before_of(a, i), n = new_of(a, i);
            a.cu[i] = at;
            a.kv_lens[i] = (int32_t)min(s + n, a.cap);
            at += n;
        }
        if (t == 0) {
            a.cu[a.num_seqs] = total;
            *a.cursor_out = a.granted ? cursor + blocks : cursor;
        }
    }
    __syncthreads();
    for (int64_t r = (int64_t)blockIdx.x * kThreads + t; r < a.num_rows; r += (int64_t)gridDim.x * kThreads) {
        if (r >= total) {  // a row of the batch's padding
            a.slots[r] = -1;
            a.positions[r] = -1;
            a.rows[r] = -1;
            continue;
        }
        int lo = 0, hi = kThreads;  // the last run that begins at or before r
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (tok_at[mid] <= r) lo = mid;
            else hi = mid;
        }
        int i = lo * per;
        int64_t at = tok_at[lo], base = cursor + blk_at[lo], s = before_of(a, i), n = new_of(a, i);
        while (r >= at + n) {  // ends inside the run: r < total
            at += n;
            base += blocks_of(s + n, a) - blocks_of(s, a);
            ++i;
            s = before_of(a, i);
            n = new_of(a, i);
        }
        const int64_t pos = s + (r - at);
        int64_t slot = -1;
        if (pos < a.cap) {
            const int64_t page = (uint64_t)pos / (uint32_t)a.block_size, tib = pos - page * a.block_size;
            int32_t *entry = a.tables + (size_t)i * a.max_blocks + page;
            const int64_t p0 = blocks_of(s, a);
            int32_t b;
            if (a.granted && page >= p0) {
                const int64_t g = base + (page - p0);
                b = g < a.num_granted ? a.granted[g] : -1;
                if (tib == 0) *entry = b;
            } else {
                b = *entry;
            }
            if (b >= 0) slot = (int64_t)b * a.block_size + tib;
        }
        a.slots[r] = slot;
        a.positions[r] = (int32_t)min(pos, (int64_t)0x7fffffff);
        a.rows[r] = i;
    }
}

}  // namespace

extern "C" int zk_step_tables(int32_t *block_tables, int num_seqs, int max_blocks_per_seq, const int32_t *seq_lens,
                              const int32_t *new_lens, int block_size, const int32_t *new_blocks,
                              int64_t num_new_blocks, const int64_t *cursor, int64_t *cursor_out,
                              int64_t *slot_mapping, int32_t *positions, int32_t *token_row, int64_t num_rows,
                              int64_t *cu_seqlens, int32_t *kv_lens, void *stream) {
    if (num_seqs < 0 || max_blocks_per_seq <= 0 || block_size <= 0 || num_new_blocks < 0 || num_rows < 0 ||
        num_new_blocks > 0x7fffffff || num_rows > 0x7fffffff ||
        (int64_t)max_blocks_per_seq * block_size > 0x7fffffff)
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_step_tables: bad shape");
    if (!cursor_out || !cu_seqlens || (num_seqs > 0 && (!block_tables || !seq_lens || !new_lens || !kv_lens)) ||
        (num_rows > 0 && (!slot_mapping || !positions || !token_row)) || (num_new_blocks > 0 && !new_blocks))
        return set_error(ZK_ERR_INVALID_ARGUMENT, "Internal error: zk_step_tables: NULL pointer");
    // workgroups read the inputs while others write: what is written meets nothing else
    const struct {
        const void *p;
        int64_t bytes;
    } all[] = {{block_tables, 4 * (int64_t)num_seqs * max_blocks_per_seq},
               {cursor_out, 8},
               {slot_mapping, 8 * num_rows},
               {positions, 4 * num_rows},
               {token_row, 4 * num_rows},
               {cu_seqlens, 8 * ((int64_t)num_seqs + 1)},
               {kv_lens, 4 * (int64_t)num_seqs},
               {seq_lens, 4 * (int64_t)num_seqs},
               {new_lens, 4 * (int64_t)num_seqs},
               {new_blocks, 4 * num_new_blocks},
               {cursor, cursor ? 8 : 0}};
    for (int i = 0; i < 7; ++i)
        for (int j = i + 1; j < 11; ++j) {
            const uintptr_t u = (uintptr_t)all[i].p, v = (uintptr_t)all[j].p;
            if (all[i].bytes > 0 && all[j].bytes > 0 && u < v + all[j].bytes && v < u + all[i].bytes)
                return set_error(ZK_ERR_INVALID_ARGUMENT,
                                 "Internal error: zk_step_tables: outputs must not be inputs, the tables or each other");
        }
    StepArgs a{};
    a.tables = block_tables;
    a.seq_lens = seq_lens;
    a.new_lens = new_lens;
    a.granted = new_blocks;
    a.cursor = cursor;
    a.cursor_out = cursor_out;
    a.slots = slot_mapping;
    a.cu = cu_seqlens;
    a.positions = positions;
    a.rows = token_row;
    a.kv_lens = kv_lens;
    a.num_granted = num_new_blocks;
    a.num_rows = num_rows;
    a.cap = (int64_t)max_blocks_per_seq * block_size;
    a.num_seqs = num_seqs;
    a.max_blocks = max_blocks_per_seq;
    a.block_size = block_size;
    hipStream_t s = (hipStream_t)stream;
    // a row a thread, the scan repeated in at most 512 workgroups; large batches:
    // four times the threads, so that a thread scans fewer sequences (4096 of one
    // token: 24 us with 256 threads)
    KernelTimer timer("step_tables", s);
    auto go = [&](auto kernel, int threads) {
        const int64_t grid = std::max<int64_t>(1, std::min<int64_t>((num_rows + threads - 1) / threads, 512));
        kernel<<<(unsigned)grid, threads, 0, s>>>(a);
    };
    if (num_seqs <= 512) go(step_tables_kernel<256>, 256);
    else go(step_tables_kernel<1024>, 1024);
    if (hipError_t e = hipGetLastError(); e != hipSuccess)
        return set_error(ZK_ERR_HIP, std::string("Internal error: zk_step_tables: ") + hipGetErrorString(e));
    return ZK_OK;
}
