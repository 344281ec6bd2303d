/*
 * zealot_dense.h -- C ABI of the dense ops around the paged-KV path (gfx950):
 * the elementwise / normalisation kernels and projections of a Llama layer
 * that the reference runner launches around its KV calls
 * (src/cuda_runner.rs:287-660).  Asynchronous on `stream`; shapes are checked
 * on the host first and nothing is launched when a check fails.  Tensors are
 * row-major, f32 or bf16 (zk_dtype of zealot_kv.h) with f32 arithmetic.
 */
#ifndef ZEALOT_DENSE_H
#define ZEALOT_DENSE_H

#include "zealot_kv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* RMSNorm (attention/kernels/rms_norm.cu:4-55):
 *   out[i] = s[r] * rsqrt(mean(s[r]^2) + eps) * weight
 * over rows r = rows ? rows[i] : i (i < num_rows), with s = x, or, when
 * `residual` is given, s = x + residual (the reference's add_kernel,
 * activation.cu:14-20, fused in) written to residual_out[i] (which may be
 * `residual` itself).  dim <= 32768 (bf16) / 16384 (f32) for 16-byte rows,
 * <= 4096 otherwise.  out / residual_out are packed [num_rows, dim]; out may
 * be x when rows is NULL. */
int zk_rms_norm(const void *x, const void *residual, const void *weight, void *out,
                void *residual_out, const int64_t *rows, int64_t num_rows, int64_t dim, float eps,
                zk_dtype dtype, void *stream);

/* silu_gate_mul (activation.cu:4-12): out[r, c] = silu(gate[r, c]) * up[r, c]
 * with silu(g) = g / (1 + exp(-g)); gate / up rows are gate_stride /
 * up_stride elements apart (0 = cols), so the halves of a fused gate|up
 * projection [rows, 2 * cols] feed it in place. */
int zk_silu_mul(const void *gate, const void *up, void *out, int64_t rows, int64_t cols,
                int64_t gate_stride, int64_t up_stride, zk_dtype dtype, void *stream);

/* add_kernel (activation.cu:14-20): out = a + b over n elements. */
int zk_add(const void *a, const void *b, void *out, int64_t n, zk_dtype dtype, void *stream);

/* embedding_gather_kernel (embedding.cu:4-22): out[t] = table[ids[t]]
 * (ids: device int64 [num_tokens]); an id outside [0, vocab) gives a zero row
 * (the reference reads out of bounds). */
int zk_embedding(const int64_t *ids, const void *table, void *out, int64_t num_tokens, int64_t vocab,
                 int64_t dim, zk_dtype dtype, void *stream);

/* Norms of the query and key heads and the rotary position embedding in one
 * pass.  No reference counterpart (its runner applies neither between the
 * projections and the KV write, cuda_runner.rs:331-461).  Every head row x of
 * q [num_tokens, num_heads, head_dim] and k [num_tokens, num_kv_heads,
 * head_dim]:
 *   y = x * rsqrt(mean(x^2) + eps) * weight       (weight NULL: y = x)
 *   (y_a, y_b) -> (y_a c_i - y_b s_i, y_b c_i + y_a s_i),  i < rot_dim / 2,
 * (a, b) = (i, i + rot_dim / 2), or (2 i, 2 i + 1) when interleaved; dimensions
 * from rot_dim on keep y.  Row p of rope (f32 [max_positions, rot_dim]) holds
 * the rot_dim / 2 cosines of position p, then its sines; rot_dim 0: no rotation
 * (rope and positions may be NULL).  A token whose position lies outside [0,
 * max_positions) gets zero rows.  Arithmetic in f32, one rounding.  Token rows
 * are *_stride elements apart (0 = packed), so columns of a fused projection
 * are read, and with q_out == q (k_out == k) and equal strides written, in
 * place; an output that otherwise overlaps q, k, v or the other one is refused.
 * head_dim <= 1024, num_tokens < 2^24. */
int zk_qk_norm_rope(const void *q, int64_t q_stride, const void *k, int64_t k_stride, zk_dtype dtype,
                    int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, const void *q_weight,
                    const void *k_weight, float eps, const int32_t *positions, const float *rope,
                    int64_t max_positions, int rot_dim, int interleaved, void *q_out, int64_t q_out_stride,
                    void *k_out, int64_t k_out_stride, void *stream);
/* zk_qk_norm_rope with zk_append of the resulting K rows and of v in the same
 * launch: K is rounded once, to the pool's type (with an F32 or BF16 pool of the
 * source's type, bit for bit the two calls).  Slots, pools, scales and token_row
 * as for zk_append; a token without a slot still gets its q row. */
int zk_qk_norm_rope_append(void *k_pool, void *v_pool, zk_dtype cache_dtype, const void *q, int64_t q_stride,
                           const void *k, int64_t k_stride, const void *v, int64_t v_stride, zk_dtype dtype,
                           int64_t num_tokens, int num_heads, int num_kv_heads, int head_dim, const void *q_weight,
                           const void *k_weight, float eps, const int32_t *positions, const float *rope,
                           int64_t max_positions, int rot_dim, int interleaved, void *q_out, int64_t q_out_stride,
                           const int64_t *slot_mapping, int block_size, int64_t num_blocks, const float *k_scales,
                           const float *v_scales, const int32_t *token_row, void *stream);

/* Projection y[m, n] = x[m, k] . w[n, k]^T (w in nn.Linear layout), the
 * product of every cublasSgemm_v2 site (attention/cublas.rs:72-114;
 * cuda_runner.rs:331-369, :483-495, :531-559, :577-589, :627-639), with
 * f32 accumulation, on hipBLASLt or (bf16, m <= 64) on this library's
 * weight-streaming kernel (zk_linear_skinny): the fastest is chosen per shape
 * (see zk_linear_tuning).  in_dtype F32 -> out F32; in_dtype BF16 ->
 * out BF16 or F32 (e.g. f32 logits).  Each (device, stream) has its own
 * workspaces (up to 8 streams a device; a ninth replaces the least recently
 * used one after a device synchronization), so calls on different streams
 * may overlap. */
int zk_linear(const void *x, const void *w, void *y, int64_t m, int64_t n, int64_t k, zk_dtype in_dtype,
              zk_dtype out_dtype, void *stream);
/* No counterpart in the reference: the weight-streaming kernel zk_linear's
 * tuning may pick for bf16 products with m <= 64, called directly (for
 * tests, and callers that want it without tuning).  x, w bf16, y f32 or bf16,
 * all 16-byte aligned.  Workgroups own tile_rows (64 or 128) weight rows and
 * k / splits of k: needs n % tile_rows == 0, k % (128 * splits) == 0,
 * splits <= 64 and splits * m * n * 4 <= 32 MiB.  With splits > 1 the
 * ranges' sums are added in range order by a second kernel (the result does
 * not depend on scheduling), in the stream's own workspace as for
 * zk_linear. */
int zk_linear_skinny(const void *x, const void *w, void *y, int64_t m, int64_t n, int64_t k, zk_dtype out_dtype,
                     int tile_rows, int splits, void *stream);
/* No counterpart in the reference (which launches its GEMM, add_kernel and
 * rms_norm_kernel one after the other, cuda_runner.rs:483-529): the
 * projection y = x . w^T (bf16, as zk_linear) followed by
 * zk_rms_norm(y, residual, norm_weight, out, residual_out, NULL rows), bit for
 * bit, with y itself not kept.  When zk_linear's tuning finds the
 * weight-streaming kernel with split k as fast as its choice, to within the
 * launch this saves, the norm kernel adds the split-k sums as it reads its
 * rows (two launches instead of three); otherwise the projection writes `out`
 * and the norm runs in place.  residual_out may be residual; dim n % 8 == 0
 * and <= 32768 for the fused form. */
int zk_linear_rms_norm(const void *x, const void *w, int64_t m, int64_t n, int64_t k, const void *residual,
                       const void *norm_weight, float eps, void *out, void *residual_out, void *stream);
/* No counterpart in the reference (which launches gate and up sgemms and
 * silu_gate_mul_kernel, cuda_runner.rs:531-571): act[m, inter] = silu(gate) *
 * up for x[m, k] (bf16) against w[2 inter, k] whose rows hold gate and up
 * interleaved in blocks of 16 -- rows 32 b .. 32 b + 15 are gate rows
 * 16 b .. 16 b + 15, the next 16 the up rows of the same columns -- bit for
 * bit zk_linear(x, w) followed by SiLU * up of the rounded outputs.  When
 * zk_linear's tuning keeps the weight-streaming kernel with 128-row tiles and
 * no split for (m, 2 inter, k), that kernel's waves hold the gate and up
 * outputs of the same columns and write act directly (one launch); otherwise
 * the projection goes to gu [m, 2 inter] (bf16, always required: the tuning
 * also writes there) and a second kernel forms act.  inter % 16 == 0. */
int zk_linear_silu_mul(const void *x, const void *w, void *act, int64_t m, int64_t inter, int64_t k, void *gu,
                       void *stream);
/* No counterpart in the reference: what zk_linear's plan for (m, n, k,
 * dtypes) on the current device runs, once a call has made it:
 * choice = {splits, tile_rows, fused_splits, fused_rows}; splits 0 means
 * hipBLASLt, else the weight-streaming kernel with that split of k and
 * tile; fused_* is what zk_linear_rms_norm runs (fused_splits 0: the
 * projection as zk_linear, then the norm). */
int zk_linear_choice(int64_t m, int64_t n, int64_t k, zk_dtype in_dtype, zk_dtype out_dtype, int choice[4]);

/* Tiled weights.  No counterpart in the reference, whose weights stay in
 * nn.Linear layout for cuBLAS (model_loader.rs:241, cuda_runner.rs:331-639):
 * the layout the weight-streaming kernel reads with contiguous 1 KiB loads,
 * [k / 128][n / 16][16 rows][16 units of 8 bf16], unit u of row r holding
 * columns 8 (u ^ r) .. 8 (u ^ r) + 7 of its 128-column chunk.  A model
 * converts its large decode-time weights once at load; the products below
 * read them 17-19 % faster than row-major weights on the Llama-3-8B
 * gate|up and lm_head shapes, bit for bit the same results as the
 * weight-streaming kernel on the row-major weights (same configuration).
 * The tiled products run on that kernel only (no hipBLASLt), for any m: up
 * to 64 rows of x per pass over the weights, so they suit decode-sized m.
 * All operands 16-byte aligned. */
/* wt = row-major bf16 w [n, k] tiled; n % 16 == 0, k % 128 == 0, w and wt
 * must not overlap. */
int zk_weight_tile(const void *w, void *wt, int64_t n, int64_t k, void *stream);
/* zk_linear for bf16 x and tiled weights (y bf16 or f32): the fastest
 * configuration of the weight-streaming kernel (tile rows, split of k) is
 * timed on first use of (m, n, k, out_dtype) as zk_linear times its
 * candidates.  Needs n % 64 == 0 and k % 128 == 0. */
int zk_linear_tiled(const void *x, const void *wt, void *y, int64_t m, int64_t n, int64_t k, zk_dtype out_dtype,
                    void *stream);
/* zk_linear_rms_norm (same arguments, bf16) for tiled weights. */
int zk_linear_rms_norm_tiled(const void *x, const void *wt, int64_t m, int64_t n, int64_t k, const void *residual,
                             const void *norm_weight, float eps, void *out, void *residual_out, void *stream);
/* zk_linear_silu_mul for the tiled form of the interleaved gate|up weight
 * [2 inter, k]: always one launch (the kernel's 128-row tiles hold gate and
 * up of the same columns), so no projection buffer; inter % 64 == 0. */
int zk_linear_silu_mul_tiled(const void *x, const void *wt, void *act, int64_t m, int64_t inter, int64_t k,
                             void *stream);
/* zk_linear_choice for the plan zk_linear_tiled / zk_linear_rms_norm_tiled
 * made for (m, n, k, out_dtype): {splits, tile_rows, fused_splits,
 * fused_rows}. */
int zk_linear_tiled_choice(int64_t m, int64_t n, int64_t k, zk_dtype out_dtype, int choice[4]);

/* No counterpart in the reference.  Pins the split-k configuration that
 * zk_linear_rms_norm[_tiled] and zk_cache_write_batch_qkv fold for the plan
 * an earlier call made for (m, n, k, dtypes; tiled: the tiled plan):
 * fused_splits > 1 ranges of k over tiles of fused_rows weight rows, or
 * fused_splits 0 for none (the projection, then its consumer).  For callers
 * that fix a configuration they measured, and for tests that must run the
 * folded kernels whatever the tuning chose.  ZK_ERR_INVALID_ARGUMENT if no
 * plan exists yet or the configuration does not fit the shape. */
int zk_linear_pin_split(int64_t m, int64_t n, int64_t k, zk_dtype in_dtype, zk_dtype out_dtype, int tiled,
                        int fused_splits, int fused_rows);

/* ---- projections in 8 bits.  No reference counterpart (its projections are
 * f32 sgemms, attention/cublas.rs:72-114).  8 bits are e4m3 (OCP; largest value
 * 448); a row y is held as one f32 scale and 8-bit values,
 *   scale = max(max |y| / 448, 2^-126),  q = e4m3(y / scale), nearest even;
 * a row that holds a NaN has a NaN scale and NaN values.
 *
 * zk_rms_norm (as there: s = x + residual rounded to the tensors' type and
 * written to residual_out) whose rows are written in 8 bits, from f32 and
 * rounded once: q [num_rows, dim] bytes, scales [num_rows].  rows (device int64
 * [num_rows], NULL: all, x_rows == num_rows) selects rows of x [x_rows, dim] and
 * of the residual; one outside [0, x_rows) gives zeros.  residual_out may be x
 * or the residual itself when rows is NULL; outputs overlap nothing else.
 * dim <= 32768 (bf16) / 16384 (f32) where it is a multiple of 8 / 4, <= 4096
 * otherwise. */
int zk_rms_norm_fp8(const void *x, const void *residual, const void *weight, void *q, float *scales,
                    void *residual_out, const int64_t *rows, int64_t x_rows, int64_t num_rows, int64_t dim, float eps,
                    zk_dtype dtype, void *stream);
/* zk_silu_mul (rows gate_stride / up_stride elements apart, 0 = cols) whose rows
 * are written in 8 bits; as there a gate below -88.72, whose exp(-g) is no f32,
 * gives 0.  cols as dim above. */
int zk_silu_mul_fp8(const void *gate, const void *up, void *q, float *scales, int64_t rows, int64_t cols,
                    int64_t gate_stride, int64_t up_stride, zk_dtype dtype, void *stream);
/* A weight w [n, k] (nn.Linear layout) in 8 bits with one scale a row, packed
 * once for zk_linear_fp8: [ceil(n / 64)][4 tiles][ceil(k / 128)][8 units][16
 * rows][16 bytes], unit u of a chunk holding its columns 16 u .. 16 u + 15 and
 * row i of tile t of group G being row 64 G + 16 (i / 4) + 4 t + i % 4; zeros
 * behind n and k.  dtype F32 or BF16: scales [n] is written (as for the rows
 * above); FP8_E4M3: w holds the 8-bit values, whose scales the caller has (scales
 * is not touched and may be NULL).  packed: zk_fp8_weight_bytes(n, k) bytes,
 * 16-byte aligned. */
size_t zk_fp8_weight_bytes(int64_t n, int64_t k);
int zk_fp8_weight(const void *w, zk_dtype dtype, void *packed, float *scales, int64_t n, int64_t k, void *stream);
/* y[m, n] = x_scales[m] w_scales[n] sum_k x[m, k] w[n, k] for x [m, k] in 8 bits
 * (packed rows; k % 16 == 0) and a packed weight; y F32 or BF16.  Sums in f32; for
 * BF16 each eight products are first cut to a multiple of 2^-13 of the largest
 * one's power of two (the 8-bit matrix instruction's own rounding), F32 results
 * keep their 24 bits.  x, the weight and y 16-byte aligned.  Nothing is tuned: a
 * call launches what its sizes say, and values are added in a fixed order.
 * workspace: zk_linear_fp8_workspace_size bytes (0: none needed), 16-byte aligned;
 * calls that share one must not overlap in time. */
size_t zk_linear_fp8_workspace_size(int64_t m, int64_t n, int64_t k, zk_dtype out_dtype);
int zk_linear_fp8(const void *x, const float *x_scales, const void *packed, const float *w_scales, void *y, int64_t m,
                  int64_t n, int64_t k, zk_dtype out_dtype, void *workspace, size_t workspace_bytes, void *stream);

/* ---- low-rank adapters of many requests beside a shared projection.  No
 * reference counterpart (one set of weights, model_loader.rs:241).
 *
 * The plan of a step: row t belongs to a request with adapter adapter_ids[t]
 * (device int32 [num_rows]; outside [0, num_adapters): none).
 *   order [num_rows]            the rows with an adapter, sorted by it, in their
 *                               order within one; then -1
 *   offsets [num_adapters + 1]  where each adapter's rows begin in order
 *   tiles [zk_lora_max_tiles][2]  runs of rows that zk_lora works on (its own)
 * It holds for every projection of the step.  At most 2^24 rows and 2048
 * adapters; outputs overlap nothing. */
int64_t zk_lora_max_tiles(int64_t num_rows, int64_t num_adapters);
int zk_lora_plan(const int32_t *adapter_ids, int64_t num_rows, int64_t num_adapters, int32_t *order, int32_t *offsets,
                 int32_t *tiles, void *stream);
/* y[t] += scales[a] b[a] (a_weights[a] x[t]) for the rows of a plan (made for the
 * same num_rows and num_adapters), a their adapter; other rows of y are left as
 * they are.  x [num_rows, k] (rows x_stride
 * elements apart, 0 = k), a_weights [num_adapters, num_parts * rank, k], b
 * [num_adapters, n, rank], scales f32 [num_adapters] (NULL: 1), y [num_rows, n]
 * (rows y_stride apart, 0 = n), all of `dtype` (F32, BF16); beside BF16 x may be
 * FP8_E4M3 rows with x_scales [num_rows].  With num_parts > 1 the columns of y
 * come in parts that have ranks of their own: part p (its columns: part_cols[p]
 * behind those of the parts before it, host int64 [num_parts]) meets rows p rank
 * .. of a_weights[a] alone.  part_block > 0 instead: the columns take their
 * parts in turn, part_block at a time (the gate and up rows of
 * zk_linear_silu_mul: 2 parts, blocks of 16).  f32 sums; the ranks' values keep
 * 16 bits or more between the two products.  rank <= 256, num_parts <= 4, rank *
 * num_parts <= 512.  workspace: zk_lora_workspace_size bytes, 16-byte aligned;
 * calls that share one must not overlap in time.  y and the workspace overlap
 * no operand. */
size_t zk_lora_workspace_size(int64_t num_rows, int64_t num_adapters, int64_t k, int rank, int num_parts, zk_dtype dtype);
int zk_lora(const void *x, const float *x_scales, int64_t x_stride, zk_dtype x_dtype, const void *a_weights,
            const void *b_weights, const float *scales, zk_dtype dtype, const int32_t *order, const int32_t *tiles,
            int64_t num_rows, int64_t num_adapters, int64_t k, int64_t n, int rank, int num_parts, const int64_t *part_cols,
            int part_block, void *y, int64_t y_stride, void *workspace, size_t workspace_bytes,
            void *stream);

/* On (default): the first call of each (m, n, k, dtypes) times hipBLASLt's
 * candidate algorithms on its operands (synchronizing the stream once) and
 * keeps the fastest.  Off: the heuristic's first choice, no synchronization
 * (for callers under stream capture). */
int zk_linear_tuning(int on);

#ifdef __cplusplus
}
#endif

#endif /* ZEALOT_DENSE_H */
