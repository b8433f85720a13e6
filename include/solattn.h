/*
 * solattn.h -- C ABI of libsolattn.so, the gfx950 (MI355X) implementation of
 * Sol-Attn's sparse attention path.
 *
 * Conventions shared by every entry point:
 *  - Device pointers are plain pointers into HBM; "bf16" buffers hold bfloat16
 *    bit patterns (uint16_t). Strides are in ELEMENTS unless a name ends in
 *    _bytes. Inputs q/k/v are BTHD ([batch, tokens, heads, head_dim]) with only
 *    the last dim required to be contiguous; every other buffer is a dense
 *    allocation in the layout written next to it.
 *  - block is the routing block size in tokens (64 or 128); NT = ceil(T/block)
 *    query/key blocks; npad is the block dim of kc/vc (>= NT, zero padded).
 *  - Every function returns 0 on success or a negative SOLATTN_E* code and
 *    records a message readable with solattn_last_error() (thread-local).
 *  - The library never allocates device memory and never synchronises: every
 *    launch goes on the hipStream_t passed in (NULL = the null stream).
 *  - head_dim must be 128 for the per-kernel entry points (the reference
 *    node's only eligible head size, /root/reference/__init__.py:41,178); the
 *    one-call pipelines (solattn_sol_attn*) also take head dims that are
 *    multiples of 8 below 128 (the reference kernels' D = 64 configs,
 *    /root/reference/_tri_fwd.py:209). BF16 calls run heads of up to 64
 *    channels on 64-channel kernels, everything else runs at 128; a head dim
 *    that is neither is zero-padded to it in the workspace: zero channels add
 *    exact zeros to every dot product and sum, so routing, codes and outputs
 *    are those of the unpadded problem.
 *
 * Arithmetic contract (the CPU oracle restates the same operation order, so
 * pooled keys, thresholds, routing masks and INT8 codes are bit-exact):
 *  - pooled sums: for each (block, channel) sixteen fp32 partial sums p_g over
 *    the block's rows r = g (mod 16) taken in ascending order (rows past T add
 *    0.0f), combined pairwise as ((((p0+p1)+(p2+p3))+((p4+p5)+(p6+p7))) +
 *    (((p8+p9)+(p10+p11))+((p12+p13)+(p14+p15)))).
 *  - kc = bf16_rne(sum / len); vc = bf16_rne(sum); qbar = sum / len (fp32).
 *  - moments: 8 fp32 partials over blocks j = g (mod 8), ascending, combined
 *    ((p0+p1)+(p2+p3)) + ((p4+p5)+(p6+p7)); no FMA.
 *  - routing score R[i][j] = (fmaf chain over d of qbar_i[d] * kc_j[d]) * c,
 *    c = scale * 1.4426950408889634f; thresholds as documented per function.
 */
#ifndef SOLATTN_H
#define SOLATTN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

typedef struct ihipStream_t* solattn_stream_t; /* == hipStream_t */

enum {
  SOLATTN_OK = 0,
  SOLATTN_EINVAL = -1,    /* bad argument (shape, stride, null pointer) */
  SOLATTN_EUNSUPPORTED = -2, /* valid but not implemented (e.g. head_dim != 128) */
  SOLATTN_ELAUNCH = -3,   /* HIP launch error */
  SOLATTN_ESIZE = -4      /* buffer too small */
};

enum { SOLATTN_CURVE_3D = 0, SOLATTN_CURVE_2D_FRAME = 1 };

/* int8_pv of the INT8 entry points: how P.V runs (solattn_fwd_int8). */
enum {
  SOLATTN_PV_BF16 = 0,         /* bf16 P against bf16 v */
  SOLATTN_PV_INT8 = 1,         /* int8 codes against each routed block's row max */
  SOLATTN_PV_INT8_RUNNING = 2  /* int8 codes against the row's running max */
};

/* Message for the last failing call on this thread ("" if none). */
const char* solattn_last_error(void);
/* ABI version: (major << 16) | minor. */
int solattn_abi_version(void);

/* ---------------------------------------------------------------- Morton --
 * Host function (no device work). Z-order permutation of a frames x height x
 * width latent grid laid out frame-major, then row-major, and its inverse.
 * curve SOLATTN_CURVE_3D interleaves x, y, t bits; SOLATTN_CURVE_2D_FRAME keeps
 * the frame index as the most significant key. roll != 0 rotates perm by roll
 * places (torch.roll semantics) before the inverse is taken.
 * perm/inverse: host int64 arrays of frames*height*width entries.
 * Replaces: morton_perm, /root/reference/_morton.py:35-73, and the span roll of
 * _perm_for, /root/reference/_morton_h3.py:42-61. */
int solattn_morton_perm(int64_t frames, int64_t height, int64_t width, int curve,
                        int64_t roll, int64_t* perm, int64_t* inverse);

/* --------------------------------------------------------------- reorder --
 * Row gather: dst[b, t, :] = src[b, index[t], :] for t < rows, b < batch.
 * A row is row_bytes contiguous bytes (row_bytes % 16 == 0, 16-byte aligned
 * rows). index: device int64 [rows], each entry in [0, src_rows).
 * Replaces: the torch index_select / fancy-index gathers of the Morton hooks,
 * /root/reference/_morton.py:113,128,148 and /root/reference/_morton_h3.py:193,217. */
int solattn_reorder_rows(const void* src, int64_t src_rows, int64_t src_stride_b_bytes,
                         int64_t src_stride_row_bytes, void* dst, int64_t dst_stride_b_bytes,
                         int64_t dst_stride_row_bytes, int64_t batch, int64_t rows,
                         int64_t row_bytes, const int64_t* index, solattn_stream_t stream);

/* ------------------------------------------------------------------ pool --
 * One pass over q, k and v per (batch, block, head):
 *   kc[b, j, h, :] = bf16_rne(sum_k / len_j)      kc, vc: bf16 [B, npad, H, D]
 *   vc[b, j, h, :] = bf16_rne(sum_v)              (rows j >= NT are not written)
 *   qbar[b, h, j, :] = sum_q / len_j              qbar: fp32 [B, H, NT, D]
 *   vamax_part[b, j, h, :] = max_r |v|            fp32 [B, NT, H, D], may be NULL
 * Token strides must lie in [0, 2^26) elements and T <= 65535 * 128
 * (SOLATTN_EUNSUPPORTED otherwise).
 * Replaces: _reduce_kc_kernel / _reduce_vc_kernel / _reduce_kv,
 * /root/reference/_preprocess.py:23-113,172-224, and the Q centroid of
 * _diag_threshold_kernel (:144-149) / _q_quant_threshold_kernel
 * (/root/reference/_fused_prep.py:16-59). */
int solattn_pool(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                 const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                 const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                 int64_t B, int64_t T, int64_t H, int64_t D, int64_t block,
                 uint16_t* kc, uint16_t* vc, int64_t npad, float* qbar,
                 float* vamax_part, solattn_stream_t stream);

/* --------------------------------------------------------------- moments --
 * Per (b, h, d) over blocks j < NT, in ascending j:
 *   mean = (sum_j kc) / NT
 *   centre == 0 (BF16 path, /root/reference/_preprocess.py:241-243):
 *     var = (sum_j (kc - mean)^2) / NT
 *   centre == 1 (INT8 path, /root/reference/_fused_prep.py:77-81):
 *     kc[b, j, h, d] = bf16_rne(kc - mean) (in place); var = (sum_j kc'^2) / NT
 * kc_mean, kc_var: fp32 [B, H, D].
 * If vamax_part != NULL also vscale[b, h, d] = max(max_j vamax_part * (1/127)f, 1e-8)
 * (/root/reference/_fused_quant.py:102-105: torch divides by a scalar as a
 * multiply by its fp32 reciprocal). kc and vamax_part must be 16-byte aligned;
 * with vamax_part, H < 32768 (SOLATTN_EUNSUPPORTED otherwise). */
int solattn_moments(uint16_t* kc, int64_t npad, int64_t B, int64_t NT, int64_t H,
                    int64_t D, int centre, float* kc_mean, float* kc_var,
                    const float* vamax_part, float* vscale, solattn_stream_t stream);

/* ----------------------------------------------------------------- route --
 * Thresholds, routing decisions and per-query-block exact-block masks.
 *   mode 0 (BF16, /root/reference/_preprocess.py:150-163):
 *     mu  = (fmaf chain qbar*kc_mean) * c
 *     var = (fmaf chain (qbar*qbar)*kc_var) * (c*c)
 *     thr = mu + tau * sqrtf(fmaxf(var, 0) + 1e-6f)
 *   mode 1 (INT8, /root/reference/_fused_prep.py:50-59, kc already centred):
 *     thr = tau * sqrtf(var + 1e-6f)
 *   R[i][j] = (fmaf chain qbar_i*kc_j) * c
 *   exact(i, j) = i in [sink_q_lo, sink_q_hi) ? 1
 *               : R > thr || |i - j| <= 1 || j in [sink_kv_lo, sink_kv_hi)
 *   (the forward's rule, /root/reference/_tri_fwd.py:279-286).
 * Outputs: thr fp32 [B, NT, H]; counts int32 [B, H, NT] (exact blocks per
 * query block); mask uint32 [B, H, NT, ceil(NT/32)] (bit j%32 of word j/32 =
 * exact; bits j >= NT are 0). The reference keeps no list either: it re-derives
 * the decisions in every forward program. */
int solattn_route(const float* qbar, const uint16_t* kc, int64_t npad, const float* kc_mean,
                  const float* kc_var, int64_t B, int64_t T, int64_t H, int64_t D,
                  int64_t block, float scale, float tau, int mode, int64_t sink_kv_lo,
                  int64_t sink_kv_hi, int64_t sink_q_lo, int64_t sink_q_hi, float* thr,
                  int32_t* counts, uint32_t* mask, solattn_stream_t stream);

/* ----------------------------------------------------------------- quant --
 * Per-token INT8 of a BTHD bf16 tensor, optionally smoothed by mean [B, H, D]:
 *   y = x - mean; s = max|y| / 127; s = s > 1e-8 ? s : 1e-8
 *   code = clamp(y/s >= 0 ? trunc(y/s + 0.5) : trunc(y/s - 0.5), -127, 127)
 * xi: int8 [B, TP, H, D]; xs: fp32 [B, TP, H]; rows t >= T are not written.
 * Replaces: _quant_kernel / quantize_bthd, /root/reference/_fused_quant.py:8-58
 * (and the Q half of _q_quant_threshold_kernel, _fused_prep.py:42-48). */
int solattn_quant_rows(const uint16_t* x, int64_t sx_b, int64_t sx_t, int64_t sx_h,
                       int64_t B, int64_t T, int64_t H, int64_t D, const float* mean,
                       int8_t* xi, float* xs, int64_t TP, solattn_stream_t stream);

/* Tokens per scale of the per-block INT8 variant below. */
#define SOLATTN_QUANT_BLOCK 128

/* solattn_quant_rows with one scale per block of SOLATTN_QUANT_BLOCK tokens
 * (per batch and head) instead of one per token: s = max(fl(amax / 127),
 * 1e-8) with amax the |max| of y over the block's tokens and channels, the
 * same code rule, and s written to xs for every token of the block. No
 * counterpart in the reference, which quantises Q and K per token: this is
 * BASELINE config 3's "Q/K quantised per 128-token block" wording, reported
 * beside the per-token parity mode. */
int solattn_quant_rows_blocked(const uint16_t* x, int64_t sx_b, int64_t sx_t, int64_t sx_h,
                               int64_t B, int64_t T, int64_t H, int64_t D, const float* mean,
                               int8_t* xi, float* xs, int64_t TP, solattn_stream_t stream);

/* Per-channel INT8 of V with vscale fp32 [B, H, D]:
 *   code = clamp(round_half_away(v / vscale[d]), -127, 127); vi: int8 [B, TP, H, D].
 * Replaces: _quant_v_kernel / quantize_v_per_channel,
 * /root/reference/_fused_quant.py:61-113. */
int solattn_quant_v(const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B,
                    int64_t T, int64_t H, int64_t D, const float* vscale, int8_t* vi,
                    int64_t TP, solattn_stream_t stream);

/* ------------------------------------------------------ INT8 preparation --
 * Everything the INT8 forward reads, in four launches: pool with the per-token
 * Q codes from the same read, moments (centre = 1), route (mode 1), then the
 * smoothed K codes and (vscale != NULL, which also needs vamax_part and vi) the
 * V codes in one launch. The outputs and layouts are those of solattn_pool,
 * solattn_moments, solattn_route, solattn_quant_rows and solattn_quant_v with
 * TP = T, bit for bit; rows [NT, npad) of kc and vc are zeroed. qk_block != 0: Q
 * and K codes as solattn_quant_rows_blocked (Q is then read twice).
 * Replaces: fused_preprocess, /root/reference/_fused_prep.py:62-98. */
int solattn_preprocess_int8(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                            const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                            const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B,
                            int64_t T, int64_t H, int64_t D, int64_t block, float scale, float tau,
                            int64_t sink_kv_lo, int64_t sink_kv_hi, int64_t sink_q_lo,
                            int64_t sink_q_hi, int qk_block, uint16_t* kc, uint16_t* vc, int64_t npad,
                            float* qbar, float* kc_mean, float* kc_var, float* vamax_part,
                            float* vscale, float* thr, int32_t* counts, uint32_t* mask, int8_t* qi,
                            float* qs, int8_t* ki, float* ks, int8_t* vi, solattn_stream_t stream);

/* ------------------------------------------------------- single-read INT8 --
 * The INT8 path's preparation with one read of q, k and v: pooled keys and
 * values, query centroids, centred kc and its moments (solattn_moments with
 * centre = 1), the V scale, per-token Q codes, per-token K codes smoothed by
 * kc_mean and (vscale != NULL) per-channel V codes -- the outputs of
 * solattn_pool + solattn_moments + solattn_quant_rows / solattn_quant_v, bit
 * for bit. Each head's K and V rows stay in registers until its moments are
 * known: the launch is cooperative (all workgroups resident) and the
 * workgroups of a head meet at two barriers in device memory. Returns
 * SOLATTN_EUNSUPPORTED when fewer than two heads' rows fit on the device at
 * once (or D != 128); the caller then uses the two-pass entry points.
 * vamax_part: fp32 [B, NT, H, D] scratch (with vscale); ks: [B, H, TP]
 * (ks_head_major != 0) or [B, TP, H]; sync: device scratch of at least
 * solattn_prep_int8_sync_bytes(B, H) bytes, reset by the call itself; its
 * first uint32 is nonzero after the call only if a barrier was not met within
 * ~0.1 s (results then invalid), which cannot happen with every workgroup
 * resident.
 * Replaces: fused_preprocess, /root/reference/_fused_prep.py:62-98, which reads
 * K and V twice. */
int64_t solattn_prep_int8_sync_bytes(int64_t B, int64_t H);
int solattn_prep_int8(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                      const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                      const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B,
                      int64_t T, int64_t H, int64_t D, int64_t block, uint16_t* kc,
                      uint16_t* vc, int64_t npad, float* qbar, float* kc_mean, float* kc_var,
                      float* vamax_part, float* vscale, int8_t* qi, float* qs, int8_t* ki,
                      float* ks, int ks_head_major, int8_t* vi, int64_t TP, void* sync,
                      int64_t sync_bytes, solattn_stream_t stream);

/* ------------------------------------------------------------- forwards --
 * Sparse attention over exact blocks (flash attention on MFMA) plus the pooled
 * branch (one pooled key kc_j and value vc_j per approximate block, softmax
 * weight times len_j), one online softmax per query row.
 * counts/mask come from solattn_route for the same B, T, H and block. Each
 * workgroup builds its tile list from its mask row (mask bits at or past NT
 * are ignored, so any mask contents stay inside the tensors); counts only
 * order the dispatch (longest query blocks first). o: bf16, element
 * (b, t, h, d) at o + b*so_b + t*so_t + h*so_h + d, 16-byte aligned with
 * strides multiples of 8 elements (rows are written as 16-byte stores); rows
 * t >= T are not written.
 * Replaces: _forward_ptr + sol_attn, /root/reference/_tri_fwd.py:215-410. */
int solattn_fwd_bf16(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                     const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                     const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                     const uint16_t* kc, const uint16_t* vc, int64_t npad,
                     const int32_t* counts, const uint32_t* mask,
                     int64_t B, int64_t T, int64_t H, int64_t D, int64_t block, float scale,
                     uint16_t* o, int64_t so_b, int64_t so_t, int64_t so_h,
                     solattn_stream_t stream);

/* INT8 exact branch: S = int32(qi . ki) * (qs * c) * ks. int8_pv ==
 * SOLATTN_PV_BF16 runs P.V in bf16 against v, with P rounded to bf16 as in
 * solattn_fwd_bf16.
 * SOLATTN_PV_INT8 quantises P per row against the row max of each routed block:
 *   code = v_cvt_pk_u8_f32(exp2(s + log2(127) - rowmax_blk))
 * i.e. round to nearest, ties to even, of 127 * exp2(s - rowmax_blk) (at most
 * 127 by construction); the products int32(code . vi) are scaled by
 * (beta / 127) * vscale[d] with beta = exp2(rowmax_blk - m). The softmax
 * denominator adds the integer codes themselves, times beta / 127, so it is
 * the sum of the quantised P that the P.V multiplies.
 * Deliberate departures from /root/reference/_int8_fwd.py:348-353, which
 * rounds trunc(pe * 127 + 0.5) and sums the fp32 pe: the rounding rule and the
 * code-sum denominator (both within the INT8 tolerance, cosine >= 0.999), and,
 * at block 128, a ragged last block whose tiles take the max of each 64-key
 * tile instead of the whole block's.
 * SOLATTN_PV_INT8_RUNNING quantises P against the row's running max instead,
 * an integer m_int (log2 domain) at or above every scaled score seen:
 *   code = v_cvt_pk_u8_f32(exp2(s + log2(127) - m_int))
 * so the products of all exact blocks accumulate in int32 with no per-block
 * conversion; a block whose row max exceeds m_int raises it to ceil(max),
 * shifts the int32 sums right by the difference (floor) and scales the code
 * sum, kept in fp32, by the same power of two (exact); when a lane's half of
 * a row's code sum exceeds 2^23, m_int rises by one more, so the sums (at
 * most 127 times the code sum) stay below 2^31. After the exact blocks O = sums * vscale[d] / 127 and l = code sum /
 * 127, relative to 2^m_int. Codes of blocks below the
 * running max are coarser than against their own max: a further departure
 * from the reference, within the INT8 tolerance (cosine >= 0.999 per query
 * block against the reference arithmetic).
 * The pooled branch is BF16 as above (q, kc, vc); routing inputs as for
 * solattn_fwd_bf16. qi/ki/vi int8 [B, TP, H, D]; qs/ks fp32 [B, TP, H].
 * Replaces: _forward_int8_ptr + sol_attn_int8, /root/reference/_int8_fwd.py:208-432. */
int solattn_fwd_int8(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                     const int8_t* qi, const float* qs, const int8_t* ki, const float* ks,
                     const int8_t* vi, const float* vscale, const uint16_t* v, int64_t sv_b,
                     int64_t sv_t, int64_t sv_h, int64_t TP, const uint16_t* kc,
                     const uint16_t* vc, int64_t npad, const int32_t* counts,
                     const uint32_t* mask, int64_t B, int64_t T,
                     int64_t H, int64_t D, int64_t block, float scale, int int8_pv,
                     uint16_t* o, int64_t so_b, int64_t so_t, int64_t so_h,
                     solattn_stream_t stream);

/* ------------------------------------------------------ whole pipeline --
 * sol_attn in one call: pool -> moments -> route -> fwd_bf16, with every
 * intermediate carved out of a caller-owned device workspace of at least
 * solattn_sol_attn_workspace_bytes(...) bytes (256-byte aligned base).
 * Replaces: sol_attn, /root/reference/_tri_fwd.py:354-410. */
int64_t solattn_sol_attn_workspace_bytes(int64_t B, int64_t T, int64_t H, int64_t D,
                                         int64_t block, int int8);
int solattn_sol_attn(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                     const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                     const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                     int64_t B, int64_t T, int64_t H, int64_t D, int64_t block,
                     float scale, float tau, int64_t sink_kv_lo, int64_t sink_kv_hi,
                     int64_t sink_q_lo, int64_t sink_q_hi, void* workspace,
                     int64_t workspace_bytes, uint16_t* o, int64_t so_b, int64_t so_t,
                     int64_t so_h, solattn_stream_t stream);

/* sol_attn_int8 in one call: pool -> moments(centre) -> route(mode 1) ->
 * quant(q, k smoothed, v) -> fwd_int8. Replaces: sol_attn_int8,
 * /root/reference/_int8_fwd.py:379-432. */
int solattn_sol_attn_int8(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                          const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                          const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                          int64_t B, int64_t T, int64_t H, int64_t D, int64_t block,
                          float scale, float tau, int64_t sink_kv_lo, int64_t sink_kv_hi,
                          int64_t sink_q_lo, int64_t sink_q_hi, int int8_pv,
                          void* workspace, int64_t workspace_bytes, uint16_t* o,
                          int64_t so_b, int64_t so_t, int64_t so_h,
                          solattn_stream_t stream);

/* solattn_sol_attn_int8 with Q and smoothed K quantised per
 * SOLATTN_QUANT_BLOCK-token block (solattn_quant_rows_blocked) instead of per
 * token; V, routing and the forward as there. No counterpart in the
 * reference: the config 3 variant above. */
int solattn_sol_attn_int8_qblock(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                                 const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                                 const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                                 int64_t B, int64_t T, int64_t H, int64_t D, int64_t block,
                                 float scale, float tau, int64_t sink_kv_lo, int64_t sink_kv_hi,
                                 int64_t sink_q_lo, int64_t sink_q_hi, int int8_pv,
                                 void* workspace, int64_t workspace_bytes, uint16_t* o,
                                 int64_t so_b, int64_t so_t, int64_t so_h,
                                 solattn_stream_t stream);

/* ------------------------------------------------ allocation-free BF16 --
 * solattn_sol_attn without a workspace argument, for callers that cannot
 * allocate device memory (code under HIP graph capture, serving loops and
 * harnesses that forbid hipMalloc). No counterpart in the reference: it exists
 * for those callers only. The intermediates live in one fixed array of
 * SOLATTN_NOALLOC_SCRATCH_BYTES per device (held from the library's first use
 * on that device until the process ends); shapes whose intermediates exceed it
 * (solattn_sol_attn_workspace_bytes(B, T, H, D, block, 0) >
 * SOLATTN_NOALLOC_SCRATCH_BYTES) return SOLATTN_ESIZE. Every call on one
 * device shares that array: calls that overlap on one device (different
 * streams, or threads without ordering) race and must be serialised by the
 * caller. Nothing in the array needs clearing between calls. Same arguments,
 * results and errors as solattn_sol_attn otherwise; the device is the current
 * one. 32 MiB covers a B1 H40 T75600 call at block 128 (26 MiB) and a B1 H24
 * T32760 call at either block size (13 MiB at block 64). */
#define SOLATTN_NOALLOC_SCRATCH_BYTES (32ll << 20)
int solattn_sol_attn_noalloc(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h,
                             const uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                             const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
                             int64_t B, int64_t T, int64_t H, int64_t D, int64_t block,
                             float scale, float tau, int64_t sink_kv_lo, int64_t sink_kv_hi,
                             int64_t sink_q_lo, int64_t sink_q_hi, uint16_t* o, int64_t so_b,
                             int64_t so_t, int64_t so_h, solattn_stream_t stream);

/* ------------------------------------------------ operators around attention --
 * Norms and rotation of queries and keys, sliding-window attention with sinks
 * and attention of one new token over a paged cache: no counterpart in the
 * reference. q, o: BTHD with H query heads; k, v: BTHD with Hkv kv heads, each
 * shared by the H / Hkv query heads behind one another (H % Hkv == 0). Rows
 * (the last dim) are contiguous, 16-byte aligned, and every stride keeps them
 * so; strides may be 0 for inputs, token strides below 2^24 elements. Sums, softmax statistics and
 * accumulators are fp32; outputs are rounded once. */
enum { SOLATTN_BF16 = 0, SOLATTN_FP16 = 1, SOLATTN_FP32 = 2 }; /* dtype arguments */
enum { SOLATTN_INT8 = 1, SOLATTN_E4M3 = 2 };                   /* cache_type arguments */

/* Per (batch, token, head) row x of q and k, D channels (a multiple of 8 up to 128):
 *   n = x / sqrt(mean(x^2) + eps) * weight        (weight null: 1)
 *   y[i1] = n[i1] cos - n[i2] sin, y[i2] = n[i2] cos + n[i1] sin for the R / 2 pairs
 *   of the first R channels, (i, i + R/2), or (2i, 2i + 1) when interleaved; the
 *   other channels are n. R: a multiple of 16 (interleaved: 8), 0 for none.
 * cos, sin: fp32 [P][R/2] by position. positions: int32 [B][T] with row stride
 * pos_stride_b (0: shared), clamped to [0, P); null: token t is at t (T <= P).
 * weights: fp32 [D]. dtype of q, k and the outputs: any SOLATTN_*; weights and
 * tables 16-byte aligned. Hkv may be 0 (q alone). Outputs may be the inputs. */
int solattn_qk_norm_rope(const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k,
                         int64_t sk_b, int64_t sk_t, int64_t sk_h, int64_t B, int64_t T, int64_t H,
                         int64_t Hkv, int64_t D, int dtype, const float* q_weight,
                         const float* k_weight, const float* cos, const float* sin, int64_t P,
                         int64_t R, int interleaved, const int32_t* positions,
                         int64_t pos_stride_b, float eps, void* qo, int64_t sqo_b, int64_t sqo_t,
                         int64_t sqo_h, void* ko, int64_t sko_b, int64_t sko_t, int64_t sko_h,
                         solattn_stream_t stream);

/* The same for the newest T tokens of sequences of lengths[b] tokens (these
 * included): token t is at position lengths[b] - T + t; its k goes, turned, and its
 * v as it is, to slot position % page_size of page page_table[b][position /
 * page_size]. k_cache, v_cache: [pages][page_size][Hkv][D] with the strides given.
 * Tokens before position 0, past the table, or whose page id is not in
 * [0, pages) are not written (their rows of qo are finite but mean nothing). No two
 * tokens of a call may have the same slot of the same page: it holds a mixture of both then. */
int solattn_qk_norm_rope_append(
    const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_b,
    int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B,
    int64_t T, int64_t H, int64_t Hkv, int64_t D, int dtype, const float* q_weight,
    const float* k_weight, const float* cos, const float* sin, int64_t P, int64_t R, int interleaved,
    float eps, void* qo, int64_t sqo_b, int64_t sqo_t, int64_t sqo_h, void* k_cache, int64_t skc_p,
    int64_t skc_s, int64_t skc_h, void* v_cache, int64_t svc_p, int64_t svc_s, int64_t svc_h,
    int64_t pages, int64_t page_size, const int32_t* page_table, int64_t table_stride,
    int64_t max_pages, const int32_t* lengths, solattn_stream_t stream);

/* Gradients of solattn_qk_norm_rope: dq, dk from the inputs q, k and the outputs'
 * gradients dqo, dko; dq_weight, dk_weight: fp32 [D], null to leave out (with either,
 * a 256-byte aligned workspace of the size below; the order of every sum is fixed). */
int64_t solattn_qk_norm_rope_bwd_workspace_bytes(int64_t D);
int solattn_qk_norm_rope_bwd(
    const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_b,
    int64_t sk_t, int64_t sk_h, const void* dqo, int64_t sdq_b, int64_t sdq_t, int64_t sdq_h,
    const void* dko, int64_t sdk_b, int64_t sdk_t, int64_t sdk_h, int64_t B, int64_t T, int64_t H,
    int64_t Hkv, int64_t D, int dtype, const float* q_weight, const float* k_weight, const float* cos,
    const float* sin, int64_t P, int64_t R, int interleaved, const int32_t* positions,
    int64_t pos_stride_b, float eps, void* dq, int64_t sgq_b, int64_t sgq_t, int64_t sgq_h, void* dk,
    int64_t sgk_b, int64_t sgk_t, int64_t sgk_h, float* dq_weight, float* dk_weight, void* workspace,
    int64_t workspace_bytes, solattn_stream_t stream);

/* Row t of q sits at position p = q_start + t (q_start + Tq <= Tk) and sees the keys
 *   causal:    j <= p and (p - j < window or j < sinks)
 *   otherwise: |p - j| < window or j < sinks
 * of j < len, len = lengths[b] clamped to [0, Tk] (int32 [B]; null: Tk).
 *   o = sum_j softmax_j(scale q.k_j) v_j; rows at p >= len are zeros.
 * lse: fp32 [B][H][Tq], log2 of the row's softmax sum (+inf for a row without keys),
 * what the backward reads; null: not written. o_lo: [B][Tq][H][D] of dtype, what
 * rounding o took away, rounded itself, for a backward of full precision; null: not
 * written. dtype bf16 or fp16, D 64 or 128
 * (D: multiples of 8 up to 128 for the call below). Keys that no row of a call sees
 * are never read; what k holds at a key reaches the rows that see it only, but a
 * NaN or infinity in v (backward: also in k, q, do) can reach rows that do not see
 * it within the same 128 rows.
 * workspace: 256-byte aligned, of the size below (0: may be null; enough with and
 * without lengths): short launches run split over the keys, one causal row per sequence
 * without lse as solattn_paged_attn. */
int64_t solattn_window_attn_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv,
                                            int64_t D, int64_t q_start, int64_t window, int64_t sinks,
                                            int causal, int with_lse);
int solattn_window_attn(const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const uint16_t* k,
                        int64_t sk_b, int64_t sk_t, int64_t sk_h, const uint16_t* v, int64_t sv_b,
                        int64_t sv_t, int64_t sv_h, int64_t B, int64_t Tq, int64_t Tk, int64_t H,
                        int64_t Hkv, int64_t D, int dtype, int64_t q_start, const int32_t* lengths,
                        int64_t window, int64_t sinks, int causal, float scale, uint16_t* o,
                        int64_t so_b, int64_t so_t, int64_t so_h, float* lse, uint16_t* o_lo, void* workspace,
                        int64_t workspace_bytes, solattn_stream_t stream);

/* Gradients of solattn_window_attn from its inputs, o, lse, o_lo (or null) and do: dq like q, dk and dv
 * like k (every row written, zeros where nothing is seen). P and dS are rounded to
 * dtype, in two parts where the call's rows see fewer than 512 keys, all of them fewer
 * than 1024, or there are fewer than 128 rows (lengths are not looked at). workspace:
 * 256-byte aligned. No atomics: the same inputs give the same bits. */
int64_t solattn_window_attn_bwd_workspace_bytes(int64_t B, int64_t Tq, int64_t Tk, int64_t H, int64_t Hkv,
                                                int64_t D, int64_t window, int64_t sinks, int causal);
int solattn_window_attn_bwd(
    const uint16_t* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const uint16_t* k, int64_t sk_b,
    int64_t sk_t, int64_t sk_h, const uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h,
    const uint16_t* o, int64_t so_b, int64_t so_t, int64_t so_h, const uint16_t* d_o, int64_t sg_b,
    int64_t sg_t, int64_t sg_h, const float* lse,
    const uint16_t* o_lo, int64_t B, int64_t Tq, int64_t Tk, int64_t H,
    int64_t Hkv, int64_t D, int dtype, int64_t q_start, const int32_t* lengths, int64_t window,
    int64_t sinks, int causal, float scale, uint16_t* dq, int64_t sdq_b, int64_t sdq_t, int64_t sdq_h,
    uint16_t* dk, int64_t sdk_b, int64_t sdk_t, int64_t sdk_h, uint16_t* dv, int64_t sdv_b,
    int64_t sdv_t, int64_t sdv_h, void* workspace, int64_t workspace_bytes, solattn_stream_t stream);

/* One new token of each sequence, the last of its lengths[b] (int32 [B], clamped to
 * [0, max_pages page_size]): o[b][h] over the keys j < len, with a window (0: none)
 * those of j >= len - window or j < sinks. Key j is slot j % page_size of page
 * page_table[b][j / page_size] of k_cache, v_cache [pages][page_size][Hkv][D]
 * (strides given; page_size a multiple of 8); keys of a page id outside
 * [0, pages) are not visible. A sequence without visible keys gives zeros. Slots
 * behind a sequence's last key may hold anything. dtype bf16 or fp16, D a multiple
 * of 8 up to 128. workspace: 256-byte aligned, of the size below (0: may be null). */
int64_t solattn_paged_attn_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages,
                                           int64_t page_size, int64_t window, int64_t sinks);
int solattn_paged_attn(const uint16_t* q, int64_t sq_b, int64_t sq_h, const uint16_t* k_cache, int64_t sk_p,
                       int64_t sk_s, int64_t sk_h, const uint16_t* v_cache, int64_t sv_p, int64_t sv_s,
                       int64_t sv_h, int64_t pages, int64_t page_size, const int32_t* page_table,
                       int64_t table_stride, int64_t max_pages, const int32_t* lengths, int64_t B,
                       int64_t H, int64_t Hkv, int64_t D, int dtype, int64_t window, int64_t sinks,
                       float scale, void* workspace, int64_t workspace_bytes, uint16_t* o, int64_t so_b,
                       int64_t so_h, solattn_stream_t stream);

/* ------------------------------------------------------- caches of 8 bits --
 * A cache k_cache, v_cache [pages][page_size][Hkv][D] of codes (cache_type SOLATTN_INT8:
 * two's complement; SOLATTN_E4M3: four bits of exponent, three of mantissa, no
 * infinities) with k_scale, v_scale [pages][Hkv][page_size], an exponent byte b for each
 * row: a value is code 2^(b - 127). Codes' rows are 16-byte aligned and every stride
 * keeps them so (D a multiple of 16 up to 128); scales' last dim is contiguous, their
 * strides are those of pages and heads.
 * Written rows: the smallest power of two that keeps the row's largest magnitude within
 * 127 or 448 (below 2^-110: a row of zeros), codes rounded to nearest even. A row that
 * holds a NaN or an infinity reads as NaN in every channel. Its byte is
 * 255, with codes 0 or e4m3's NaN; zeros have byte 0 and codes 0. Other codes beside these
 * two bytes mean nothing.
 * A value is exact in 16 bits: in bf16, and in fp16 within fp16's range. An fp16 read, and
 * an fp16 call over shared keys, may round values below 2^-14; a read rounds those from
 * 65520 on to infinities, a call takes them as they are.
 *
 * solattn_qk_norm_rope_append with such a cache; k' is rounded once, from fp32. */
int solattn_qk_norm_rope_append8(
    const void* q, int64_t sq_b, int64_t sq_t, int64_t sq_h, const void* k, int64_t sk_b,
    int64_t sk_t, int64_t sk_h, const void* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B,
    int64_t T, int64_t H, int64_t Hkv, int64_t D, int dtype, const float* q_weight,
    const float* k_weight, const float* cos, const float* sin, int64_t P, int64_t R, int interleaved,
    float eps, void* qo, int64_t sqo_b, int64_t sqo_t, int64_t sqo_h, void* k_cache, int64_t skc_p,
    int64_t skc_s, int64_t skc_h, void* v_cache, int64_t svc_p, int64_t svc_s, int64_t svc_h,
    int64_t pages, int64_t page_size, int cache_type, uint8_t* k_scale, int64_t sks_p, int64_t sks_h,
    uint8_t* v_scale, int64_t svs_p, int64_t svs_h, const int32_t* page_table, int64_t table_stride,
    int64_t max_pages, const int32_t* lengths, solattn_stream_t stream);

/* k and v [B][T][Hkv][D] (any dtype), the newest T tokens of sequences of lengths[b]
 * tokens, as they are: what solattn_qk_norm_rope_append8 does of k' and v, with its rule
 * of the places. */
int solattn_cache_append(const void* k, int64_t sk_b, int64_t sk_t, int64_t sk_h, const void* v,
                         int64_t sv_b, int64_t sv_t, int64_t sv_h, int64_t B, int64_t T, int64_t Hkv,
                         int64_t D, int dtype, void* k_cache, int64_t skc_p, int64_t skc_s,
                         int64_t skc_h, void* v_cache, int64_t svc_p, int64_t svc_s, int64_t svc_h,
                         int64_t pages, int64_t page_size, int cache_type, uint8_t* k_scale,
                         int64_t sks_p, int64_t sks_h, uint8_t* v_scale, int64_t svs_p, int64_t svs_h,
                         const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                         const int32_t* lengths, solattn_stream_t stream);

/* Row t of k and v [B][T][Hkv][D] (bf16 or fp16) becomes key start[b] + t of sequence b
 * (start null: t); zeros where that is not in [0, lengths[b]), past the table, or on a
 * page id outside [0, pages). */
int solattn_cache_read(const void* k_cache, int64_t skc_p, int64_t skc_s, int64_t skc_h,
                       const void* v_cache, int64_t svc_p, int64_t svc_s, int64_t svc_h, int64_t pages,
                       int64_t page_size, int cache_type, const uint8_t* k_scale, int64_t sks_p,
                       int64_t sks_h, const uint8_t* v_scale, int64_t svs_p, int64_t svs_h,
                       const int32_t* page_table, int64_t table_stride, int64_t max_pages,
                       const int32_t* lengths, const int32_t* start, int64_t B, int64_t T, int64_t Hkv,
                       int64_t D, int dtype, uint16_t* k, int64_t sk_b, int64_t sk_t, int64_t sk_h,
                       uint16_t* v, int64_t sv_b, int64_t sv_t, int64_t sv_h, solattn_stream_t stream);

/* solattn_paged_attn with a cache of codes (cache_type 0: of dtype, scales null;
 * page_size and scales' strides multiples of 8, scales 8-byte aligned), and for batches
 * whose sequences have keys in common: of each of `groups` runs of B / groups sequences
 * the first `shared` keys are the same, and are read once, from the pages of the run's
 * longest sequence (the first of these); the other sequences' pages for them are not
 * looked at; a sequence that is shorter than `shared` sees lengths[b] of them. With
 * shared > 0: no window. */
int64_t solattn_paged_attn_shared_workspace_bytes(int64_t B, int64_t H, int64_t Hkv, int64_t D, int64_t max_pages,
                                            int64_t page_size, int64_t window, int64_t sinks,
                                            int cache_type, int64_t shared, int64_t groups);
int solattn_paged_attn_shared(const uint16_t* q, int64_t sq_b, int64_t sq_h, const void* k_cache, int64_t sk_p,
                        int64_t sk_s, int64_t sk_h, const void* v_cache, int64_t sv_p, int64_t sv_s,
                        int64_t sv_h, int64_t pages, int64_t page_size, int cache_type,
                        const uint8_t* k_scale, int64_t sks_p, int64_t sks_h, const uint8_t* v_scale,
                        int64_t svs_p, int64_t svs_h, const int32_t* page_table, int64_t table_stride,
                        int64_t max_pages, const int32_t* lengths, int64_t B, int64_t H, int64_t Hkv,
                        int64_t D, int dtype, int64_t window, int64_t sinks, int64_t shared,
                        int64_t groups, float scale, void* workspace, int64_t workspace_bytes, uint16_t* o,
                        int64_t so_b, int64_t so_h, solattn_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* SOLATTN_H */
