/* Elementwise test entry points next to the fused CE (names and signatures of the reference's
 * src/kernels/elementwise/capi_ew.h:22,29-30,36). Conventions as in capi.h. */
#ifndef MARINCPP_CAPI_EW_H
#define MARINCPP_CAPI_EW_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

int64_t nm_norm_partial_rows(int64_t T);
/* out[col] (+)= fixed-order sum over n_blocks partial rows [n_blocks, width]; round_bf16 rounds the reduced value */
int nm_reduce_partials_rows(const float* partial, int n_blocks, int width, float* out, int accumulate, int round_bf16,
                            void* stream);
/* out[0] = sum(x[0..n)) in a fixed order (the trainer sums the CE's loss_partial slots with it) */
int nm_sum_fixed(const float* x, int64_t n, float* out, void* stream);
/* raw partials of the RMSNorm backward ([nm_norm_partial_rows(T), D] f32) */
int nm_rmsnorm_bwd_add_partial(int dtype, int rounding, const void* dy, const void* x, const void* gain,
                               const float* rstd, const void* dres, void* dx, float* dgain_partial, int64_t T, int D,
                               float eps, void* stream);

/* The sandwich tail backward with raw gain-gradient partials ([nm_norm_partial_rows(T), D] f32 each, nullptr: skipped),
 * as the trainer calls it with buffers of its memory plan; nm_sandwich_tail_bwd (capi.h) is the same kernel followed by
 * the fixed-order reduction of the partials. */
int nm_sandwich_tail_bwd_partial(int dtype, int rounding, const void* dx_out, const void* da_next, const void* x_out,
                                 const void* g_next, const float* rstd_next, const void* branch, const void* g_post,
                                 const float* rstd_post, void* dx_in, void* dbranch, float* pg_next, float* pg_post,
                                 int64_t T, int D, float eps, void* stream);
/* The norm backward kernels (nm_rmsnorm_bwd_add, nm_rmsnorm_bwd_add_partial, nm_sandwich_tail_bwd) stage their operands
 * through a ring in shared memory whose waits are bounded; one that ran out leaves a bit in a per-GPU word built into the
 * library. This reads the word after the stream's work (it synchronises the stream), clears it when set, and returns
 * NM_ERR_DEVICE with the bits in *status_host when it was not 0. */
int nm_norm_bwd_device_status(void* stream, uint32_t* status_host);
/* Test hook: a millisecond-bounded wait on a barrier that nothing completes (limit_cycles <= 2e6), pointed at that word:
 * afterwards nm_norm_bwd_device_status reports what a kernel whose wait ran out would have left. */
int nm_norm_bwd_test_timeout(int64_t limit_cycles, void* stream);

/* ---- embedding (the reference's trunk has its own, src/kernels/elementwise/embed.cu; names and workspace here are this
 * library's). dtype: storage of table / out / dy, 1 = bf16, 0 = f32. D % 8 == 0, D <= 65536, rows contiguous and
 * 16-byte aligned.
 * forward:  out[t, :] = round(scale * table[tokens[t], :]), the f32 product rounded to the storage; a token outside [0, V)
 * gives a row of zeros. */
int nm_embed_fwd(int dtype, const void* table, const int32_t* tokens, void* out, float scale, int64_t T, int D, int V,
                 void* stream);
/* backward: dtable[v, :] (f32 [V, D]) = or += scale * sum over t with tokens[t] = v of dy[t, :]. accumulate 0 writes all
 * V rows (zeros for absent tokens), 1 adds and leaves absent rows untouched (a tied head's dW may be the buffer); tokens
 * outside [0, V) contribute nothing. Sums are f32 in an order that depends on the tokens alone: the same call gives the
 * same bits. With accumulate a row's sum is added at L2, where values below 2^-126 count as 0. workspace:
 * nm_embed_bwd_workspace_bytes (0 on error; does not fall as T grows, so that of the longest call serves all), 256-byte
 * aligned, scratch between calls; calls that may overlap need one each. Nothing is allocated; the calls can be captured
 * into a CUDA graph. */
uint64_t nm_embed_bwd_workspace_bytes(int64_t T, int D, int V);
int nm_embed_bwd(int dtype, const void* dy, const int32_t* tokens, float* dtable, float scale, int accumulate, int64_t T,
                 int D, int V, void* workspace, uint64_t workspace_bytes, void* stream);

/* ---- gated sandwich tail: the norms before and after a block, fused with the block's gate and the scaled residual (the
 * ungated tail is nm_sandwich_tail_fwd / _bwd, capi.h). dtype: storage of the row tensors, the gate and the gains, 1 = bf16
 * (D <= 8192), 0 = f32 (D <= 4096); D % 8 == 0, rows contiguous, pointers 16-byte aligned (a gate per token: its element
 * size). f32 inside, one rounding per stored output.
 *   y = g_post ? g_post * branch * rstd_post : branch        rstd_post = 1 / sqrt(mean(branch^2) + eps)
 *   x_out = round(res_scale * x_in + sigmoid(gate) * y)      gate_kind 0: no gate (NULL), 1: gate [T], 2: gate [T, D]
 *   a_next = round(g_next * x_out * rstd_next)               rstd_next = 1 / sqrt(mean(x_out^2) + eps), of the rounded x_out
 * NULL: res_scale ([D]; 1), g_post ([D]; no post-norm, and rstd_post is left as it was), a_next (then g_next too),
 * rstd_post / rstd_next (not returned). Statistics and [D] gradients are 4-byte aligned.
 * x_out may be x_in and a_next may be branch. */
int nm_gated_tail_fwd(int dtype, int gate_kind, const void* branch, const void* x_in, const void* gate,
                      const void* res_scale, const void* g_post, const void* g_next, void* x_out, void* a_next,
                      float* rstd_post, float* rstd_next, int64_t T, int D, float eps, void* stream);
/* Gradients of dx_out (gradient that reaches x_out from elsewhere; NULL: none) and da_next with respect to x_in, branch,
 * gate (dgate, same shape), and, each f32 [D] and overwritten, NULL to skip: g_next, g_post, res_scale. x_in, branch, gate,
 * the gains and the statistics are those of the forward call (x_out is formed again and not needed). dx_in may be dx_out,
 * dbranch may be branch, dgate may be gate. Sums have a fixed order: the same call gives the same bits. workspace
 * (nm_gated_tail_workspace_bytes, 0 on error; not needed when no [D] gradient is asked for): scratch between calls; calls
 * that may overlap need one each. Nothing is allocated. Waits of these two kernels are bounded: nm_norm_bwd_device_status
 * reports one that ran out; make the first call on a device outside a stream capture. */
uint64_t nm_gated_tail_workspace_bytes(int64_t T, int D);
int nm_gated_tail_bwd(int dtype, int gate_kind, const void* dx_out, const void* da_next, const void* x_in,
                      const void* branch, const void* gate, const void* res_scale, const void* g_post, const void* g_next,
                      const float* rstd_post, const float* rstd_next, void* dx_in, void* dbranch, void* dgate,
                      float* dg_next, float* dg_post, float* dres_scale, int64_t T, int D, void* workspace,
                      uint64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif
