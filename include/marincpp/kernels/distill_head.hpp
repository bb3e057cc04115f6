// Distillation head: the fused LM head trained on a teacher's top logits, optionally mixed with the hard targets.
//
// For row t with hidden state x_t, z = x_t W^T (never held for more than one chunk of rows), temperature tau, listed teacher
// entries (id_k, t_k), k < K:
//   q_k = exp(t_k / tau - n_t),  n_t = teacher_lse[t] when given, else log sum_k exp(t_k / tau)  (the list renormalised)
//   kl_t = sum_k q_k (log q_k - log p_tau[id_k]),  p_tau = softmax(z / tau) over the whole vocabulary
//   loss_t = soft_weight tau^2 kl_t + hard_weight (lse(z) - z[target_t])
//   n_t = soft_weight tau ((sum_k q_k) p_tau - q) + hard_weight (p_1 - onehot(target_t))     (gradient of loss_t wrt z)
//   dX[t] (+)= grad_scale weight_t n_t W;   dW += grad_scale sum_t weight_t n_t^T x_t
// With teacher_lse (log sum over the teacher's whole vocabulary of exp(. / tau)) the q_k keep their true mass and kl_t is the
// listed part of the divergence. An entry whose id lies outside [0, V) is padding: its logit is not looked at. Ids may repeat
// within a row (their masses add). A row without entries has no soft term, a row whose target lies outside [0, V) or equals
// ignore_index no hard term, a row of weight 0 neither loss nor gradient; its x must be finite all the same where dW is asked
// for (0 x_t is taken, as in the fused head).
// Precision: the logits, statistics and losses are f32. n is held as two bf16 terms (2^-17 of it): dW takes both and adds at most
// 1152 rows in one (truncating) accumulator, 2e-6 to 4e-6 from float64 in the 2-norm. dX, stored in bf16, takes both in chunks of
// up to 128 rows (1.7e-3, the storage itself) and the first alone, n rounded to bf16, in longer ones (2.3e-3): a row's dX depends
// in its last bit on the length of its chunk. One accumulator over a vocabulary of 128256 leaves dX 1.3e-4 small, four shares of
// it 3e-5.
// No counterpart in the reference, whose heads take hard targets only.
#pragma once

#include <cstdint>

#include "marincpp/core.hpp"

namespace nm {

struct DistillHeadShape {
  int64_t T;             // rows in the call
  int D, V;              // D a multiple of 8, V at most 2^30
  int K;                 // teacher entries per row, 1 .. 512
  int chunk_rows;        // min(T, chunk_rows) at most 2^30
  bool forward_only;     // no logits are stored: a much smaller workspace
};

struct DistillHeadArgs {
  const void* x;                     // [T, D] bf16
  const void* w;                     // [V, D] bf16
  const int32_t* teacher_ids;        // [T, K]
  const void* teacher_logits;        // [T, K]
  DType teacher_dtype;               // bf16 or f32
  const float* teacher_lse;          // [T] or nullptr
  const int32_t* targets;            // [T]; may be nullptr when hard_weight is 0
  const float* weight;               // [T]
  const float* grad_scale;           // device scalar; a gradient call needs it
  float temperature;                 // > 0
  float soft_weight, hard_weight;    // >= 0
  float* loss_tok;                   // [T]
  float* kl_tok;                     // [T] or nullptr
  float* lse;                        // [T] or nullptr: log sum exp(z / tau)
  float* loss_partial;               // [ceil(T / chunk_rows)] or nullptr: sum of weight * loss per chunk
  void* dx;                          // [T, D] bf16 or nullptr; may be x unless accumulated
  bool accumulate_dx;                // dx = round(dx + .)
  float* dw;                         // [V, D] f32, added to, or nullptr
  int32_t ignore_index = INT32_MIN;
};

uint64_t distill_head_workspace_bytes(const DistillHeadShape& s);
void distill_head(const DistillHeadShape& s, const DistillHeadArgs& a, void* ws, uint64_t ws_bytes, cudaStream_t st);

}  // namespace nm
