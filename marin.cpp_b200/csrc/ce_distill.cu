// Distillation head (include/marincpp/kernels/distill_head.hpp): the row kernels around the three contractions of
// ce_gemm.cu, the order in which one call issues them, and the C entry points.
//
// Precision. Loss, statistics and dW are f32 results, so nothing on their way has fewer bits than they need: the logits are
// stored in f32, and the normalised gradient n is held as two bf16 terms hi + lo (hi = bf16(n), lo = bf16(n - hi), 2^-17
// relative), both of which the dW contraction takes; dX is a bf16 result and takes hi alone. The two terms of 64 columns lie
// where the 64 f32 logits lay, so the rewrite is in place and the store is 4 bytes per logit throughout.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cmath>
#include <string>

#include "abi_guard.hpp"
#include "ce_internal.hpp"
#include "ew_rows.cuh"
#include "marincpp/capi_ce.h"
#include "marincpp/kernels/distill_head.hpp"
#include "ptx.cuh"

namespace nm {
namespace ce {
namespace {

using nm::ew::warp_sum;
using nm::ptx::ex2_approx;
using nm::ptx::exponent_of;
using nm::ptx::exponent_step;

constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;
constexpr int kMaxEntries = 512, kMaxExtent = 1 << 30;

// What the rewrite of a row's logits needs: n = a_t 2^(z log2e / tau - r_t) + a_1 2^(z log2e - r_1) - (listed entries), with r
// the reference exponent round(max z c) that the row's sums count from, and the sums' reciprocals in a. (With the log-sum-exp as
// the reference its own rounding, half a step of a number of the size of z / tau, would scale every probability.)
struct alignas(16) DistillRow {
  float r_t, a_t, r_1, a_1;
};
__device__ __forceinline__ float dense_part(float z, const DistillRow& f, float tau_log2e) {
  float n = __fmul_rn(f.a_t, ex2_approx(fmaf(z, tau_log2e, -f.r_t)));
  if (f.a_1 != 0.f) n = fmaf(f.a_1, ex2_approx(fmaf(z, kLog2e, -f.r_1)), n);
  return n;
}

struct DistillRowsArgs {
  const float* tmax; const float* tsum; const float* tsum1; int64_t ldT; int NT;
  const int32_t* ids; const void* logits; bool logits_bf16; const float* teacher_lse; int K;
  const int32_t* targets; const float* weight; const float* zt;
  const float* store; int64_t ldS;      // logits of the chunk, or nullptr:
  const float* zk;                      // [rows, K] student logits of the listed ids
  int rows, V;
  float tau, soft, hard;
  int32_t ignore_index;
  float* loss; float* kl; float* lse;   // kl may be nullptr
  DistillRow* rowf; int32_t* pcol; float* pval;   // nullptr in a forward-only call; patches [rows, K + 1]
};

// Eight rows per CTA. First the tile partials are merged: the vocabulary's tiles are cut into 32 strips, lane = (row, one of
// four strips) of a warp, eight tiles at a time so that their loads are in flight together, in ascending order; then warp w
// joins the strips of row w (a butterfly: the same order always) and stays with that row, its lanes the listed entries. Bound
// by latency: a CTA waits for some ten dependent round trips. (With 32 rows per CTA 25 us instead of 12 us for 2125 rows.)
constexpr int kRowsPerCta = 8, kStrips = 32;
__global__ void __launch_bounds__(32 * kRowsPerCta) k_distill_rows(const DistillRowsArgs p) {
  __shared__ float sm[kStrips][kRowsPerCta], ss[kStrips][kRowsPerCta], s1[kStrips][kRowsPerCta];
  extern __shared__ int32_t entries[];   // per warp: ids [K], masses [K]
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const float inv_tau = __fdiv_rn(1.f, p.tau), tau_log2e = __fdiv_rn(kLog2e, p.tau);   // as the logits kernel's
  nm::ptx::release_next();
  nm::ptx::after_previous();
  {
    const int local = lane & 7, strip = w * 4 + (lane >> 3), r = blockIdx.x * kRowsPerCta + local;
    const int i0 = int(int64_t(p.NT) * strip / kStrips), i1 = int(int64_t(p.NT) * (strip + 1) / kStrips);
    float m = -INFINITY, s = 0.f, o = 0.f;
    if (r < p.rows) {
      for (int i = i0; i < i1; i += 8) {
        float tm[8], ts[8], to[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          const int64_t at = int64_t(min(i + q, i1 - 1)) * p.ldT + r;
          tm[q] = p.tmax[at], ts[q] = p.tsum[at], to[q] = p.tsum1 ? p.tsum1[at] : 0.f;
        }
        float nm = m;
#pragma unroll
        for (int q = 0; q < 8; ++q) nm = fmaxf(nm, tm[q]);
        const float base = isfinite(nm) ? nm : 0.f, from = isfinite(m) ? m : base;   // no sums yet where m is not finite
        s *= exp2f(exponent_step(from, base, tau_log2e)), o *= exp2f(exponent_step(from, base, kLog2e));
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          if (i + q >= i1) break;
          s = fmaf(ts[q], exp2f(exponent_step(tm[q], base, tau_log2e)), s);
          if (p.tsum1) o = fmaf(to[q], exp2f(exponent_step(tm[q], base, kLog2e)), o);
        }
        m = nm;
      }
    }
    sm[strip][local] = m, ss[strip][local] = s, s1[strip][local] = o;
    __syncthreads();
  }
  const int r = blockIdx.x * kRowsPerCta + w;
  if (r >= p.rows) return;
  float M, S, S1;    // the maximum and the sums of 2^(z c - exponent_of(M, c)) at the temperature and at 1
  {
    float m = sm[lane][w];
    M = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    if (!isfinite(M)) M = 0.f;
    if (!isfinite(m)) m = M;                     // an empty strip has sums of 0
    S = warp_sum(ss[lane][w] * exp2f(exponent_step(m, M, tau_log2e)));
    S1 = S;                                      // at temperature 1 one sum serves both
    if (p.tsum1) S1 = warp_sum(s1[lane][w] * exp2f(exponent_step(m, M, kLog2e)));
  }
  const float r_t = exponent_of(M, tau_log2e), log2_s = log2f(S);
  // a log of a sum in nats, counted from M c as it is instead of from its rounding
  auto log_above_max = [&](float sum, float c) { return fmaf(-kLn2, fmaf(M, c, -exponent_of(M, c)), logf(sum)); };
  if (lane == 0) p.lse[r] = __fdiv_rn(M, p.tau) + log_above_max(S, tau_log2e);
  int32_t* const id_s = entries + w * 2 * p.K;
  float* const q_s = reinterpret_cast<float*>(id_s + p.K);
  const float wt = p.weight[r];
  const bool live = wt != 0.f;
  const int tg = p.targets ? p.targets[r] : -1;
  const bool labelled = live && p.hard != 0.f && tg >= 0 && tg < p.V && tg != p.ignore_index;
  const int64_t row_k = int64_t(r) * p.K;
  // the listed entries of this row: id (or -1) and teacher's logit
  auto teacher = [&](int k) {
    return p.logits_bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p.logits)[row_k + k])
                         : static_cast<const float*>(p.logits)[row_k + k];
  };
  __syncwarp();
  float top = -INFINITY;
  for (int k = lane; k < p.K; k += 32) {
    const int32_t id = p.ids[row_k + k];
    const bool in = live && id >= 0 && id < p.V;
    id_s[k] = in ? id : -1;
    if (in && !p.teacher_lse) top = fmaxf(top, teacher(k));
  }
  float norm = 0.f;   // of the logits counted from `top`, or the given one
  bool any = false;
  if (p.teacher_lse) {
    norm = p.teacher_lse[r];
  } else {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    any = top != -INFINITY;
    float s = 0.f;
    for (int k = lane; k < p.K; k += 32)
      if (id_s[k] >= 0 && any) s += expf(__fdiv_rn(teacher(k) - top, p.tau));
    s = warp_sum(s);
    norm = any ? logf(s) : INFINITY;            // nothing listed: every mass is 0
  }
  auto log_mass = [&](int k) {
    const float t = teacher(k);
    if (!p.teacher_lse) return (any ? __fdiv_rn(t - top, p.tau) : t) - norm;
    const float d = __fdiv_rn(t, p.tau);        // and what the quotient lacks, which the difference would show
    return (d - norm) + (isfinite(d) ? fmaf(-d, p.tau, t) * inv_tau : 0.f);
  };
  float kl = 0.f, mass = 0.f;
  for (int k = lane; k < p.K; k += 32) {
    const int32_t id = id_s[k];
    float q = 0.f;
    if (id >= 0) {
      const float lq = log_mass(k);
      q = expf(lq);
      const float z = p.store ? p.store[int64_t(r) * p.ldS + id] : p.zk[row_k + k];
      if (q != 0.f) kl = fmaf(q, fmaf(-kLn2, fmaf(z, tau_log2e, -r_t) - log2_s, lq), kl);
    }
    q_s[k] = q;
    mass += q;
  }
  kl = warp_sum(kl);
  mass = warp_sum(mass);
  if (!p.teacher_lse) mass = any ? 1.f : mass;   // by definition (a NaN among the logits shows in kl)
  if (lane == 0) {
    float loss = 0.f;
    if (live) {
      loss = p.soft * p.tau * p.tau * kl;
      if (labelled) loss = fmaf(p.hard, (M - p.zt[r]) + log_above_max(S1, kLog2e), loss);
    }
    p.loss[r] = loss;
    if (p.kl) p.kl[r] = live ? kl : 0.f;
  }
  if (p.rowf == nullptr) return;
  DistillRow f{0.f, 0.f, 0.f, 0.f};
  const float unit = live ? wt * p.soft * p.tau : 0.f;   // gradient of one unit of teacher mass
  const float hit = labelled ? wt * p.hard : 0.f;
  if (live) f = DistillRow{r_t, __fdiv_rn(unit * mass, S), exponent_of(M, kLog2e), __fdiv_rn(hit, S1)};
  if (lane == 0) p.rowf[r] = f;
  __syncwarp();
  // the elements of n that are not dense alone, whole: every listed id, and the target where it is not listed
  const int64_t row_p = int64_t(r) * (p.K + 1);
  bool listed = false;
  for (int k = lane; k < p.K; k += 32) {
    const int32_t id = id_s[k];
    float v = 0.f;
    if (id >= 0) {
      float q = 0.f;
      for (int o = 0; o < p.K; ++o) q += id_s[o] == id ? q_s[o] : 0.f;   // the same id twice: both write this sum
      v = fmaf(-unit, q, dense_part(p.store[int64_t(r) * p.ldS + id], f, tau_log2e));
      if (labelled && id == tg) v -= hit, listed = true;
    }
    p.pcol[row_p + k] = id;
    p.pval[row_p + k] = v;
  }
  listed = __any_sync(0xffffffffu, listed);
  if (lane == 0) {
    const bool own = labelled && !listed;
    p.pcol[row_p + p.K] = own ? tg : -1;
    p.pval[row_p + p.K] = own ? dense_part(p.zt[r], f, tau_log2e) - hit : 0.f;
  }
}

// Student logits of the listed ids for a call that stores none: one f32 dot product of x_t and W[id] each. A warp takes four
// entries of a row at a time, a lane every 32nd 16-byte piece of the two rows. The only form there is for such a call, whatever
// K: storing the logits would need the large workspace that the caller did not give, and 4 T V bytes of traffic each way against
// 2 T K D here. The whole call in us for K = 1 / 16 / 64 / 128 / 256 / 512: 2125 x 512 x 128256 222 / 225 / 246 / 271 / 318 / 410;
// 8192 x 2048 x 128256 3061 / 3073 / 3412 / 3855 / 4697 / 6335; 1000 x 1024 x 32000 85 / 85 / 100 / 118 / 163 / 242.
constexpr int kDotEntries = 4;
__global__ void __launch_bounds__(256) k_distill_dots(const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ w,
                                                      const int32_t* __restrict__ ids, const float* __restrict__ weight,
                                                      int rows, int D, int V, int K, float* __restrict__ zk) {
  using namespace nm::ew;
  nm::ptx::release_next();
  nm::ptx::after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int groups = (K + kDotEntries - 1) / kDotEntries;
  for (int64_t job = int64_t(blockIdx.x) * 8 + warp; job < int64_t(rows) * groups; job += int64_t(gridDim.x) * 8) {
    const int r = int(job / groups), k0 = int(job % groups) * kDotEntries;
    if (weight[r] == 0.f) continue;               // the row's entries are not looked at
    int32_t id[kDotEntries];
    float s[kDotEntries];
#pragma unroll
    for (int e = 0; e < kDotEntries; ++e) {
      id[e] = k0 + e < K ? __ldg(ids + int64_t(r) * K + k0 + e) : -1;
      if (id[e] >= V) id[e] = -1;
      s[e] = 0.f;
    }
    for (int c = lane * 8; c < D; c += 256) {
      float a[8], b[8];
      unpack8(ldg16(x + int64_t(r) * D + c), a);
#pragma unroll
      for (int e = 0; e < kDotEntries; ++e) {
        if (id[e] < 0) continue;                  // uniform over the warp
        unpack8(ldg16(w + int64_t(id[e]) * D + c), b);
#pragma unroll
        for (int q = 0; q < 8; ++q) s[e] = fmaf(a[q], b[q], s[e]);
      }
    }
#pragma unroll
    for (int e = 0; e < kDotEntries; ++e) s[e] = warp_sum(s[e]);
    if (lane == 0) {
#pragma unroll
      for (int e = 0; e < kDotEntries; ++e)
        if (k0 + e < K) zk[int64_t(r) * K + k0 + e] = s[e];
    }
  }
}

// f32 logits -> the two-term gradient in place, then the listed elements on top. A CTA takes kSegment columns of a row; eight
// lanes of a warp hold the 64 logits of a block before any of them is overwritten. Bound by HBM: 4 bytes in, 4 out,
// 8192 x 128256 in 1.21 ms (6.9 TB/s).
constexpr int kSegment = 4096, kGradThreads = 256;
struct TwoTerm {
  uint16_t hi, lo;
};
__device__ __forceinline__ TwoTerm split_two(float n) {
  const __nv_bfloat16 hi = __float2bfloat16_rn(n);
  const __nv_bfloat16 lo = __float2bfloat16_rn(__fsub_rn(n, __bfloat162float(hi)));
  return TwoTerm{__bfloat16_as_ushort(hi), __bfloat16_as_ushort(lo)};
}
__global__ void __launch_bounds__(kGradThreads) k_distill_grad(float* store, int64_t ldS, const DistillRow* __restrict__ rowf,
                                                               const int32_t* __restrict__ pcol,
                                                               const float* __restrict__ pval, int V, int patches,
                                                               float tau_log2e) {
  nm::ptx::release_next();
  nm::ptx::after_previous();
  const int r = blockIdx.y, c0 = blockIdx.x * kSegment, c1 = int(min(int64_t(c0) + kSegment, ldS));
  const DistillRow f = rowf[r];
  const bool dead = f.a_t == 0.f && f.a_1 == 0.f;
  uint8_t* const row = reinterpret_cast<uint8_t*>(store + int64_t(r) * ldS);
  constexpr int kStep = kGradThreads * 8, kBatch = kSegment / kStep;
  float z[kBatch][8];
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int c = c0 + i * kStep + int(threadIdx.x) * 8;
    if (c < c1) {
      const float4* s = reinterpret_cast<const float4*>(row + int64_t(c) * 4);
      const float4 a = s[0], b = s[1];
      z[i][0] = a.x, z[i][1] = a.y, z[i][2] = a.z, z[i][3] = a.w, z[i][4] = b.x, z[i][5] = b.y, z[i][6] = b.z, z[i][7] = b.w;
    }
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kBatch; ++i) {
    const int c = c0 + i * kStep + int(threadIdx.x) * 8;
    if (c < c1) {
      uint32_t hi[4], lo[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float n[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) n[e] = (dead || c + 2 * q + e >= V) ? 0.f : dense_part(z[i][2 * q + e], f, tau_log2e);
        const __nv_bfloat162 h = __floats2bfloat162_rn(n[0], n[1]);
        hi[q] = *reinterpret_cast<const uint32_t*>(&h);
        const __nv_bfloat162 l = __floats2bfloat162_rn(__fsub_rn(n[0], __uint_as_float(hi[q] << 16)),
                                                       __fsub_rn(n[1], __uint_as_float(hi[q] & 0xffff0000u)));
        lo[q] = *reinterpret_cast<const uint32_t*>(&l);
      }
      uint8_t* block = row + int64_t(c / 64) * 256 + (c % 64) * 2;
      *reinterpret_cast<uint4*>(block) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
      *reinterpret_cast<uint4*>(block + 128) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    }
  }
  __syncthreads();
  for (int k = threadIdx.x; k < patches; k += kGradThreads) {
    const int c = pcol[int64_t(r) * patches + k];
    if (c >= c0 && c < c1) {
      const TwoTerm t = split_two(pval[int64_t(r) * patches + k]);
      uint8_t* at = row + int64_t(c / 64) * 256 + (c % 64) * 2;
      *reinterpret_cast<uint16_t*>(at) = t.hi;
      *reinterpret_cast<uint16_t*>(at + 128) = t.lo;
    }
  }
}

// dx = round(scale * sum of the shares in order (+ dx)); bound by HBM and launch latency (2125 x 1024, two shares: 6 us)
__global__ void __launch_bounds__(256) k_distill_dx_join(const float* __restrict__ part, int shares, int64_t n8,
                                                         const float* __restrict__ scale, __nv_bfloat16* dx, bool add) {
  using namespace nm::ew;
  nm::ptx::release_next();
  nm::ptx::after_previous();
  const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
  if (i >= n8) return;
  const float g = __ldg(scale);
  float s[8] = {};
#pragma unroll 4
  for (int k = 0; k < shares; ++k) {
    const float4* src = reinterpret_cast<const float4*>(part) + (int64_t(k) * n8 + i) * 2;
    const float4 a = __ldcs(src), b = __ldcs(src + 1);
    s[0] += a.x, s[1] += a.y, s[2] += a.z, s[3] += a.w, s[4] += b.x, s[5] += b.y, s[6] += b.z, s[7] += b.w;
  }
  float old[8] = {};
  if (add) load8(dx + i * 8, old);
#pragma unroll
  for (int q = 0; q < 8; ++q) s[q] = fmaf(s[q], g, old[q]);
  store8(dx + i * 8, s);
}

// ------------------------------------------------------------------------------------------------ host
struct DistillRegions {
  uint32_t* status;
  float* tmax; float* tsum; float* tsum1; float* lse; float* zt; float* zk;
  DistillRow* rowf; int32_t* pcol; float* pval; float* store; float* dxpart;
  int64_t ldS;
  uint64_t bytes;
};
DistillRegions layout(const DistillHeadShape& s, void* base) {
  Arena arena(base);
  const uint64_t rows = uint64_t(std::min<int64_t>(s.chunk_rows, std::max<int64_t>(s.T, 1))), NT = uint64_t(stats_tiles(s.V));
  DistillRegions r{};
  r.status = arena.take<uint32_t>(64);
  r.tmax = arena.take<float>(NT * rows);
  r.tsum = arena.take<float>(NT * rows);
  r.tsum1 = arena.take<float>(NT * rows);
  r.lse = arena.take<float>(rows);
  r.zt = arena.take<float>(rows);
  if (s.forward_only) {
    r.zk = arena.take<float>(rows * uint64_t(s.K));
  } else {
    r.rowf = arena.take<DistillRow>(rows);
    r.pcol = arena.take<int32_t>(rows * uint64_t(s.K + 1));
    r.pval = arena.take<float>(rows * uint64_t(s.K + 1));
    r.ldS = round_up(s.V, 64);
    r.store = arena.take<float>(rows * uint64_t(r.ldS));
    r.dxpart = arena.take<float>(std::min<uint64_t>(kMaxDxShareRows, kMaxDxShares * rows) * uint64_t(s.D));
  }
  r.bytes = arena.bytes();
  return r;
}

void require_shape(const DistillHeadShape& s) {
  NM_REQUIRE(s.T >= 0, "distillation: the row count T cannot be negative");
  NM_REQUIRE(s.D > 0 && s.D % 8 == 0, "distillation: D must be a positive multiple of 8 (rows are moved in 16-byte pieces)");
  // the two-term gradient is 2 V columns wide and its TMA coordinates are 32-bit
  NM_REQUIRE(s.V > 0 && s.V <= kMaxExtent, "distillation: the vocabulary size V must be positive and at most 2^30");
  NM_REQUIRE(s.K >= 1 && s.K <= kMaxEntries, "distillation: 1 to 512 teacher entries per row");
  NM_REQUIRE(s.chunk_rows > 0, "distillation: chunk_rows must be positive");
  NM_REQUIRE(std::min<int64_t>(s.T, s.chunk_rows) <= kMaxExtent, "distillation: at most 2^30 rows per chunk");
}
bool aligned(const void* p, uintptr_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }

}  // namespace
}  // namespace ce

uint64_t distill_head_workspace_bytes(const DistillHeadShape& s) {
  ce::require_shape(s);
  return ce::layout(s, nullptr).bytes;
}

void distill_head(const DistillHeadShape& s, const DistillHeadArgs& a, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  using namespace ce;
  require_shape(s);
  if (s.T == 0) return;
  NM_REQUIRE(a.x && a.w && a.teacher_ids && a.teacher_logits && a.weight && a.loss_tok,
             "distillation: x, w, teacher_ids, teacher_logits, weight and loss_tok are required");
  NM_REQUIRE(std::isfinite(a.temperature) && a.temperature > 0.f, "distillation: the temperature must be positive");
  NM_REQUIRE(std::isfinite(a.soft_weight) && a.soft_weight >= 0.f && std::isfinite(a.hard_weight) && a.hard_weight >= 0.f,
             "distillation: soft_weight and hard_weight cannot be negative");
  NM_REQUIRE(a.targets || a.hard_weight == 0.f, "distillation: a hard term needs targets");
  NM_REQUIRE(!s.forward_only || (!a.dx && !a.dw), "distillation: a forward-only call has no dx and no dw");
  const bool grads = !s.forward_only && (a.dx || a.dw);
  NM_REQUIRE(!grads || a.grad_scale, "distillation: a gradient call needs the device scalar grad_scale");
  NM_REQUIRE(!(a.accumulate_dx && a.dx == a.x), "distillation: dx may be x or accumulate, not both");
  NM_REQUIRE(aligned(a.x, 16) && aligned(a.w, 16) && aligned(a.dx, 16) && aligned(a.dw, 16),
             "distillation: x, w, dx and dw must be 16-byte aligned");
  NM_REQUIRE(aligned(a.teacher_ids, 4) && aligned(a.teacher_logits, dtype_size(a.teacher_dtype)),
             "distillation: teacher entries must be aligned to their size");
  for (const void* p : {static_cast<const void*>(a.teacher_lse), static_cast<const void*>(a.targets),
                        static_cast<const void*>(a.weight), static_cast<const void*>(a.grad_scale),
                        static_cast<const void*>(a.loss_tok), static_cast<const void*>(a.kl_tok),
                        static_cast<const void*>(a.lse), static_cast<const void*>(a.loss_partial)})
    NM_REQUIRE(aligned(p, 4), "distillation: targets, weights, statistics and losses must be 4-byte aligned");
  NM_REQUIRE(ws != nullptr && aligned(ws, kArenaAlign), "distillation: a 256-byte aligned workspace is required");
  NM_REQUIRE(ws_bytes >= layout(s, nullptr).bytes, "distillation: the workspace is smaller than "
                                                   "nm_ce_distill_workspace_bytes()");
  NM_REQUIRE(device_arch() >= 100, "distillation: every kernel of this library is sm_100a code");
  const DistillRegions w = layout(s, ws);
  const int D = s.D, V = s.V, K = s.K;
  const bool hard = a.hard_weight != 0.f, second_sum = hard && a.temperature != 1.f;
  const float tau_log2e = 1.4426950408889634f / a.temperature;
  const size_t teacher_size = dtype_size(a.teacher_dtype);
  NM_CUDA(cudaMemsetAsync(w.status, 0, sizeof(uint32_t), st));

  int64_t slot = 0;
  for (int64_t r0 = 0; r0 < s.T; r0 += s.chunk_rows, ++slot) {
    const int n = int(std::min<int64_t>(s.chunk_rows, s.T - r0));
    const uint16_t* x = static_cast<const uint16_t*>(a.x) + r0 * D;
    const int32_t* ids = a.teacher_ids + r0 * K;
    DistillLogitsArgs la{x, a.w, hard ? a.targets + r0 : nullptr, n, D, V, a.temperature, grads ? w.store : nullptr, w.ldS,
                         w.tmax, w.tsum, second_sum ? w.tsum1 : nullptr, n, w.zt, w.status};
    {
      ProfScope t(0, st);
      launch_distill_logits(la, st);
    }
    // a call that asks for no gradient stores no logits, whichever workspace it was given
    float* zk = s.forward_only ? w.zk : w.pval;
    if (!grads) {
      const int64_t jobs = int64_t(n) * ((K + kDotEntries - 1) / kDotEntries);
      launch_after(k_distill_dots, dim3(unsigned(std::min<int64_t>((jobs + 7) / 8, int64_t(sm_count()) * 64))), 256, 0, st,
                   reinterpret_cast<const __nv_bfloat16*>(x), static_cast<const __nv_bfloat16*>(a.w), ids, a.weight + r0, n, D, V,
                   K, zk);
    }
    DistillRowsArgs ra{};
    ra.tmax = w.tmax, ra.tsum = w.tsum, ra.tsum1 = second_sum ? w.tsum1 : nullptr, ra.ldT = n, ra.NT = stats_tiles(V);
    ra.ids = ids, ra.logits = static_cast<const uint8_t*>(a.teacher_logits) + r0 * K * int64_t(teacher_size);
    ra.logits_bf16 = a.teacher_dtype == DType::bf16, ra.teacher_lse = a.teacher_lse ? a.teacher_lse + r0 : nullptr, ra.K = K;
    ra.targets = hard ? a.targets + r0 : nullptr, ra.weight = a.weight + r0, ra.zt = w.zt;
    ra.store = grads ? w.store : nullptr, ra.ldS = w.ldS, ra.zk = zk, ra.rows = n, ra.V = V;
    ra.tau = a.temperature, ra.soft = a.soft_weight, ra.hard = a.hard_weight, ra.ignore_index = a.ignore_index;
    ra.loss = a.loss_tok + r0, ra.kl = a.kl_tok ? a.kl_tok + r0 : nullptr, ra.lse = a.lse ? a.lse + r0 : w.lse;
    ra.rowf = grads ? w.rowf : nullptr, ra.pcol = w.pcol, ra.pval = w.pval;
    {
      ProfScope t(1, st);
      const int entry_bytes = kRowsPerCta * 2 * K * 4;
      launch_after(k_distill_rows, dim3(unsigned((n + kRowsPerCta - 1) / kRowsPerCta)), 32 * kRowsPerCta, unsigned(entry_bytes), st, ra);
    }
    if (a.loss_partial) {
      ProfScope t(5, st);
      launch_chunk_loss(a.loss_tok + r0, a.weight + r0, n, a.loss_partial + slot, st);
    }
    if (!grads) continue;
    {
      ProfScope t(2, st);
      for (int y0 = 0; y0 < n; y0 += 65535) {   // rows of one launch: the grid's second extent
        const int ny = std::min(n - y0, 65535);
        launch_after(k_distill_grad, dim3(unsigned((w.ldS + kSegment - 1) / kSegment), unsigned(ny)), kGradThreads, 0, st,
                     w.store + int64_t(y0) * w.ldS, w.ldS, w.rowf + y0, w.pcol + int64_t(y0) * (K + 1),
                     w.pval + int64_t(y0) * (K + 1), V, K + 1, tau_log2e);
      }
    }
    if (a.dw) {   // before dX, which may be written over x
      ProfScope t(3, st);
      launch_distill_wgrad(DistillWgradArgs{w.store, 2 * w.ldS, x, n, D, V, a.grad_scale, a.dw, w.status}, st);
    }
    if (a.dx) {
      uint16_t* dx = static_cast<uint16_t*>(a.dx) + r0 * D;
      const int shares = distill_dgrad_shares(n, D, V);
      ProfScope t(4, st);
      launch_distill_dgrad(DistillDgradArgs{w.store, 2 * w.ldS, a.w, n, D, V, a.grad_scale, a.accumulate_dx ? dx : nullptr, dx, 2,
                                            w.dxpart, shares, w.status}, st);
      if (shares > 1) {
        const int64_t n8 = int64_t(n) * D / 8;
        launch_after(k_distill_dx_join, dim3(unsigned((n8 + 255) / 256)), 256, 0, st, w.dxpart, shares, n8, a.grad_scale,
                     reinterpret_cast<__nv_bfloat16*>(dx), a.accumulate_dx);
      }
    }
  }
}

}  // namespace nm

extern "C" {

uint64_t nm_ce_distill_workspace_bytes(int64_t T, int D, int V, int K, int chunk_rows, int forward_only) {
  return nm::abi::guarded_value<uint64_t>(0, [&] {
    return nm::distill_head_workspace_bytes(nm::DistillHeadShape{T, D, V, K, chunk_rows, forward_only != 0});
  });
}

int nm_ce_distill(int teacher_dtype, const void* x, const void* w, const int32_t* teacher_ids, const void* teacher_logits,
                  const float* teacher_lse, const int32_t* targets, const float* weight, const float* grad_scale,
                  float temperature, float soft_weight, float hard_weight, float* loss_tok, float* kl_tok, float* lse,
                  float* loss_partial, void* dx, int accumulate_dx, float* dw, int forward_only, int64_t T, int D, int V, int K,
                  int chunk_rows, int32_t ignore_index, void* workspace, uint64_t workspace_bytes, void* stream) {
  return nm::abi::guarded([&] {
    NM_REQUIRE(teacher_dtype == 0 || teacher_dtype == 1, "nm_ce_distill: teacher_dtype 0 (f32) or 1 (bf16)");
    nm::DistillHeadArgs a{};
    a.x = x;
    a.w = w;
    a.teacher_ids = teacher_ids;
    a.teacher_logits = teacher_logits;
    a.teacher_dtype = teacher_dtype == 0 ? nm::DType::f32 : nm::DType::bf16;
    a.teacher_lse = teacher_lse;
    a.targets = targets;
    a.weight = weight;
    a.grad_scale = grad_scale;
    a.temperature = temperature;
    a.soft_weight = soft_weight;
    a.hard_weight = hard_weight;
    a.loss_tok = loss_tok;
    a.kl_tok = kl_tok;
    a.lse = lse;
    a.loss_partial = loss_partial;
    a.dx = dx;
    a.accumulate_dx = accumulate_dx != 0;
    a.dw = dw;
    a.ignore_index = ignore_index;
    nm::distill_head(nm::DistillHeadShape{T, D, V, K, chunk_rows, forward_only != 0}, a, workspace, workspace_bytes,
                     static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
