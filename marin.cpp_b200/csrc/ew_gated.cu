// The gated sandwich tail: the norms before and after a block, fused with the block's gate and the scaled residual.
//   forward   y = g_post ? g_post (branch r_p) : branch,  r_p = rsqrt(mean(branch^2) + eps)
//             x_out = round(s x_in + sigmoid(gate) y);  a_next = round(g_next (x_out r_n)),  r_n = rsqrt(mean(x_out^2) + eps)
//   backward  a = g_next da;  m = dx_out + r_n a - x_out (r_n^3 sum(x_out a) / D)      (gradient of x_out, not rounded)
//             dx_in = round(s m);  ds += x_in m;  dg_next += da x_out r_n
//             dgate = m y sigmoid'(gate) (summed over the row for a gate per token);  t = sigmoid(gate) m
//             dg_post += t branch r_p;  p = g_post t;  dbranch = round(r_p p - branch (r_p^3 sum(branch p) / D))
// gate (per token or per element), s and g_post are optional. f32 inside, one rounding per stored output (the accurate
// policy of the sandwich tail); x_out is what the residual stream holds, so the next norm reads its rounded values. The
// backward forms x_out again from x_in, branch and gate instead of reading it: bit for bit the stored one, because both
// directions share outer() below, and 2 bytes per element less.
// sigmoid(g) and its derivative come from e = exp(-|g|), r = 1 / (1 + e): r or e r, and e r^2: no cancellation.
// Row groups and batch ring as in ew_rows.cuh. What bounds them is HBM (10 and 16 bytes per element in bf16 with a gate per
// element).
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <string>

#include "abi_guard.hpp"
#include "ce_internal.hpp"
#include "ew_api.hpp"
#include "ew_rows.cuh"
#include "marincpp/capi_ew.h"

namespace nm::ew {
namespace {

enum GateKind : int { kNoGate = 0, kTokenGate = 1, kElementGate = 2 };

// Eight consecutive elements: as stored, and as four f32 pairs.
template <bool BF16>
struct Raw {
  static constexpr int kBytes = BF16 ? 16 : 32;
  uint4 q[BF16 ? 1 : 2];
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (auto& v : q) v = make_uint4(0u, 0u, 0u, 0u);
  }
  __device__ __forceinline__ void from_shared(uint32_t at) {
    q[0] = nm::ptx::ld_shared_v4(at);
    if constexpr (!BF16) q[1] = nm::ptx::ld_shared_v4(at + 16u);
  }
  __device__ __forceinline__ void from_global(const void* p, int64_t element) {
    const uint4* s = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(p) + element * (BF16 ? 2 : 4));
    q[0] = __ldg(s);
    if constexpr (!BF16) q[1] = __ldg(s + 1);
  }
  __device__ __forceinline__ void to_global(void* p, int64_t element) const {
    uint4* d = reinterpret_cast<uint4*>(static_cast<uint8_t*>(p) + element * (BF16 ? 2 : 4));
    d[0] = q[0];
    if constexpr (!BF16) d[1] = q[1];
  }
  __device__ __forceinline__ F2 pair(int i) const {
    if constexpr (BF16) {
      return f2_of(word_of(q[0], i));
    } else {
      const uint4& h = q[i >> 1];
      return (i & 1) ? f2(__uint_as_float(h.z), __uint_as_float(h.w)) : f2(__uint_as_float(h.x), __uint_as_float(h.y));
    }
  }
  __device__ __forceinline__ void round(const F2 (&v)[4]) {   // to the storage type
    if constexpr (BF16) {
      q[0] = make_uint4(bf16x2_of(v[0]), bf16x2_of(v[1]), bf16x2_of(v[2]), bf16x2_of(v[3]));
    } else {
      float f[8];
#pragma unroll
      for (int i = 0; i < 4; ++i) f2_get(v[i], f[2 * i], f[2 * i + 1]);
      q[0] = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
      q[1] = make_uint4(__float_as_uint(f[4]), __float_as_uint(f[5]), __float_as_uint(f[6]), __float_as_uint(f[7]));
    }
  }
};
__device__ __forceinline__ float scalar_of(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

struct Gate {
  float on, slope;   // sigmoid(g) and its derivative
};
__device__ __forceinline__ Gate gate_of(float g) {
  const float e = nm::ptx::ex2_approx(-fabsf(g) * 1.4426950408889634f);
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.f + e));
  const float er = e * r;
  return Gate{g >= 0.f ? r : er, er * r};   // a NaN stays one through e
}
struct Gate2 {
  F2 on, slope;
};
__device__ __forceinline__ Gate2 gate_of(F2 g) {
  float a, b;
  f2_get(g, a, b);
  const Gate x = gate_of(a), y = gate_of(b);
  return Gate2{f2(x.on, y.on), f2(x.slope, y.slope)};
}

// The value of x_out before it is rounded, two elements. `n` is the normalised branch (post) or the branch itself. Every
// product that feeds a sum is an explicit fma or an operand of one, so forward and backward get the same bits.
template <int GATE>
__device__ __forceinline__ F2 outer(F2 n, F2 gp, bool post, F2 on, F2 x, F2 s, bool scaled) {
  if constexpr (GATE == kNoGate) {
    if (scaled) return f2_fma(s, x, post ? f2_mul(n, gp) : n);
    return post ? f2_fma(n, gp, x) : f2_add(n, x);
  } else {
    const F2 y = post ? f2_mul(n, gp) : n;
    return scaled ? f2_fma(s, x, f2_mul(on, y)) : f2_fma(on, y, x);
  }
}
__device__ __forceinline__ float both(F2 v) {
  float lo, hi;
  f2_get(v, lo, hi);
  return lo + hi;
}

struct TailParams {
  const void* branch; const void* x_in; const void* gate; const void* res_scale; const void* g_post; const void* g_next;
  void* x_out; void* a_next;
  float* rstd_post; float* rstd_next;            // written forward, read backward
  // backward
  const void* dx_out; const void* da_next;
  void* dx_in; void* dbranch; void* dgate;
  float* pg_next; float* pg_post; float* pg_scale;   // [parts, D] partial sums, or nullptr
  int64_t T, parts;
  int D, G, stages, nops;
  uint32_t op_bytes;
  float eps;
  uint32_t* status;
};

// Ring set-up shared by both directions; `fetch` (thread 0) brings one batch of every operand into a slot.
template <bool BF16>
struct TailRing {
  RowRing ring;
  const uint8_t* op[5];
  int D;
  __device__ __forceinline__ void begin(uint8_t* raw, const TailParams& p, int* abort_word) {
    using namespace nm::ptx;
    D = p.D;
    ring.data = (smem_u32(raw) + 127u) & ~127u;
    ring.op_bytes = p.op_bytes, ring.stages = p.stages, ring.nops = p.nops;
    ring.full = ring.data + uint32_t(p.stages * p.nops) * p.op_bytes;
    ring.empty = ring.full + 8u * p.stages;
    if (threadIdx.x == 0) {
      for (int s = 0; s < p.stages; ++s) mbar_init(ring.full + 8u * s, 1), mbar_init(ring.empty + 8u * s, kRingWarps);
      *abort_word = 0;
      fence_barrier_init();
    }
    __syncthreads();
  }
  __device__ __forceinline__ void fetch(int s, const BatchWalk& b, int groups) const {
    using namespace nm::ptx;
    const uint32_t bytes = b.rows(groups) * uint32_t(D) * (BF16 ? 2u : 4u);
    const uint32_t bar = ring.full + 8u * s;
    mbar_arrive_expect_tx(bar, bytes * uint32_t(ring.nops));
#pragma unroll
    for (int o = 0; o < 5; ++o)
      if (o < ring.nops) bulk_load(ring.slot(s, o), op[o] + b.row * D * (BF16 ? 2 : 4), bytes, bar);
  }
};

template <bool BF16, int PP, int GATE>
__global__ void __launch_bounds__(kGroupThreads, PP <= 2 ? 2 : 1) k_gated_fwd(const TailParams p) {
  using namespace nm::ptx;
  extern __shared__ __align__(128) uint8_t ring_raw[];
  __shared__ __align__(16) float red[2 * 8];
  __shared__ __align__(16) float red1[2 * 8];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const RowGroup rg = row_group(p.G);
  const int D = p.D, pieces = D / 8;
  const bool post = p.g_post != nullptr, scaled = p.res_scale != nullptr;
  TailRing<BF16> tr;
  tr.op[0] = static_cast<const uint8_t*>(p.branch);
  tr.op[1] = static_cast<const uint8_t*>(p.x_in);
  tr.op[2] = static_cast<const uint8_t*>(p.gate);
  tr.op[3] = tr.op[4] = nullptr;
  tr.begin(ring_raw, p, &abort_word);
  BatchWalk w, ahead;
  w.begin(p.T, p.parts);
  ahead = w;
  if (threadIdx.x == 0)
    for (int s = 0; s < p.stages - 1 && !ahead.done(p.parts); ++s, ahead.next(rg.groups, p.T, p.parts)) tr.fetch(s, ahead, rg.groups);
  Raw<BF16> gn[PP], gp[PP], sc[PP];
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int pc = rg.tg + i * rg.G;
    gn[i].zero(), gp[i].zero(), sc[i].zero();
    if (pc < pieces) {
      if (p.a_next) gn[i].from_global(p.g_next, pc * 8);
      if (post) gp[i].from_global(p.g_post, pc * 8);
      if (scaled) sc[i].from_global(p.res_scale, pc * 8);
    }
  }
  const float inv_d = 1.f / float(D);
  int flip = 0, flip1 = 0, s = 0;
  uint32_t phase = 0;
  for (; !w.done(p.parts); w.next(rg.groups, p.T, p.parts)) {
    const int64_t row = w.row + rg.group;
    const bool on_row = row < w.end;
    const int64_t off = row * D;
    float tg = 0.f;
    if constexpr (GATE == kTokenGate) tg = on_row ? gate_of(scalar_of(p.gate, row, BF16)).on : 0.f;
    const F2 token_on = f2(tg, tg);
    mbar_wait<true>(tr.ring.full + 8u * s, phase, abort_flag, p.status, kErrTransformWait);
    const uint32_t at0 = tr.ring.slot(s, 0) + uint32_t(rg.group * D + rg.tg * 8) * (BF16 ? 2u : 4u);
    auto piece = [&](int op, int i) {
      Raw<BF16> r;
      r.zero();
      if (on_row && rg.tg + i * rg.G < pieces)
        r.from_shared(at0 + uint32_t(op) * p.op_bytes + uint32_t(i * rg.G) * uint32_t(Raw<BF16>::kBytes));
      return r;
    };
    F2 rp = f2(1.f, 1.f);
    if (post) {   // uniform over the CTA
      F2 sbb = f2(0.f, 0.f);
#pragma unroll
      for (int i = 0; i < PP; ++i) {
        const Raw<BF16> b = piece(0, i);
#pragma unroll
        for (int q = 0; q < 4; ++q) sbb = f2_fma(b.pair(q), b.pair(q), sbb);
      }
      float sum[1] = {both(sbb)};
      group_sum<1>(sum, rg, red, flip);
      const float r = rsqrtf(fmaf(sum[0], inv_d, p.eps));
      if (on_row && p.rstd_post && rg.tg == 0) p.rstd_post[row] = r;
      rp = f2(r, r);
    }
    Raw<BF16> xo[PP];
    F2 sxx = f2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const Raw<BF16> b = piece(0, i), x = piece(1, i);
      Raw<BF16> g;
      if constexpr (GATE == kElementGate) g = piece(2, i);
      F2 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        F2 on = token_on;
        if constexpr (GATE == kElementGate) on = gate_of(g.pair(q)).on;
        const F2 n = post ? f2_mul(b.pair(q), rp) : b.pair(q);
        v[q] = outer<GATE>(n, gp[i].pair(q), post, on, x.pair(q), sc[i].pair(q), scaled);
      }
      xo[i].round(v);
      if (on_row && rg.tg + i * rg.G < pieces) {
        xo[i].to_global(p.x_out, off + (rg.tg + i * rg.G) * 8);
#pragma unroll
        for (int q = 0; q < 4; ++q) sxx = f2_fma(xo[i].pair(q), xo[i].pair(q), sxx);
      }
    }
    float sum[1] = {both(sxx)};
    group_sum<1>(sum, rg, red1, flip1);
    if (threadIdx.x == 0 && !ahead.done(p.parts)) {   // the slot of the batch before takes the batch stages - 1 ahead
      const int prev = s == 0 ? p.stages - 1 : s - 1;
      mbar_wait(tr.ring.empty + 8u * prev, s == 0 ? phase ^ 1u : phase, abort_flag, p.status, kErrProducerWait);
      tr.fetch(prev, ahead, rg.groups);
      ahead.next(rg.groups, p.T, p.parts);
    }
    __syncwarp();   // the slot is not read again
    if ((threadIdx.x & 31) == 0) mbar_arrive(tr.ring.empty + 8u * s);
    if (++s == p.stages) s = 0, phase ^= 1u;
    if (on_row) {
      const float r = rsqrtf(fmaf(sum[0], inv_d, p.eps));
      if (p.rstd_next && rg.tg == 0) p.rstd_next[row] = r;
      if (p.a_next) {
        const F2 rn = f2(r, r);
#pragma unroll
        for (int i = 0; i < PP; ++i) {
          const int pc = rg.tg + i * rg.G;
          if (pc < pieces) {
            F2 v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = f2_mul(gn[i].pair(q), f2_mul(xo[i].pair(q), rn));
            Raw<BF16> o;
            o.round(v);
            o.to_global(p.a_next, off + pc * 8);
          }
        }
      }
    }
  }
  if (threadIdx.x == 0 && *abort_flag) __nanosleep(200000);   // an expired wait: let copies in flight land first
}

template <bool BF16, int PP, int GATE>
__global__ void __launch_bounds__(kGroupThreads, PP <= 2 && BF16 ? 2 : 1) k_gated_bwd(const TailParams p) {
  using namespace nm::ptx;
  extern __shared__ __align__(128) uint8_t ring_raw[];
  __shared__ __align__(16) float red[2 * 8];
  __shared__ __align__(16) float red2[2 * 8 * 2];
  __shared__ __align__(16) float gsm[kGroupThreads * 4];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  const RowGroup rg = row_group(p.G);
  const int D = p.D, pieces = D / 8;
  const bool post = p.g_post != nullptr, scaled = p.res_scale != nullptr, carried = p.dx_out != nullptr;
  constexpr int kGateOp = 3, kCarriedOp = GATE == kElementGate ? 4 : 3;
  TailRing<BF16> tr;
  tr.op[0] = static_cast<const uint8_t*>(p.branch);
  tr.op[1] = static_cast<const uint8_t*>(p.x_in);
  tr.op[2] = static_cast<const uint8_t*>(p.da_next);
  tr.op[3] = tr.op[4] = static_cast<const uint8_t*>(p.dx_out);
  if constexpr (GATE == kElementGate) tr.op[kGateOp] = static_cast<const uint8_t*>(p.gate);
  tr.begin(ring_raw, p, &abort_word);
  BatchWalk w, ahead;
  w.begin(p.T, p.parts);
  ahead = w;
  if (threadIdx.x == 0)
    for (int s = 0; s < p.stages - 1 && !ahead.done(p.parts); ++s, ahead.next(rg.groups, p.T, p.parts)) tr.fetch(s, ahead, rg.groups);
  Raw<BF16> gn[PP], gp[PP], sc[PP];
  F2 dgn[PP][4], dgp[PP][4], dsc[PP][4];
#pragma unroll
  for (int i = 0; i < PP; ++i) {
    const int pc = rg.tg + i * rg.G;
    gn[i].zero(), gp[i].zero(), sc[i].zero();
    if (pc < pieces) {
      gn[i].from_global(p.g_next, pc * 8);
      if (post) gp[i].from_global(p.g_post, pc * 8);
      if (scaled) sc[i].from_global(p.res_scale, pc * 8);
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) dgn[i][q] = dgp[i][q] = dsc[i][q] = f2(0.f, 0.f);
  }
  const float inv_d = 1.f / float(D);
  int flip = 0, flip2 = 0, s = 0;
  uint32_t phase = 0;
  for (; !w.done(p.parts); w.next(rg.groups, p.T, p.parts)) {
    const int64_t row = w.row + rg.group;
    const bool on_row = row < w.end;
    const int64_t off = row * D;
    // the row's scalars are asked for before the wait, so that they land with the batch
    const float r_n = on_row ? __ldg(p.rstd_next + row) : 0.f;
    const float r_p = on_row && post ? __ldg(p.rstd_post + row) : 0.f;
    Gate tgate{0.f, 0.f};
    if constexpr (GATE == kTokenGate)
      if (on_row) tgate = gate_of(scalar_of(p.gate, row, BF16));
    const F2 token_on = f2(tgate.on, tgate.on), rn = f2(r_n, r_n), rp = f2(r_p, r_p);
    mbar_wait<true>(tr.ring.full + 8u * s, phase, abort_flag, p.status, kErrTransformWait);
    const uint32_t at0 = tr.ring.slot(s, 0) + uint32_t(rg.group * D + rg.tg * 8) * (BF16 ? 2u : 4u);
    auto piece = [&](int op, int i) {
      Raw<BF16> r;
      r.zero();
      if (on_row && rg.tg + i * rg.G < pieces)
        r.from_shared(at0 + uint32_t(op) * p.op_bytes + uint32_t(i * rg.G) * uint32_t(Raw<BF16>::kBytes));
      return r;
    };
    // x_out again, and sum(x_out a)
    Raw<BF16> xo[PP];
    F2 sxa = f2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const Raw<BF16> b = piece(0, i), x = piece(1, i), da = piece(2, i);
      Raw<BF16> g;
      if constexpr (GATE == kElementGate) g = piece(kGateOp, i);
      F2 v[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        F2 on = token_on;
        if constexpr (GATE == kElementGate) on = gate_of(g.pair(q)).on;
        const F2 n = post ? f2_mul(b.pair(q), rp) : b.pair(q);
        v[q] = outer<GATE>(n, gp[i].pair(q), post, on, x.pair(q), sc[i].pair(q), scaled);
      }
      xo[i].round(v);
#pragma unroll
      for (int q = 0; q < 4; ++q) sxa = f2_fma(xo[i].pair(q), f2_mul(gn[i].pair(q), da.pair(q)), sxa);
    }
    float s1[1] = {both(sxa)};
    group_sum<1>(s1, rg, red, flip);
    if (threadIdx.x == 0 && !ahead.done(p.parts)) {   // the slot of the batch before takes the batch stages - 1 ahead
      const int prev = s == 0 ? p.stages - 1 : s - 1;
      mbar_wait(tr.ring.empty + 8u * prev, s == 0 ? phase ^ 1u : phase, abort_flag, p.status, kErrProducerWait);
      tr.fetch(prev, ahead, rg.groups);
      ahead.next(rg.groups, p.T, p.parts);
    }
    const float cn = -(r_n * r_n) * r_n * (s1[0] * inv_d);
    const F2 c_n = f2(cn, cn);
    F2 pv[PP][4];   // p = g_post t (post), for the last pass
    F2 sbp = f2(0.f, 0.f), sgate = f2(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < PP; ++i) {
      const int pc = rg.tg + i * rg.G;
      const bool on = on_row && pc < pieces;
      const Raw<BF16> b = piece(0, i), x = piece(1, i), da = piece(2, i);
      Raw<BF16> g, dxo;
      dxo.zero();
      if constexpr (GATE == kElementGate) g = piece(kGateOp, i);
      if (carried) dxo = piece(kCarriedOp, i);
      F2 vx[4], vg[4], vt[4];
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const F2 xoq = xo[i].pair(q), a = f2_mul(gn[i].pair(q), da.pair(q));
        const F2 m = f2_fma(c_n, xoq, f2_fma(rn, a, dxo.pair(q)));
        dgn[i][q] = f2_fma(da.pair(q), f2_mul(xoq, rn), dgn[i][q]);
        vx[q] = scaled ? f2_mul(m, sc[i].pair(q)) : m;
        if (scaled) dsc[i][q] = f2_fma(m, x.pair(q), dsc[i][q]);
        const F2 n = post ? f2_mul(b.pair(q), rp) : b.pair(q);
        F2 t = m;
        if constexpr (GATE != kNoGate) {
          const F2 my = f2_mul(m, post ? f2_mul(n, gp[i].pair(q)) : n);
          if constexpr (GATE == kElementGate) {
            const Gate2 z = gate_of(g.pair(q));
            vg[q] = f2_mul(my, z.slope);
            t = f2_mul(m, z.on);
          } else {
            sgate = f2_add(sgate, my);
            t = f2_mul(m, token_on);
          }
        }
        vt[q] = t;
        if (post) {
          dgp[i][q] = f2_fma(t, n, dgp[i][q]);
          pv[i][q] = f2_mul(gp[i].pair(q), t);
          sbp = f2_fma(b.pair(q), pv[i][q], sbp);
        }
      }
      if (on) {
        Raw<BF16> o;
        o.round(vx);
        o.to_global(p.dx_in, off + pc * 8);
        if constexpr (GATE == kElementGate) {
          o.round(vg);
          o.to_global(p.dgate, off + pc * 8);
        }
        if (!post) {
          o.round(vt);
          o.to_global(p.dbranch, off + pc * 8);
        }
      }
    }
    if (post || GATE == kTokenGate) {   // uniform over the CTA
      float s2[2] = {both(sbp), both(sgate)};
      group_sum<2>(s2, rg, red2, flip2);
      if constexpr (GATE == kTokenGate) {
        if (on_row && rg.tg == 0) {
          const float d = s2[1] * tgate.slope;
          if constexpr (BF16) static_cast<__nv_bfloat16*>(p.dgate)[row] = __float2bfloat16_rn(d);
          else static_cast<float*>(p.dgate)[row] = d;
        }
      }
      if (post && on_row) {
        const float cp = -(r_p * r_p) * r_p * (s2[0] * inv_d);
        const F2 c_p = f2(cp, cp);
#pragma unroll
        for (int i = 0; i < PP; ++i) {
          const int pc = rg.tg + i * rg.G;
          if (pc < pieces) {
            const Raw<BF16> b = piece(0, i);
            F2 v[4];
#pragma unroll
            for (int q = 0; q < 4; ++q) v[q] = f2_fma(c_p, b.pair(q), f2_mul(rp, pv[i][q]));
            Raw<BF16> o;
            o.round(v);
            o.to_global(p.dbranch, off + pc * 8);
          }
        }
      }
    }
    __syncwarp();   // the warp has read all it needs of the slot
    if ((threadIdx.x & 31) == 0) mbar_arrive(tr.ring.empty + 8u * s);
    if (++s == p.stages) s = 0, phase ^= 1u;
    if (w.last_of_part(rg.groups)) {
      if (p.pg_next) write_gain_partial<PP>(dgn, rg, pieces, gsm, p.pg_next + int64_t(w.part) * D);
      if (p.pg_post) write_gain_partial<PP>(dgp, rg, pieces, gsm, p.pg_post + int64_t(w.part) * D);
      if (p.pg_scale) write_gain_partial<PP>(dsc, rg, pieces, gsm, p.pg_scale + int64_t(w.part) * D);
#pragma unroll
      for (int i = 0; i < PP; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) dgn[i][q] = dgp[i][q] = dsc[i][q] = f2(0.f, 0.f);
    }
  }
  if (threadIdx.x == 0 && *abort_flag) __nanosleep(200000);   // an expired wait: let copies in flight land first
}

// out[a][col] = sum over the parts, a the three gains (blockIdx.y): 32 columns per CTA, the parts dealt to 32 row lanes
// whose sums are added in lane order.
struct GainSums {
  const float* part[3];
  float* out[3];
  int parts, D;
};
__global__ void __launch_bounds__(1024) k_gated_gain_sums(const GainSums p) {
  __shared__ float red[32][33];
  const int col = blockIdx.x * 32 + (threadIdx.x & 31), lane_row = threadIdx.x >> 5;
  const float* part = p.part[blockIdx.y];
  float s = 0.f;
  if (col < p.D) {
#pragma unroll 8
    for (int r = lane_row; r < p.parts; r += 32) s += part[int64_t(r) * p.D + col];
  }
  red[lane_row][threadIdx.x & 31] = s;
  __syncthreads();
  if (lane_row == 0 && col < p.D) {
    float t = 0.f;
#pragma unroll
    for (int r = 0; r < 32; ++r) t += red[r][threadIdx.x];
    p.out[blockIdx.y][col] = t;
  }
}

// ------------------------------------------------------------------------------------------------ host
struct Geometry {
  int pp, G, ctas, stages;
  int64_t parts;
  uint32_t op_bytes, smem;
};
constexpr int kMaxParts = 1024;
Geometry geometry(int64_t T, int D, bool bf16, int nops, bool backward) {
  Geometry g{};
  const int pieces = D / 8;
  g.pp = pieces_per_thread_for(pieces);
  g.G = group_threads_for(pieces, g.pp);
  const int groups = kGroupThreads / g.G;
  g.ctas = g.pp <= 2 && (bf16 || !backward) ? 2 : 1;
  g.op_bytes = (uint32_t(groups) * uint32_t(D) * (bf16 ? 2u : 4u) + 127u) & ~127u;
  if (g.ctas == 2 && 2 * nops * int64_t(g.op_bytes) > 100 * 1024) g.ctas = 1;   // two stages have to fit
  g.stages = ring_stages_for(g.ctas, nops, g.op_bytes, 4608, 6);
  g.smem = ring_bytes(g.stages, nops, g.op_bytes);
  // one part per resident CTA: the fewest partial rows, and the rows are dealt evenly
  g.parts = std::min<int64_t>(std::min<int64_t>(kMaxParts, int64_t(ce::sm_count()) * g.ctas), (T + groups - 1) / groups);
  return g;
}

void require_shape(bool bf16, int64_t T, int D, const std::string& who) {
  NM_REQUIRE(T >= 0, who + ": the row count T cannot be negative");
  NM_REQUIRE(D > 0 && D % 8 == 0, who + ": D must be a positive multiple of 8 (rows are moved in 16-byte pieces)");
  NM_REQUIRE(D <= (bf16 ? 8192 : 4096), who + ": D <= 8192 (bf16 storage) or 4096 (f32)");
}
void require_gate(int gate_kind, const void* gate, const std::string& who) {
  NM_REQUIRE(gate_kind >= kNoGate && gate_kind <= kElementGate, who + ": gate_kind 0 (none), 1 (per token) or 2 (per element)");
  NM_REQUIRE((gate != nullptr) == (gate_kind != kNoGate), who + ": a gate goes with gate_kind 1 or 2, and only with those");
}
template <bool BF16, int PP, int GATE>
void launch_one(bool backward, const TailParams& p, const Geometry& g, cudaStream_t st) {
  auto kern = backward ? k_gated_bwd<BF16, PP, GATE> : k_gated_fwd<BF16, PP, GATE>;
  NM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(g.smem)));
  kern<<<unsigned(g.parts), kGroupThreads, g.smem, st>>>(p);
  NM_CUDA(cudaGetLastError());
}
template <bool BF16, int PP>
void launch_gate(int gate, bool backward, const TailParams& p, const Geometry& g, cudaStream_t st) {
  if (gate == kNoGate) launch_one<BF16, PP, kNoGate>(backward, p, g, st);
  else if (gate == kTokenGate) launch_one<BF16, PP, kTokenGate>(backward, p, g, st);
  else launch_one<BF16, PP, kElementGate>(backward, p, g, st);
}
template <bool BF16>
void launch_pp(int gate, bool backward, const TailParams& p, const Geometry& g, cudaStream_t st) {
  if (g.pp == 1) launch_gate<BF16, 1>(gate, backward, p, g, st);
  else if (g.pp == 2) launch_gate<BF16, 2>(gate, backward, p, g, st);
  else launch_gate<BF16, 4>(gate, backward, p, g, st);
}
void launch(bool bf16, int gate, bool backward, TailParams& p, int nops, cudaStream_t st) {
  NM_REQUIRE(ce::device_arch() >= 100, "gated tail: this library holds sm_100a code only");
  const Geometry g = geometry(p.T, p.D, bf16, nops, backward);
  p.parts = g.parts, p.G = g.G, p.stages = g.stages, p.nops = nops, p.op_bytes = g.op_bytes;
  p.status = row_status_word();
  if (bf16) launch_pp<true>(gate, backward, p, g, st);
  else launch_pp<false>(gate, backward, p, g, st);
}

}  // namespace

void gated_tail_fwd(bool bf16, int gate_kind, const void* branch, const void* x_in, const void* gate, const void* res_scale,
                    const void* g_post, const void* g_next, void* x_out, void* a_next, float* rstd_post, float* rstd_next,
                    int64_t T, int D, float eps, cudaStream_t st) {
  const std::string who = "gated_tail_fwd";
  require_shape(bf16, T, D, who);
  NM_REQUIRE(gate_kind >= kNoGate && gate_kind <= kElementGate, who + ": gate_kind 0 (none), 1 (per token) or 2 (per element)");
  if (T == 0) return;
  require_gate(gate_kind, gate, who);
  NM_REQUIRE(branch && x_in && x_out, who + ": branch, x_in and x_out are required");
  NM_REQUIRE(!a_next || g_next, who + ": a_next needs g_next");
  NM_REQUIRE(aligned16(branch, x_in, res_scale, g_post, g_next, x_out, a_next), who + ": every row pointer must be 16-byte aligned");
  NM_REQUIRE(gate_kind != kElementGate || aligned16(gate), who + ": a gate per element must be 16-byte aligned");
  TailParams p{};
  p.branch = branch, p.x_in = x_in, p.gate = gate, p.res_scale = res_scale, p.g_post = g_post, p.g_next = g_next;
  p.x_out = x_out, p.a_next = a_next, p.rstd_post = rstd_post, p.rstd_next = rstd_next;
  p.T = T, p.D = D, p.eps = eps;
  launch(bf16, gate_kind, false, p, gate_kind == kElementGate ? 3 : 2, st);
}

uint64_t gated_tail_workspace_bytes(int64_t T, int D) {
  require_shape(true, T, D, "gated_tail");
  // an upper bound that does not depend on the device: a part holds one row at least
  return uint64_t(3) * uint64_t(std::min<int64_t>(std::max<int64_t>(T, 1), kMaxParts)) * uint64_t(D) * 4;
}

void gated_tail_bwd(bool bf16, int gate_kind, const void* dx_out, const void* da_next, const void* x_in, const void* branch,
                    const void* gate, const void* res_scale, const void* g_post, const void* g_next, const float* rstd_post,
                    const float* rstd_next, void* dx_in, void* dbranch, void* dgate, float* dg_next, float* dg_post,
                    float* dres_scale, int64_t T, int D, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  const std::string who = "gated_tail_bwd";
  require_shape(bf16, T, D, who);
  NM_REQUIRE(gate_kind >= kNoGate && gate_kind <= kElementGate, who + ": gate_kind 0 (none), 1 (per token) or 2 (per element)");
  NM_REQUIRE(!dg_post || g_post || T == 0, who + ": dg_post without g_post");
  NM_REQUIRE(!dres_scale || res_scale || T == 0, who + ": dres_scale without res_scale");
  const bool sums = dg_next || dg_post || dres_scale;
  if (T == 0 && !sums) return;
  TailParams p{};
  if (T > 0) {
    require_gate(gate_kind, gate, who);
    NM_REQUIRE(da_next && x_in && branch && g_next && rstd_next, who + ": da_next, x_in, branch, g_next and rstd_next are required");
    NM_REQUIRE(!g_post || rstd_post, who + ": a post-norm needs rstd_post");
    NM_REQUIRE(dx_in && dbranch, who + ": dx_in and dbranch are required");
    NM_REQUIRE((dgate != nullptr) == (gate_kind != kNoGate), who + ": dgate goes with a gate, and only with one");
    NM_REQUIRE(aligned16(dx_out, da_next, x_in, branch, res_scale, g_post, g_next, dx_in, dbranch),
               who + ": every row pointer must be 16-byte aligned");
    NM_REQUIRE(gate_kind != kElementGate || aligned16(gate, dgate), who + ": a gate per element must be 16-byte aligned");
  }
  if (sums) {
    NM_REQUIRE(ws != nullptr && reinterpret_cast<uintptr_t>(ws) % 16 == 0, who + ": a 16-byte aligned workspace is required");
    NM_REQUIRE(ws_bytes >= gated_tail_workspace_bytes(T, D), who + ": the workspace is smaller than nm_gated_tail_workspace_bytes()");
  }
  GainSums gs{};
  const int64_t stride = std::min<int64_t>(std::max<int64_t>(T, 1), kMaxParts) * D;
  float* part = static_cast<float*>(ws);
  int n = 0;
  auto sum_into = [&](float* out) -> float* {
    if (!out) return nullptr;
    gs.part[n] = part + n * stride, gs.out[n] = out;
    return part + (n++) * stride;
  };
  p.pg_next = sum_into(dg_next), p.pg_post = sum_into(dg_post), p.pg_scale = sum_into(dres_scale);
  if (T > 0) {
    p.branch = branch, p.x_in = x_in, p.gate = gate, p.res_scale = res_scale, p.g_post = g_post, p.g_next = g_next;
    p.rstd_post = const_cast<float*>(rstd_post), p.rstd_next = const_cast<float*>(rstd_next);
    p.dx_out = dx_out, p.da_next = da_next, p.dx_in = dx_in, p.dbranch = dbranch, p.dgate = dgate;
    p.T = T, p.D = D;
    launch(bf16, gate_kind, true, p, 3 + (gate_kind == kElementGate ? 1 : 0) + (dx_out ? 1 : 0), st);
  }
  if (n > 0) {
    NM_REQUIRE(ce::device_arch() >= 100, "gated tail: this library holds sm_100a code only");
    gs.parts = int(p.parts), gs.D = D;   // no rows: no parts, the gradient of nothing
    k_gated_gain_sums<<<dim3(unsigned((D + 31) / 32), unsigned(n)), 1024, 0, st>>>(gs);
    NM_CUDA(cudaGetLastError());
  }
}

}  // namespace nm::ew

extern "C" {

int nm_gated_tail_fwd(int dtype, int gate_kind, const void* branch, const void* x_in, const void* gate,
                      const void* res_scale, const void* g_post, const void* g_next, void* x_out, void* a_next,
                      float* rstd_post, float* rstd_next, int64_t T, int D, float eps, void* stream) {
  return nm::abi::guarded([&] {
    NM_REQUIRE(dtype == 0 || dtype == 1, "nm_gated_tail_fwd: storage 0 (f32) or 1 (bf16)");
    nm::ew::gated_tail_fwd(dtype == 1, gate_kind, branch, x_in, gate, res_scale, g_post, g_next, x_out, a_next, rstd_post,
                           rstd_next, T, D, eps, static_cast<cudaStream_t>(stream));
  });
}

uint64_t nm_gated_tail_workspace_bytes(int64_t T, int D) {
  return nm::abi::guarded_value<uint64_t>(0, [&] { return nm::ew::gated_tail_workspace_bytes(T, D); });
}

int nm_gated_tail_bwd(int dtype, int gate_kind, const void* dx_out, const void* da_next, const void* x_in,
                      const void* branch, const void* gate, const void* res_scale, const void* g_post, const void* g_next,
                      const float* rstd_post, const float* rstd_next, void* dx_in, void* dbranch, void* dgate,
                      float* dg_next, float* dg_post, float* dres_scale, int64_t T, int D, void* workspace,
                      uint64_t workspace_bytes, void* stream) {
  return nm::abi::guarded([&] {
    NM_REQUIRE(dtype == 0 || dtype == 1, "nm_gated_tail_bwd: storage 0 (f32) or 1 (bf16)");
    nm::ew::gated_tail_bwd(dtype == 1, gate_kind, dx_out, da_next, x_in, branch, gate, res_scale, g_post, g_next, rstd_post,
                           rstd_next, dx_in, dbranch, dgate, dg_next, dg_post, dres_scale, T, D, workspace, workspace_bytes,
                           static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
