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
// directions share through() below, and 2 bytes per element less.
// sigmoid(g) = r = 1 / (1 + e) and 1 - sigmoid(g) = e r with e = exp(-g): no cancellation at either end.
// Row groups and batch ring as in ew_rows.cuh, a CTA per part of consecutive rows. What bounds them is HBM (10 and 16 bytes
// per element in bf16 with a gate per element), and under the board's power cap, at 1.7 GHz, the issue slots. Forward,
// 65536 x 2048: 229 us (5.9 TB/s), 244 to 260 us under the cap; the backward's figures stand at its kernel.
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

// Two neighbouring f32 values, each operation individually rounded: the packed f32x2 form (fma2, mul2) and the plain one give
// the same bits. Written as one asm block each: with the values held as 64-bit registers between the operations (ew_rows.cuh)
// the moves that put single results side by side ate the gain. Backward, 65536 x 2048: 279 million warp instructions with
// plain arithmetic, 243 million packed (390 -> 387 us under the power cap, 349 us at full clock either way: HBM; before the
// quotient below was corrected). Forward, the same size: 232 -> 231 us, 251 -> 250 us under the cap.
struct Two {
  float x, y;
};
__device__ __forceinline__ Two two(float a, float b) { return Two{a, b}; }
__device__ __forceinline__ Two mul(Two a, Two b) { return Two{__fmul_rn(a.x, b.x), __fmul_rn(a.y, b.y)}; }
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("{\n\t"
      ".reg .b64 a, b, c;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 a, a, b, c;\n\t"
      "mov.b64 {%0, %1}, a;\n\t"
      "}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("{\n\t"
      ".reg .b64 a, b;\n\t"
      "mov.b64 a, {%2, %3};\n\t"
      "mov.b64 b, {%4, %5};\n\t"
      "mul.rn.f32x2 a, a, b;\n\t"
      "mov.b64 {%0, %1}, a;\n\t"
      "}"
      : "=f"(r.x), "=f"(r.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return r;
}
__device__ __forceinline__ Two two_of(uint32_t w) { return Two{lo_f32(w), hi_f32(w)}; }

enum GateKind : int { kNoGate = 0, kTokenGate = 1, kElementGate = 2 };

// A thread's unit is four columns: their operands are read from the slot and used at once (with eight, the operands alone
// push the backward past its 128 registers). Warp w of a row group owns the quads [32 N w, 32 N (w + 1)), lane l of it the
// quads l, l + 32, ...: neighbours side by side, and distances between a thread's quads that are constants.
template <bool BF16>
struct Quad {
  uint32_t w[BF16 ? 2 : 4];
  static constexpr uint32_t kBytes = BF16 ? 8 : 16;
  __device__ __forceinline__ void fill(float v) {
    const uint32_t u = __float_as_uint(v);
    if constexpr (BF16) w[0] = w[1] = (u >> 16) | (u & 0xffff0000u);
    else w[0] = w[1] = w[2] = w[3] = u;
  }
  __device__ __forceinline__ void from_shared(uint32_t at) {
    if constexpr (BF16) {
      asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(w[0]), "=r"(w[1]) : "r"(at) : "memory");
    } else {
      const uint4 q = nm::ptx::ld_shared_v4(at);
      w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
    }
  }
  __device__ __forceinline__ void to_shared(uint32_t at) const {
    if constexpr (BF16) asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(at), "r"(w[0]), "r"(w[1]) : "memory");
    else nm::ptx::st_shared_v4(at, w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ void from_global(const void* p, int64_t quad) {
    if constexpr (BF16) {
      const uint2 v = __ldg(static_cast<const uint2*>(p) + quad);
      w[0] = v.x, w[1] = v.y;
    } else {
      const uint4 v = __ldg(static_cast<const uint4*>(p) + quad);
      w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
  }
  __device__ __forceinline__ void to_global(uint8_t* p) const {
    if constexpr (BF16) *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
  }
  __device__ __forceinline__ Two pair(int i) const {
    if constexpr (BF16) return two_of(w[i]);
    else return two(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
  }
  __device__ __forceinline__ void round(Two a, Two b) {   // to the storage type
    if constexpr (BF16) {
      w[0] = pack_bf16x2(a.x, a.y), w[1] = pack_bf16x2(b.x, b.y);
    } else {
      w[0] = __float_as_uint(a.x), w[1] = __float_as_uint(a.y), w[2] = __float_as_uint(b.x), w[3] = __float_as_uint(b.y);
    }
  }
};

__device__ __forceinline__ float scalar_of(const void* p, int64_t i, bool bf16) {
  return bf16 ? __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]) : static_cast<const float*>(p)[i];
}

__device__ __forceinline__ float gate_exponent(float a) {
  float r;
  asm("min.NaN.f32 %0, %1, 0f42FC0000;" : "=f"(r) : "f"(a));
  return r;
}
__device__ __forceinline__ float rcp_approx(float a) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(a));
  return r;
}
constexpr float kLog2e = 1.4426950408889634f, kLargest = 3.402823466e38f;

// What x_out is made of, s x + y / (1 + exp(-gate)), takes expf and a quotient of half a step: x_out is rounded to the storage
// type, and in bf16 a value next to a tie lands a whole step (2^-8) away for a difference of 2^-24, which every sum over x_out
// shows. With ex2.approx of a rounded product and rcp.approx the f32 sums stood up to 2e-5 from those of the formula's own f32
// operations, now 3e-7 (12 % of the forward and 6 % of the backward under the power cap). The quotient y / b is P. Markstein's
// for machines with a fused multiply-add (Computation of elementary functions on the IBM RISC System/6000 processor, IBM J. Res.
// Develop. 34, 1990): q = y r with r about 1 / b, then q + (y - q b) r, whose remainder is rounded once. With r and q each within
// 2^-22 (rcp.approx 1 ulp, the product) what the one correction leaves is under 2^-43 before the last rounding: half a step and
// a little, not always the nearest value. The gate stops at -87, where the quotient is as good as 0; a NaN
// passes through. The remainder of an infinite y is inf - inf; INF makes it a number and the quotient infinite. The backward
// does without: the row's rstd_next is 0 and 0 inf = NaN reaches all its gradients either way. A part that the call leaves out
// is a factor of one (exact), so nothing branches on it. Both directions get the same bits from these.
struct Opening {
  Two a, r;   // -(1 + exp(-gate)), and about the reciprocal of 1 + exp(-gate)
};
__device__ __forceinline__ float exp_of_minus(float g) {
  asm("max.NaN.f32 %0, %0, 0fC2AE0000;" : "+f"(g));
  return expf(-g);
}
__device__ __forceinline__ Opening opening_of(Two g) {
  const Two e = two(exp_of_minus(g.x), exp_of_minus(g.y));
  Opening o;
  o.a = fma2(e, two(-1.f, -1.f), two(-1.f, -1.f));
  o.r = two(rcp_approx(-o.a.x), rcp_approx(-o.a.y));
  return o;
}
template <bool INF = true>
__device__ __forceinline__ Two through(Two y, const Opening& o) {   // y / (1 + exp(-gate))
  const Two q = mul2(y, o.r);
  Two rest = fma2(q, o.a, y);
  if constexpr (INF) rest = two(fmaxf(rest.x, -kLargest), fmaxf(rest.y, -kLargest));
  return fma2(rest, o.r, q);
}
__device__ __forceinline__ float both(Two v) { return v.x + v.y; }

// sigmoid(g) and 1 - sigmoid(g) of two gates, for the gradients. f32 storage shows all bits of them and takes what x_out takes:
// within 6 and 7 half steps. In bf16 storage they are factors of results that are rounded to 2^-8: ex2.approx of a rounded product
// (|g| half steps of f32) and rcp.approx. There the exponent stops at 126: beyond it the open part is 2^-126 instead of 0, and
// e * on stays a number (a NaN passes through).
struct Gate2 {
  Two on, off;
};
template <bool BF16>
__device__ __forceinline__ Gate2 gate_of(Two g) {
  Two e;
  Gate2 r;
  if constexpr (BF16) {
    e = two(nm::ptx::ex2_approx(gate_exponent(__fmul_rn(g.x, -kLog2e))),
            nm::ptx::ex2_approx(gate_exponent(__fmul_rn(g.y, -kLog2e))));
    r.on = two(rcp_approx(__fadd_rn(1.f, e.x)), rcp_approx(__fadd_rn(1.f, e.y)));
  } else {
    e = two(exp_of_minus(g.x), exp_of_minus(g.y));
    r.on = through<false>(two(1.f, 1.f), opening_of(g));
  }
  r.off = mul(e, r.on);
  return r;
}

struct TailParams {
  const void* branch; const void* x_in; const void* gate; const void* res_scale; const void* g_post; const void* g_next;
  void* x_out; void* a_next;
  float* rstd_post; float* rstd_next;            // written forward, read backward
  // backward
  const void* dx_out; const void* da_next;
  void* dx_in; void* dbranch; void* dgate;
  float* pg_next; float* pg_post; float* pg_scale;   // [parts, D] partial sums, or nullptr
  const void* op[5];                             // the row operands in slot order
  int64_t T, parts;
  int D, G, stages, nops;
  uint32_t op_bytes;
  float eps;
  uint32_t* status;
};

template <int N>
__device__ __forceinline__ int first_quad(const RowGroup& rg) {
  return (rg.tg >> 5) * 32 * N + (rg.tg & 31);
}

// Ring set-up shared by both directions. A CTA owns one part, the rows [row0, row0 + rows); `fetch` (thread 0) brings the
// batch that begins at row r of it, every operand, into a slot.
template <bool BF16>
struct TailRing {
  RowRing ring;
  int D, rows;
  int64_t row0;
  __device__ __forceinline__ void begin(uint8_t* raw, const TailParams& p, int* abort_word) {
    using namespace nm::ptx;
    D = p.D;
    row0 = int64_t(blockIdx.x) * p.T / p.parts;
    rows = int((int64_t(blockIdx.x) + 1) * p.T / p.parts - row0);
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
  __device__ __forceinline__ void fetch(const TailParams& p, int s, int r, int groups) const {
    using namespace nm::ptx;
    const uint32_t bytes = uint32_t(min(groups, rows - r)) * uint32_t(D) * (BF16 ? 2u : 4u);
    const uint32_t bar = ring.full + 8u * s;
    const int64_t at = (row0 + r) * D * (BF16 ? 2 : 4);
    mbar_arrive_expect_tx(bar, bytes * uint32_t(ring.nops));
#pragma unroll
    for (int o = 0; o < 5; ++o)
      if (o < ring.nops) bulk_load(ring.slot(s, o), static_cast<const uint8_t*>(p.op[o]) + at, bytes, bar);
  }
  // the first stages - 1 batches; returns the row where fetching goes on
  __device__ __forceinline__ int fill(const TailParams& p, int groups) const {
    int r = 0;
    for (int s = 0; s < p.stages - 1 && r < rows; ++s, r += groups) fetch(p, s, r, groups);
    return r;
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
  using Q = Quad<BF16>;
  constexpr int N = 2 * PP;
  const RowGroup rg = row_group(p.G);
  const int quads = p.D / 4, first = first_quad<N>(rg);
  const bool post = p.g_post != nullptr, scaled = p.res_scale != nullptr;
  const float inv_d = 1.f / float(p.D);
  TailRing<BF16> tr;
  tr.begin(ring_raw, p, &abort_word);
  int ahead = 0;
  if (threadIdx.x == 0) ahead = tr.fill(p, rg.groups);
  Q gn[N], gp[N], sc[N];
#pragma unroll
  for (int j = 0; j < N; ++j) {
    gn[j].fill(0.f), gp[j].fill(1.f), sc[j].fill(1.f);
    if (first + 32 * j < quads) {
      if (p.a_next) gn[j].from_global(p.g_next, first + 32 * j);
      if (post) gp[j].from_global(p.g_post, first + 32 * j);
      if (scaled) sc[j].from_global(p.res_scale, first + 32 * j);
    }
  }
  auto gate_scalar = [&](int r) {
    if constexpr (GATE == kTokenGate) return r < tr.rows ? scalar_of(p.gate, tr.row0 + r, BF16) : 0.f;
    else return 0.f;
  };
  float gate_next = gate_scalar(rg.group);   // one batch ahead
  int flip = 0, flip1 = 0, s = 0;
  uint32_t phase = 0;
  for (int r0 = rg.group; r0 < tr.rows + rg.group; r0 += rg.groups) {   // batches; this thread's row of the part is r0
    const bool on_row = r0 < tr.rows;
    Opening token;
    if constexpr (GATE == kTokenGate) {
      token = opening_of(two(gate_next, gate_next));
      gate_next = gate_scalar(r0 + rg.groups);
    }
    mbar_wait<true>(tr.ring.full + 8u * s, phase, abort_flag, p.status, kErrTransformWait);
    const uint32_t at0 = tr.ring.slot(s, 0) + uint32_t(rg.group * quads + first) * Q::kBytes;
    auto quad = [&](int op, int j) {
      Q r;
      r.from_shared(at0 + uint32_t(op) * p.op_bytes + uint32_t(32 * j) * Q::kBytes);
      return r;
    };
    Two rp = two(1.f, 1.f);
    Two bb[N][2];
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!(on_row && first + 32 * j < quads)) continue;
      const Q b = quad(0, j);
      bb[j][0] = b.pair(0), bb[j][1] = b.pair(1);
    }
    if (post) {   // uniform over the CTA
      Two sbb = two(0.f, 0.f);
#pragma unroll
      for (int j = 0; j < N; ++j) {
        if (!(on_row && first + 32 * j < quads)) continue;
#pragma unroll
        for (int q = 0; q < 2; ++q) sbb = fma2(bb[j][q], bb[j][q], sbb);
      }
      float sum[1] = {both(sbb)};
      group_sum<1>(sum, rg, red, flip);
      const float r = rsqrtf(fmaf(sum[0], inv_d, p.eps));
      if (on_row && p.rstd_post && rg.tg == 0) p.rstd_post[tr.row0 + r0] = r;
      rp = two(r, r);
    }
    const int64_t out0 = ((tr.row0 + r0) * quads + first) * int64_t(Q::kBytes);
    Q xo[N];
    Two sxx = two(0.f, 0.f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!(on_row && first + 32 * j < quads)) continue;
      const Q x = quad(1, j);
      Q g;
      if constexpr (GATE == kElementGate) g = quad(2, j);
      Two v[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        Two u = mul2(mul2(bb[j][q], rp), gp[j].pair(q));
        if constexpr (GATE == kTokenGate) u = through(u, token);
        if constexpr (GATE == kElementGate) u = through(u, opening_of(g.pair(q)));
        v[q] = fma2(sc[j].pair(q), x.pair(q), u);
      }
      xo[j].round(v[0], v[1]);
      xo[j].to_global(static_cast<uint8_t*>(p.x_out) + out0 + 32 * j * int(Q::kBytes));
#pragma unroll
      for (int q = 0; q < 2; ++q) sxx = fma2(xo[j].pair(q), xo[j].pair(q), sxx);
    }
    float sum[1] = {both(sxx)};
    group_sum<1>(sum, rg, red1, flip1);
    if (threadIdx.x == 0 && ahead < tr.rows) {   // the slot of the batch before takes the batch stages - 1 ahead
      const int prev = s == 0 ? p.stages - 1 : s - 1;
      mbar_wait(tr.ring.empty + 8u * prev, s == 0 ? phase ^ 1u : phase, abort_flag, p.status, kErrProducerWait);
      tr.fetch(p, prev, ahead, rg.groups);
      ahead += rg.groups;
    }
    __syncwarp();   // the slot is not read again
    if ((threadIdx.x & 31) == 0) mbar_arrive(tr.ring.empty + 8u * s);
    if (++s == p.stages) s = 0, phase ^= 1u;
    if (on_row) {
      const float r = rsqrtf(fmaf(sum[0], inv_d, p.eps));
      if (p.rstd_next && rg.tg == 0) p.rstd_next[tr.row0 + r0] = r;
      if (p.a_next) {
        const Two rn = two(r, r);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          if (first + 32 * j >= quads) continue;
          Q o;
          o.round(mul2(gn[j].pair(0), mul2(xo[j].pair(0), rn)), mul2(gn[j].pair(1), mul2(xo[j].pair(1), rn)));
          o.to_global(static_cast<uint8_t*>(p.a_next) + out0 + 32 * j * int(Q::kBytes));
        }
      }
    }
  }
  if (threadIdx.x == 0 && *abort_flag) __nanosleep(200000);   // an expired wait: let copies in flight land first
}

// The gain sums of a CTA's row groups, added in group order, as one row of the partial buffer (smem: 256 float4).
template <int N>
__device__ __forceinline__ void write_quad_partial(const Two (&dg)[N][2], const RowGroup& rg, int quads, float* smem,
                                                   float* out_row) {
#pragma unroll
  for (int j = 0; j < N; ++j) {
    const int at = first_quad<N>(rg) + 32 * j;
    float4 v;
    v = make_float4(dg[j][0].x, dg[j][0].y, dg[j][1].x, dg[j][1].y);
    __syncthreads();
    reinterpret_cast<float4*>(smem)[threadIdx.x] = v;
    __syncthreads();
    if (rg.group == 0 && at < quads) {
      for (int g = 1; g < rg.groups; ++g) {
        const float4 o = reinterpret_cast<const float4*>(smem)[g * rg.G + rg.tg];
        v.x += o.x, v.y += o.y, v.z += o.z, v.w += o.w;
      }
      reinterpret_cast<float4*>(out_row)[at] = v;
    }
  }
}

// The second row sum needs the first (sum(branch p) is taken over m, which needs sum(x_out a)), but m is linear in it,
// m = h + c x_out with h = dx_out + r_n a and c = -r_n^3 sum(x_out a) / D, so
//   sum(u m) = sum(u h) + c sum(u x_out),   u = sigmoid(gate) y,
// and all sums are taken in the first pass, with one barrier per row. sum(branch p) = sum(u m) / r_p; for a gate per token
// sum(m y) is the same sum without the (constant) gate. x_out as stored and h stay in registers for the second pass, the
// gate is evaluated again; the gains lie in shared memory (of ones where the call has none). Beside a ring that takes
// nearly all of the SM's memory a spilled register is read back from L2, so the registers decide the form. Measured for
// 65536 x 2048 bf16 with a gate per element (floor 328 us at the copy rate): 811 us with the gate's two parts kept and eight
// columns at a time (spills), 414 us as quads without spills, 353 us with plain arithmetic instead of
// packed 64-bit registers and the next batch fetched before a batch is worked on (6.1 TB/s); 359-370 us, 402-426 us under the
// power cap, since the gate's quotient is corrected. Sixteen columns per thread beat eight (439 us).
template <bool BF16, int PP, int GATE>
__global__ void __launch_bounds__(kGroupThreads, PP <= 2 && BF16 ? 2 : 1) k_gated_bwd(const TailParams p) {
  using namespace nm::ptx;
  extern __shared__ __align__(128) uint8_t ring_raw[];
  __shared__ __align__(16) float red[2 * 8 * 4];
  __shared__ __align__(16) float gsm[kGroupThreads * 4];
  __shared__ int abort_word;
  volatile int* abort_flag = &abort_word;
  using Q = Quad<BF16>;
  using GainQ = Quad<BF16 && PP == 4>;   // gains widened to f32 where there is room for them
  constexpr int N = 2 * PP;
  const RowGroup rg = row_group(p.G);
  const int quads = p.D / 4, first = first_quad<N>(rg);
  const bool post = p.g_post != nullptr, carried = p.dx_out != nullptr;
  constexpr int kGateOp = 3, kCarriedOp = GATE == kElementGate ? 4 : 3;
  release_next();
  TailRing<BF16> tr;
  tr.begin(ring_raw, p, &abort_word);
  int ahead = 0;
  if (threadIdx.x == 0) ahead = tr.fill(p, rg.groups);
  // g_next, g_post, res_scale behind the ring (ones where the call has none)
  const uint32_t gains = (tr.ring.empty + 8u * uint32_t(p.stages) + 127u) & ~127u, gain_bytes = uint32_t(quads) * GainQ::kBytes;
  for (int a = 0; a < 3; ++a) {
    const void* src = a == 0 ? p.g_next : a == 1 ? p.g_post : p.res_scale;
    for (int at = threadIdx.x; at < quads; at += kGroupThreads) {
      Q raw;
      raw.fill(1.f);
      if (src) raw.from_global(src, at);
      GainQ wide;
      wide.round(raw.pair(0), raw.pair(1));
      wide.to_shared(gains + uint32_t(a) * gain_bytes + uint32_t(at) * GainQ::kBytes);
    }
  }
  __syncthreads();
  Two dgn[N][2], dgp[N][2], dsc[N][2];
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int q = 0; q < 2; ++q) dgn[j][q] = dgp[j][q] = dsc[j][q] = two(0.f, 0.f);
  const float inv_d = 1.f / float(p.D);
  // a row's scalars are asked for one batch ahead: every pass needs them at once
  struct Scalars {
    float r_n, r_p, gate;
  };
  auto scalars_of = [&](int r) {
    Scalars v{0.f, 1.f, 0.f};
    if (r < tr.rows) {
      const int64_t row = tr.row0 + r;
      v.r_n = __ldg(p.rstd_next + row);
      if (post) v.r_p = __ldg(p.rstd_post + row);
      if constexpr (GATE == kTokenGate) v.gate = scalar_of(p.gate, row, BF16);
    }
    return v;
  };
  Scalars mine = scalars_of(rg.group);
  int flip = 0, s = 0;
  uint32_t phase = 0;
  for (int r0 = rg.group; r0 < tr.rows + rg.group; r0 += rg.groups) {   // batches; this thread's row of the part is r0
    const bool on_row = r0 < tr.rows;
    const float r_n = mine.r_n, r_p = mine.r_p;
    Gate2 tgate{two(1.f, 1.f), two(0.f, 0.f)};
    Opening token;
    if constexpr (GATE == kTokenGate) {
      tgate = gate_of<BF16>(two(mine.gate, mine.gate));
      token = opening_of(two(mine.gate, mine.gate));
    }
    mine = scalars_of(r0 + rg.groups);
    const Two rn = two(r_n, r_n), rp = two(r_p, r_p);
    // the slot of the batch before takes the batch stages - 1 ahead, as early as can be: two stages are all that fit
    if (threadIdx.x == 0 && ahead < tr.rows) {
      const int prev = s == 0 ? p.stages - 1 : s - 1;
      mbar_wait(tr.ring.empty + 8u * prev, s == 0 ? phase ^ 1u : phase, abort_flag, p.status, kErrProducerWait);
      tr.fetch(p, prev, ahead, rg.groups);
      ahead += rg.groups;
    }
    mbar_wait<true>(tr.ring.full + 8u * s, phase, abort_flag, p.status, kErrTransformWait);
    const uint32_t at0 = tr.ring.slot(s, 0) + uint32_t(rg.group * quads + first) * Q::kBytes;
    const uint32_t gain0 = gains + uint32_t(first) * GainQ::kBytes;
    auto quad = [&](int op, int j) {
      Q r;
      r.from_shared(at0 + uint32_t(op) * p.op_bytes + uint32_t(32 * j) * Q::kBytes);
      return r;
    };
    auto gain = [&](int a, int j) {
      GainQ r;
      r.from_shared(gain0 + uint32_t(a) * gain_bytes + uint32_t(32 * j) * GainQ::kBytes);
      return r;
    };
    Q xo[N];
    Two h[N][2];
    Two sxa = two(0.f, 0.f), suh = sxa, sux = sxa;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!(on_row && first + 32 * j < quads)) continue;
      Two u[2], v[2];
      {
        Q g;
        if constexpr (GATE == kElementGate) g = quad(kGateOp, j);
        const Q b = quad(0, j), x = quad(1, j);
        const GainQ gp = gain(1, j), sc = gain(2, j);
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          u[q] = mul2(mul2(b.pair(q), rp), gp.pair(q));
          Two through_gate = u[q];
          if constexpr (GATE == kTokenGate) through_gate = through<false>(u[q], token);
          if constexpr (GATE == kElementGate) through_gate = u[q] = through<false>(u[q], opening_of(g.pair(q)));
          v[q] = fma2(sc.pair(q), x.pair(q), through_gate);
        }
      }
      xo[j].round(v[0], v[1]);
      const Q da = quad(2, j);
      Q dxo;
      dxo.fill(0.f);
      if (carried) dxo = quad(kCarriedOp, j);
      const GainQ gn = gain(0, j);
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const Two xoq = xo[j].pair(q), a = mul2(gn.pair(q), da.pair(q));
        sxa = fma2(xoq, a, sxa);
        h[j][q] = fma2(rn, a, dxo.pair(q));
        dgn[j][q] = fma2(da.pair(q), mul2(xoq, rn), dgn[j][q]);
        suh = fma2(u[q], h[j][q], suh);
        sux = fma2(u[q], xoq, sux);
      }
    }
    float sums[3] = {both(sxa), both(suh), both(sux)};
    group_sum<3>(sums, rg, red, flip);
    // the sum grows with x_out as r_n shrinks: r_n^3 by itself is 0 in f32 from x_out = 10^15 on
    const float cn = -(sums[0] * inv_d * r_n * r_n * r_n);
    const float sum_um = fmaf(cn, sums[2], sums[1]);    // without the gate when it is the token's
    const float token_on = tgate.on.x, token_off = tgate.off.x;
    if constexpr (GATE == kTokenGate) {
      if (on_row && rg.tg == 0) {
        const float d = sum_um * (token_on * token_off);
        if constexpr (BF16) static_cast<__nv_bfloat16*>(p.dgate)[tr.row0 + r0] = __float2bfloat16_rn(d);
        else static_cast<float*>(p.dgate)[tr.row0 + r0] = d;
      }
    }
    // -r_p^2 sum(branch p) / D with sum(branch p) = sum(u m) / r_p; the third r_p goes to the branch, whose size it has
    const float cp = post ? -((GATE == kTokenGate ? sum_um * token_on : sum_um) * inv_d * r_p) : 0.f;
    const Two c_n = two(cn, cn), c_p = two(cp, cp);
    const int64_t out0 = ((tr.row0 + r0) * quads + first) * int64_t(Q::kBytes);
#pragma unroll
    for (int j = 0; j < N; ++j) {
      if (!(on_row && first + 32 * j < quads)) continue;
      const Q b = quad(0, j), x = quad(1, j);
      Q g;
      if constexpr (GATE == kElementGate) g = quad(kGateOp, j);
      const GainQ gp = gain(1, j), sc = gain(2, j);
      Two vx[2], vg[2], vb[2];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const Two m = fma2(c_n, xo[j].pair(q), h[j][q]);
        vx[q] = mul2(m, sc.pair(q));
        dsc[j][q] = fma2(m, x.pair(q), dsc[j][q]);
        Two t = mul2(m, rp);   // t r_p from here on: its products with the branch are those of t with the normalised branch
        if constexpr (GATE == kTokenGate) t = mul2(t, tgate.on);
        Two off;
        if constexpr (GATE == kElementGate) {
          const Gate2 z = gate_of<BF16>(g.pair(q));
          t = mul2(t, z.on);
          off = z.off;
        }
        dgp[j][q] = fma2(t, b.pair(q), dgp[j][q]);
        const Two pr = mul2(gp.pair(q), t);
        if constexpr (GATE == kElementGate) vg[q] = mul2(mul2(pr, b.pair(q)), off);
        vb[q] = fma2(c_p, mul2(b.pair(q), rp), pr);
      }
      constexpr int kStep = 32 * int(Q::kBytes);
      Q o;
      o.round(vx[0], vx[1]);
      o.to_global(static_cast<uint8_t*>(p.dx_in) + out0 + j * kStep);
      o.round(vb[0], vb[1]);
      o.to_global(static_cast<uint8_t*>(p.dbranch) + out0 + j * kStep);
      if constexpr (GATE == kElementGate) {
        o.round(vg[0], vg[1]);
        o.to_global(static_cast<uint8_t*>(p.dgate) + out0 + j * kStep);
      }
    }
    __syncwarp();   // the warp has read all it needs of the slot
    if ((threadIdx.x & 31) == 0) mbar_arrive(tr.ring.empty + 8u * s);
    if (++s == p.stages) s = 0, phase ^= 1u;
  }
  if (p.pg_next) write_quad_partial<N>(dgn, rg, quads, gsm, p.pg_next + int64_t(blockIdx.x) * p.D);
  if (p.pg_post) write_quad_partial<N>(dgp, rg, quads, gsm, p.pg_post + int64_t(blockIdx.x) * p.D);
  if (p.pg_scale) write_quad_partial<N>(dsc, rg, quads, gsm, p.pg_scale + int64_t(blockIdx.x) * p.D);
  if (threadIdx.x == 0 && *abort_flag) __nanosleep(200000);   // an expired wait: let copies in flight land first
}

// out[a][col] = sum over the parts, a the three gains (blockIdx.y): 32 columns per CTA, the parts dealt to 32 row lanes
// whose sums are added in lane order. Bound by latency: ten loads in a row, some 5 us.
struct GainSums {
  const float* part[3];
  float* out[3];
  int parts, D;
};
__global__ void __launch_bounds__(1024) k_gated_gain_sums(const GainSums p) {
  __shared__ float red[32][33];
  nm::ptx::after_previous();
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
  g.ctas = !backward ? (g.pp <= 2 ? 2 : 1) : !bf16 ? 1 : g.pp <= 2 ? 2 : 1;
  g.op_bytes = (uint32_t(groups) * uint32_t(D) * (bf16 ? 2u : 4u) + 127u) & ~127u;
  const uint32_t gain_bytes = backward ? 3u * uint32_t(D) * (bf16 && g.pp == 4 ? 2u : 4u) + 128u : 0u;
  // two stages have to fit beside the gains
  while (g.ctas > 1 && (2 * nops * int64_t(g.op_bytes) + gain_bytes) * g.ctas > 210 * 1024) --g.ctas;
  g.stages = ring_stages_for(g.ctas, nops, g.op_bytes, 4864 + gain_bytes, 6);
  g.smem = ring_bytes(g.stages, nops, g.op_bytes) + gain_bytes;
  // one part per resident CTA: the fewest partial rows, and the rows are dealt evenly
  g.parts = std::min<int64_t>(std::min<int64_t>(kMaxParts, int64_t(ce::sm_count()) * g.ctas), (T + groups - 1) / groups);
  return g;
}

void require_shape(bool bf16, int64_t T, int D, const std::string& who) {
  NM_REQUIRE(T >= 0, who + ": the row count T cannot be negative");
  NM_REQUIRE(D > 0 && D % 8 == 0, who + ": D must be a positive multiple of 8 (rows are moved in 16-byte pieces)");
  NM_REQUIRE(D <= (bf16 ? 8192 : 4096), who + ": D <= 8192 (bf16 storage) or 4096 (f32)");
}
template <class... P>
void require_element_aligned(bool bf16, const void* gate, const void* dgate, const std::string& who, const P*... f32) {
  const uintptr_t size = bf16 ? 2 : 4;
  NM_REQUIRE(reinterpret_cast<uintptr_t>(gate) % size == 0 && reinterpret_cast<uintptr_t>(dgate) % size == 0,
             who + ": a gate per token must be aligned to its element size");
  NM_REQUIRE(((reinterpret_cast<uintptr_t>(f32) % 4 == 0) && ...), who + ": statistics and [D] gradients must be 4-byte aligned");
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
  require_element_aligned(bf16, gate, nullptr, who, rstd_post, rstd_next);
  TailParams p{};
  p.branch = branch, p.x_in = x_in, p.gate = gate, p.res_scale = res_scale, p.g_post = g_post, p.g_next = g_next;
  p.x_out = x_out, p.a_next = a_next, p.rstd_post = rstd_post, p.rstd_next = rstd_next;
  p.T = T, p.D = D, p.eps = eps;
  p.op[0] = branch, p.op[1] = x_in, p.op[2] = gate;
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
  require_element_aligned(bf16, gate, dgate, who, rstd_post, rstd_next, dg_next, dg_post, dres_scale);
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
    const bool per_element = gate_kind == kElementGate;
    p.op[0] = branch, p.op[1] = x_in, p.op[2] = da_next, p.op[3] = per_element ? gate : dx_out, p.op[4] = dx_out;
    launch(bf16, gate_kind, true, p, 3 + (gate_kind == kElementGate ? 1 : 0) + (dx_out ? 1 : 0), st);
  }
  if (n > 0) {
    NM_REQUIRE(ce::device_arch() >= 100, "gated tail: this library holds sm_100a code only");
    gs.parts = int(p.parts), gs.D = D;   // no rows: no parts, the gradient of nothing
    ce::launch_after(k_gated_gain_sums, dim3(unsigned((D + 31) / 32), unsigned(n)), 1024, 0, st, gs);
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
