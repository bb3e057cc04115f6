// Embedding lookup with scaling, and its gradient by sorted tokens: the other end of the vocabulary matrix (a tied model
// adds the gradient below into the buffer that the fused CE accumulates dW in).
//   forward   y[t, :] = round(scale * E[token_t, :])             a token outside [0, V) gives a row of zeros
//   backward  dE[v, :] (+)= scale * sum_{t: token_t = v} dy[t, :]  in f32; a token outside [0, V) contributes nothing
// The backward has no floating-point atomics: tokens are sorted by a stable radix sort, a run of equal tokens is summed
// in ascending t, and long runs are cut at places that depend on the sorted tokens alone, so that the same call gives the
// same bits. Counterpart in the reference: src/kernels/elementwise/embed.cu.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <climits>
#include <string>

#include "abi_guard.hpp"
#include "ce_internal.hpp"
#include "ew_api.hpp"
#include "ew_rows.cuh"
#include "marincpp/capi_ew.h"

namespace nm::ew {
namespace {

constexpr int kThreads = 256;

// Eight consecutive elements of a row in either storage type, as f32.
template <bool BF16>
struct Eight;
template <>
struct Eight<true> {
  uint4 q;
  __device__ __forceinline__ void load(const void* p, int64_t at) { q = __ldg(reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(p) + at)); }
  __device__ __forceinline__ void get(float* f) const { unpack8(q, f); }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* f) {
    *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at) = pack8(f);
  }
};
template <>
struct Eight<false> {
  float4 a, b;
  __device__ __forceinline__ void load(const void* p, int64_t at) {
    const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p) + at);
    a = __ldg(s), b = __ldg(s + 1);
  }
  __device__ __forceinline__ void get(float* f) const {
    f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
  }
  __device__ __forceinline__ static void store(void* p, int64_t at, const float* f) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    d[0] = make_float4(f[0], f[1], f[2], f[3]);
    d[1] = make_float4(f[4], f[5], f[6], f[7]);
  }
};

// ------------------------------------------------------------------------------------------------ forward
// G threads side by side on a row (eight elements each), kRows rows per group in flight: bound by HBM.
constexpr int kFwdRows = 4;
template <bool BF16>
__global__ void __launch_bounds__(kThreads) k_embed_fwd(const void* __restrict__ table, const int32_t* __restrict__ tokens,
                                                        void* __restrict__ out, float scale, int64_t T, int D, int V, int G) {
  const int groups = kThreads / G, pieces = D / 8;
  const int64_t row0 = (int64_t(blockIdx.x) * groups + threadIdx.x / G) * kFwdRows;
  int32_t tok[kFwdRows];
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) tok[u] = row0 + u < T ? __ldg(tokens + row0 + u) : -1;
  for (int pc = threadIdx.x % G; pc < pieces; pc += G) {
    Eight<BF16> e[kFwdRows];
#pragma unroll
    for (int u = 0; u < kFwdRows; ++u)
      if (uint32_t(tok[u]) < uint32_t(V)) e[u].load(table, int64_t(tok[u]) * D + pc * 8);
#pragma unroll
    for (int u = 0; u < kFwdRows; ++u) {
      if (row0 + u >= T) break;
      float f[8] = {};
      if (uint32_t(tok[u]) < uint32_t(V)) {
        e[u].get(f);
#pragma unroll
        for (int k = 0; k < 8; ++k) f[k] *= scale;
      }
      Eight<BF16>::store(out, (row0 + u) * D + pc * 8, f);
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
// One cluster of up to eight CTAs sorts the positions of a section by token: a least-significant-digit radix sort, nine
// bits a pass, whose items never leave shared memory between passes (a pass scatters them into the other CTAs' shared
// memory). CTA r holds the items [r * per, (r + 1) * per). Within a pass a warp ranks its items of equal digit by
// match.any, 32 consecutive items at a time, which keeps the sort stable. The remaining CTAs of the grid have nothing to
// sort; they zero the gradient rows of absent tokens when the call overwrites (the larger part of the writes when the
// vocabulary is larger than the section), so the sort costs no time of its own there.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kMaxCluster = 8, kMaxPerThread = 16;
constexpr int64_t kSection = int64_t(kMaxCluster) * kSortThreads * kMaxPerThread;   // 131072 tokens
constexpr int kZeroSlab = 65536;   // vocabulary rows whose presence a zeroing CTA marks at a time (8 KiB of bits)

struct SortParams {
  const int32_t* tokens;
  int n, V, D, per, passes;
  int32_t* keys;        // [n] sorted tokens (V for one outside [0, V))
  int32_t* pos;         // [n] their positions
  int32_t* chains;      // word 0: how many long runs the reduction has listed (zeroed here)
  float* dtable;        // rows to zero, or nullptr
  int cluster;          // CTAs that sort
};

__device__ __forceinline__ int key_of(const SortParams& p, int t) {
  const int32_t k = __ldg(p.tokens + t);
  return uint32_t(k) < uint32_t(p.V) ? k : p.V;
}
__device__ __forceinline__ int ld_cluster(uint32_t addr) {
  int v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, int v) {
  asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

inline __host__ __device__ uint32_t sort_smem_bytes(int per) {
  return uint32_t(per) * 8u + kSortWarps * kDigits * 2u + 3u * kDigits * 4u + 128u;
}

__device__ void zero_absent_rows(const SortParams& p, uint32_t* bits) {
  const int z = int(blockIdx.x) - p.cluster, zs = int(gridDim.x) - p.cluster;
  const int v_begin = int(int64_t(p.V) * z / zs), v_end = int(int64_t(p.V) * (z + 1) / zs);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int v0 = v_begin; v0 < v_end; v0 += kZeroSlab) {
    const int rows = min(kZeroSlab, v_end - v0);
    __syncthreads();
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += kSortThreads) bits[i] = 0u;
    __syncthreads();
#pragma unroll 8
    for (int t = threadIdx.x; t < p.n; t += kSortThreads) {
      const uint32_t at = uint32_t(__ldg(p.tokens + t) - v0);
      if (at < uint32_t(rows)) atomicOr(&bits[at >> 5], 1u << (at & 31));
    }
    __syncthreads();
    for (int r = warp; r < rows; r += kSortWarps) {
      if ((bits[r >> 5] >> (r & 31)) & 1u) continue;
      float4* row = reinterpret_cast<float4*>(p.dtable + int64_t(v0 + r) * p.D);
      for (int c = lane; c < p.D / 4; c += 32) row[c] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
  }
}

template <int R>   // items per thread
__global__ void __launch_bounds__(kSortThreads, 1) k_embed_sort(const SortParams p) {
  extern __shared__ __align__(16) uint8_t sort_smem[];
  if (int(blockIdx.x) >= p.cluster) {   // whole clusters: none of their CTAs sorts
    zero_absent_rows(p, reinterpret_cast<uint32_t*>(sort_smem));
    return;
  }
  using namespace nm::ptx;
  int32_t* buf = reinterpret_cast<int32_t*>(sort_smem);                        // [2][per] positions
  uint16_t* whist = reinterpret_cast<uint16_t*>(buf + 2 * p.per);              // [warps][digits]
  int32_t* counts = reinterpret_cast<int32_t*>(whist + kSortWarps * kDigits);  // [2][digits], one half per pass parity
  int32_t* start = counts + 2 * kDigits;                                       // [digits]
  __shared__ int warp_sum_s[kSortWarps];
  const int rank = int(blockIdx.x), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int base = rank * p.per;
  const int log_per = 31 - __clz(p.per);
  if (rank == 0 && threadIdx.x == 0) p.chains[0] = 0;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int shift = pass * kDigitBits;
    const int32_t* in = buf + (pass & 1) * p.per;
    uint32_t* wh = reinterpret_cast<uint32_t*>(whist);
    for (int i = threadIdx.x; i < kSortWarps * kDigits / 2; i += kSortThreads) wh[i] = 0u;
    __syncthreads();
    uint16_t* mine = whist + warp * kDigits;
    int item[R], digit[R], rk[R];
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int at = warp * (32 * R) + j * 32 + lane;
      const bool on = base + at < p.n;
      item[j] = !on ? -1 : pass == 0 ? base + at : in[at];
    }
#pragma unroll
    for (int j = 0; j < R; ++j) digit[j] = item[j] >= 0 ? (key_of(p, item[j]) >> shift) & (kDigits - 1) : -1;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const uint32_t same = __match_any_sync(0xffffffffu, digit[j]);
      rk[j] = 0;
      if (digit[j] >= 0) {
        rk[j] = mine[digit[j]] + __popc(same & ((1u << lane) - 1u));
      }
      __syncwarp();
      if (digit[j] >= 0 && lane == __ffs(same) - 1) mine[digit[j]] = uint16_t(mine[digit[j]] + __popc(same));
      __syncwarp();
    }
    __syncthreads();
    // exclusive offsets of the warps within a digit, and this CTA's count of the digit
    int32_t* cnt = counts + (pass & 1) * kDigits;
    if (threadIdx.x < kDigits) {
      int run = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = whist[w * kDigits + threadIdx.x];
        whist[w * kDigits + threadIdx.x] = uint16_t(run);
        run += c;
      }
      cnt[threadIdx.x] = run;
    }
    cluster_sync_all();
    // where this CTA's items of a digit start: all smaller digits everywhere, then this digit in the CTAs before
    int total = 0, before = 0;
    if (threadIdx.x < kDigits) {
      const uint32_t a = smem_u32(cnt + threadIdx.x);
      for (int r = 0; r < p.cluster; ++r) {
        const int c = ld_cluster(mapa_shared(a, uint32_t(r)));
        total += c;
        if (r < rank) before += c;
      }
    }
    int incl = total;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += up;
    }
    if (lane == 31) warp_sum_s[warp] = incl;
    __syncthreads();
    if (threadIdx.x < kDigits) {
      int lower = 0;
      for (int w = 0; w < warp; ++w) lower += warp_sum_s[w];
      start[threadIdx.x] = lower + incl - total + before;
    }
    __syncthreads();
    const bool last = pass + 1 == p.passes;
    const uint32_t out = smem_u32(buf + ((pass + 1) & 1) * p.per);
#pragma unroll
    for (int j = 0; j < R; ++j) {
      if (item[j] < 0) continue;
      const int dest = start[digit[j]] + mine[digit[j]] + rk[j];
      if (last) {
        p.pos[dest] = item[j];
        p.keys[dest] = key_of(p, item[j]);
      } else {
        st_cluster(mapa_shared(out + 4u * uint32_t(dest & (p.per - 1)), uint32_t(dest >> log_per)), item[j]);
      }
    }
    // the scattered items have landed; also: no CTA leaves while another may still read its counts
    cluster_sync_all();
  }
}

// ------------------------------------------------------------------------------------------------ reduction
// The sorted positions are cut into windows of kWin; G threads (eight columns each) sum the rows of a window run by run.
// A run that crosses a window's edge is finished by the window it began in, unless it extends at least kHalf to both
// sides of the edge: then it is cut there, and each piece's sum goes to a row of its own in the workspace (slot 0 of a
// window: a piece that continues a run; slot 1: a piece that begins one), to be joined afterwards in order. So short
// runs are never cut, no window has more than 2.5 kWin rows to read, and a cut costs 8 bytes of f32 traffic per column
// for at least kWin / 2 rows read.
constexpr int kWin = 32, kHalf = kWin / 2, kSpan = 3 * kWin;
constexpr int kNoKey = INT_MAX;

struct ReduceParams {
  const void* dy;
  const int32_t* keys; const int32_t* pos;
  int32_t* chains;      // [0] count, then the windows in which a cut run begins
  float* part;          // [windows][2][D]
  float* dtable;
  float scale;
  int n, V, D, G, windows, accumulate;
};

// Is the run that holds sorted index b cut at b? `key(i)` reads the sorted keys (kNoKey outside).
template <class Key>
__device__ __forceinline__ bool is_cut(const Key& key, int b, int V) {
  const int k = key(b);
  return b > 0 && k < V && key(b - 1) == k && key(b - kHalf) == k && key(b + kHalf - 1) == k;
}
// First index the window at b owns: b itself at the start of a run or at a cut, else the end of the run that b lies in
// (the window before finishes it) or the next edge when the run is cut there. Whole warps call it.
template <class Key>
__device__ __forceinline__ int first_owned(const Key& key, int b, int V, int lane) {
  const int k = key(b);
  if (b == 0 || k >= V || key(b - 1) != k || is_cut(key, b, V)) return b;
  for (int o = 0; o < kWin + kHalf; o += 32) {
    const uint32_t other = __ballot_sync(0xffffffffu, key(b + o + lane) != k);
    if (other) {
      const int e = b + o + __ffs(other) - 1;
      return (e > b + kWin && is_cut(key, b + kWin, V)) ? b + kWin : e;
    }
  }
  return b + kWin;   // the run extends further: it is cut at the next edge
}

template <bool BF16, int U>
__global__ void __launch_bounds__(kThreads) k_embed_reduce(const ReduceParams p) {
  __shared__ int32_t skey[(kThreads / 32) * kSpan];
  __shared__ int32_t spos[(kThreads / 32) * kSpan];
  const int groups = kThreads / p.G, g = threadIdx.x / p.G, tg = threadIdx.x % p.G, lane = threadIdx.x & 31;
  const int win = int(blockIdx.x) * groups + g;
  const int b = win * kWin, origin = b - kHalf;
  int32_t* const k_s = skey + g * kSpan;
  int32_t* const p_s = spos + g * kSpan;
  for (int i = tg; i < kSpan; i += p.G) {
    const int at = origin + i;
    const bool on = at >= 0 && at < p.n;
    k_s[i] = on ? __ldg(p.keys + at) : kNoKey;
    p_s[i] = on ? __ldg(p.pos + at) : 0;
  }
  __syncthreads();
  if (win >= p.windows) return;
  // an index at or beyond the span is never reached by a run that is not cut before; it reads as "another key"
  auto key = [&](int i) {
    const int at = i - origin;
    return at >= 0 && at < kSpan ? k_s[at] : kNoKey;
  };
  const int begin = first_owned(key, b, p.V, lane);
  const int end = min(p.n, first_owned(key, b + kWin, p.V, lane));
  if (begin >= end || key(begin) >= p.V) return;
  const int pc = blockIdx.y * p.G + tg;
  const bool on = pc * 8 < p.D;
  bool continues = is_cut(key, b, p.V) && begin == b;       // the first piece continues a run of the window before
  const bool cut_end = is_cut(key, end, p.V);               // the last piece goes on in the next window
  if (cut_end && tg == 0 && blockIdx.y == 0 && !(continues && key(begin) == key(end - 1)))
    p.chains[1 + atomicAdd(p.chains, 1)] = win;
  float acc[8] = {};
  for (int i0 = begin; i0 < end; i0 += U) {
    Eight<BF16> e[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (on && i0 + u < end && key(i0 + u) < p.V) e[u].load(p.dy, int64_t(p_s[i0 + u - origin]) * p.D + pc * 8);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u;
      if (i >= end) break;
      const int k = key(i);
      if (k >= p.V) return;                                  // ids outside the vocabulary sort last
      float f[8];
      if (on) e[u].get(f);
#pragma unroll
      for (int q = 0; q < 8; ++q) acc[q] += f[q];
      const bool piece_end = i + 1 >= end || key(i + 1) != k;
      if (piece_end) {
        if (on) {
          const bool goes_on = i + 1 >= end && cut_end;
          if (continues || goes_on) {
            Eight<false>::store(p.part, (int64_t(win) * 2 + (continues ? 0 : 1)) * p.D + pc * 8, acc);
          } else {
            const int64_t at = int64_t(k) * p.D + pc * 8;
            float o[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) o[q] = p.scale * acc[q];
            if (p.accumulate) {
              Eight<false> old;
              const float4* s = reinterpret_cast<const float4*>(p.dtable + at);
              old.a = s[0], old.b = s[1];
              float w[8];
              old.get(w);
#pragma unroll
              for (int q = 0; q < 8; ++q) o[q] += w[q];
            }
            Eight<false>::store(p.dtable, at, o);
          }
        }
        continues = false;
#pragma unroll
        for (int q = 0; q < 8; ++q) acc[q] = 0.f;
      }
    }
  }
}

// Joins the pieces of the listed cut runs: slot 1 of the window the run begins in, then slot 0 of the windows after it,
// in that order dealt to eight row lanes whose sums are added in lane order. 32 threads side by side on 128 columns.
constexpr int kJoinCols = 128, kJoinLanes = kThreads / 32;
__global__ void __launch_bounds__(kThreads) k_embed_join(const ReduceParams p) {
  __shared__ float4 red[kJoinLanes][32];
  const int count = p.chains[0];
  const int col_blocks = (p.D + kJoinCols - 1) / kJoinCols;
  const int tc = threadIdx.x & 31, rl = threadIdx.x >> 5;
  for (int64_t job = blockIdx.x; job < int64_t(count) * col_blocks; job += gridDim.x) {
    const int win = p.chains[1 + int(job / col_blocks)];
    const int col = int(job % col_blocks) * kJoinCols + tc * 4;
    const int edge = (win + 1) * kWin;
    const int k = __ldg(p.keys + edge);
    int lo = edge, hi = p.n;                       // end of the run: first index whose key is larger
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (__ldg(p.keys + mid) > k) hi = mid;
      else lo = mid + 1;
    }
    // the first cut: at this edge, or at the next one when the run has fewer than kHalf rows before this edge
    const bool here = edge >= kHalf && __ldg(p.keys + edge - kHalf) == k && lo >= edge + kHalf;
    const int second = here ? win + 1 : win + 2;   // the window that holds the second piece
    const int last = (lo - kHalf) / kWin;          // the last edge inside the run with kHalf rows of it behind the edge
    const int pieces = last - second + 2;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    if (col < p.D) {
#pragma unroll 4
      for (int i = rl; i < pieces; i += kJoinLanes) {
        const int64_t slot = i == 0 ? int64_t(win) * 2 + 1 : int64_t(second + i - 1) * 2;
        const float4 v = __ldcg(reinterpret_cast<const float4*>(p.part + slot * p.D + col));
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
    }
    red[rl][tc] = s;
    __syncthreads();
    if (rl == 0 && col < p.D) {
      for (int w = 1; w < kJoinLanes; ++w) {
        const float4 v = red[w][tc];
        s.x += v.x, s.y += v.y, s.z += v.z, s.w += v.w;
      }
      float4* o = reinterpret_cast<float4*>(p.dtable + int64_t(k) * p.D + col);
      float4 r = make_float4(p.scale * s.x, p.scale * s.y, p.scale * s.z, p.scale * s.w);
      if (p.accumulate) {
        const float4 old = *o;
        r.x += old.x, r.y += old.y, r.z += old.z, r.w += old.w;
      }
      *o = r;
    }
    __syncthreads();
  }
}

__global__ void k_zero(float4* p, int64_t n) {
  for (int64_t i = blockIdx.x * int64_t(blockDim.x) + threadIdx.x; i < n; i += int64_t(gridDim.x) * blockDim.x)
    p[i] = make_float4(0.f, 0.f, 0.f, 0.f);
}

int threads_per_row(int pieces) {
  int g = 32;
  while (g < pieces && g < kThreads) g *= 2;
  return g;
}

struct BwdRegions {
  int32_t* keys; int32_t* pos; int32_t* chains; float* part;
  uint64_t bytes;
};
BwdRegions bwd_layout(int64_t T, int D, void* base) {
  const int64_t n = std::min(T, kSection), windows = (n + kWin - 1) / kWin;
  ce::Arena arena(base);
  BwdRegions r{};
  r.keys = arena.take<int32_t>(uint64_t(n));
  r.pos = arena.take<int32_t>(uint64_t(n));
  r.chains = arena.take<int32_t>(uint64_t(windows) + 1);
  r.part = arena.take<float>(uint64_t(windows) * 2 * uint64_t(D));
  r.bytes = arena.bytes();
  return r;
}

void require_shape(int64_t T, int D, int V, const char* who) {
  const std::string w(who);
  NM_REQUIRE(T >= 0, w + ": the row count T cannot be negative");
  NM_REQUIRE(D > 0 && D % 8 == 0, w + ": D must be a positive multiple of 8 (rows are moved in 16-byte pieces)");
  NM_REQUIRE(V > 0, w + ": the vocabulary size V must be positive");
}
void require_arch(const char* who) {
  NM_REQUIRE(ce::device_arch() >= 100, std::string(who) + ": this library holds sm_100a code only");
}

template <int R>
void launch_sort(const SortParams& p, int cluster, int grid, cudaStream_t st) {
  const uint32_t smem = std::max(sort_smem_bytes(p.per), uint32_t(kZeroSlab / 8));
  NM_CUDA(cudaFuncSetAttribute(k_embed_sort<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(cluster); attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  NM_CUDA(cudaLaunchKernelEx(&cfg, k_embed_sort<R>, p));
}

}  // namespace

void embed_fwd(bool bf16, const void* table, const int32_t* tokens, void* out, float scale, int64_t T, int D, int V,
               cudaStream_t st) {
  require_shape(T, D, V, "embed_fwd");
  if (T == 0) return;
  NM_REQUIRE(table && tokens && out, "embed_fwd: table, tokens and out are required");
  NM_REQUIRE(aligned16(table, out), "embed_fwd: table and out must be 16-byte aligned");
  NM_REQUIRE(reinterpret_cast<uintptr_t>(tokens) % 4 == 0, "embed_fwd: tokens must be 4-byte aligned");
  require_arch("embed_fwd");
  const int G = threads_per_row(D / 8);
  const int64_t per_cta = int64_t(kThreads / G) * kFwdRows, grid = (T + per_cta - 1) / per_cta;
  NM_REQUIRE(grid <= INT_MAX, "embed_fwd: too many rows for one launch");
  auto kern = bf16 ? k_embed_fwd<true> : k_embed_fwd<false>;
  kern<<<unsigned(grid), kThreads, 0, st>>>(table, tokens, out, scale, T, D, V, G);
  NM_CUDA(cudaGetLastError());
}

uint64_t embed_bwd_workspace_bytes(int64_t T, int D, int V) {
  require_shape(T, D, V, "embed_bwd");
  return T == 0 ? kArenaAlign : bwd_layout(T, D, nullptr).bytes;
}

void embed_bwd(bool bf16, const void* dy, const int32_t* tokens, float* dtable, float scale, bool accumulate, int64_t T,
               int D, int V, void* ws, uint64_t ws_bytes, cudaStream_t st) {
  require_shape(T, D, V, "embed_bwd");
  if (T == 0 && accumulate) return;
  NM_REQUIRE(dtable && aligned16(dtable), "embed_bwd: a 16-byte aligned dtable is required");
  if (T == 0) {   // the gradient of nothing
    require_arch("embed_bwd");
    const int64_t n = int64_t(V) * D / 4;
    k_zero<<<unsigned(std::min<int64_t>((n + 255) / 256, int64_t(ce::sm_count()) * 16)), 256, 0, st>>>(
        reinterpret_cast<float4*>(dtable), n);
    NM_CUDA(cudaGetLastError());
    return;
  }
  NM_REQUIRE(dy && tokens, "embed_bwd: dy and tokens are required");
  NM_REQUIRE(aligned16(dy), "embed_bwd: dy must be 16-byte aligned");
  NM_REQUIRE(reinterpret_cast<uintptr_t>(tokens) % 4 == 0, "embed_bwd: tokens must be 4-byte aligned");
  NM_REQUIRE(ws != nullptr && reinterpret_cast<uintptr_t>(ws) % kArenaAlign == 0,
             "embed_bwd: a 256-byte aligned workspace is required");
  NM_REQUIRE(ws_bytes >= bwd_layout(T, D, nullptr).bytes, "embed_bwd: the workspace is smaller than "
                                                          "nm_embed_bwd_workspace_bytes()");
  require_arch("embed_bwd");
  const BwdRegions r = bwd_layout(T, D, ws);
  int bits = 1;
  while ((int64_t(1) << bits) <= V) ++bits;   // keys are 0 .. V
  // A call longer than a section runs section by section, the later ones adding to the rows of the earlier ones.
  for (int64_t t0 = 0; t0 < T; t0 += kSection) {
    const int n = int(std::min(kSection, T - t0));
    const bool add = accumulate || t0 > 0;
    int per = kSortThreads;
    while (int64_t(per) * kMaxCluster < n) per *= 2;
    int cluster = 1;
    while (cluster * per < n) cluster *= 2;
    SortParams sp{tokens + t0, n, V, D, per, (bits + kDigitBits - 1) / kDigitBits, r.keys, r.pos, r.chains,
                  add ? nullptr : dtable, cluster};
    const int grid = add ? cluster : cluster * std::max(2, ce::sm_count() / cluster);
    switch (per / kSortThreads) {
      case 1: launch_sort<1>(sp, cluster, grid, st); break;
      case 2: launch_sort<2>(sp, cluster, grid, st); break;
      case 4: launch_sort<4>(sp, cluster, grid, st); break;
      case 8: launch_sort<8>(sp, cluster, grid, st); break;
      default: launch_sort<16>(sp, cluster, grid, st); break;
    }
    ReduceParams rp{};
    rp.dy = static_cast<const uint8_t*>(dy) + t0 * D * (bf16 ? 2 : 4);
    rp.keys = r.keys, rp.pos = r.pos, rp.chains = r.chains, rp.part = r.part, rp.dtable = dtable, rp.scale = scale;
    rp.n = n, rp.V = V, rp.D = D, rp.G = threads_per_row(D / 8), rp.windows = (n + kWin - 1) / kWin;
    rp.accumulate = add;
    const int groups = kThreads / rp.G;
    const dim3 rg(unsigned((rp.windows + groups - 1) / groups), unsigned((D / 8 + rp.G - 1) / rp.G));
    if (bf16) k_embed_reduce<true, 8><<<rg, kThreads, 0, st>>>(rp);
    else k_embed_reduce<false, 4><<<rg, kThreads, 0, st>>>(rp);
    NM_CUDA(cudaGetLastError());
    const int64_t jobs = int64_t(rp.windows) * ((D + kJoinCols - 1) / kJoinCols);
    k_embed_join<<<unsigned(std::min<int64_t>(jobs, int64_t(ce::sm_count()) * 4)), kThreads, 0, st>>>(rp);
    NM_CUDA(cudaGetLastError());
  }
}

}  // namespace nm::ew

extern "C" {

int nm_embed_fwd(int dtype, const void* table, const int32_t* tokens, void* out, float scale, int64_t T, int D, int V,
                 void* stream) {
  return nm::abi::guarded([&] {
    NM_REQUIRE(dtype == 0 || dtype == 1, "nm_embed_fwd: storage 0 (f32) or 1 (bf16)");
    nm::ew::embed_fwd(dtype == 1, table, tokens, out, scale, T, D, V, static_cast<cudaStream_t>(stream));
  });
}

uint64_t nm_embed_bwd_workspace_bytes(int64_t T, int D, int V) {
  return nm::abi::guarded_value<uint64_t>(0, [&] { return nm::ew::embed_bwd_workspace_bytes(T, D, V); });
}

int nm_embed_bwd(int dtype, const void* dy, const int32_t* tokens, float* dtable, float scale, int accumulate, int64_t T,
                 int D, int V, void* workspace, uint64_t workspace_bytes, void* stream) {
  return nm::abi::guarded([&] {
    NM_REQUIRE(dtype == 0 || dtype == 1, "nm_embed_bwd: storage 0 (f32) or 1 (bf16)");
    nm::ew::embed_bwd(dtype == 1, dy, tokens, dtable, scale, accumulate != 0, T, D, V, workspace, workspace_bytes,
                      static_cast<cudaStream_t>(stream));
  });
}

}  // extern "C"
