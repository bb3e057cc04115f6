// Embedding lookup with scaling, and its gradient by sorted tokens: the other end of the vocabulary matrix (a tied model
// adds the gradient below into the buffer that the fused CE accumulates dW in).
//   forward   y[t, :] = round(scale * E[token_t, :])             a token outside [0, V) gives a row of zeros
//   backward  dE[v, :] (+)= scale * sum_{t: token_t = v} dy[t, :]  in f32; a token outside [0, V) contributes nothing
// No sum of the backward depends on an order of atomics: tokens are sorted by a stable radix sort, a run of equal tokens is
// summed in ascending t, long runs are cut at places that depend on the sorted tokens alone, and a call that adds makes one
// addition per element, so that the same call gives the same bits. Counterpart in the reference:
// src/kernels/elementwise/embed.cu.
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
  __device__ __forceinline__ static void stream(void* p, int64_t at, const float* f) {   // not read again soon
    __stcs(reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(p) + at), pack8(f));
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
  __device__ __forceinline__ static void stream(void* p, int64_t at, const float* f) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(p) + at);
    __stcs(d, make_float4(f[0], f[1], f[2], f[3]));
    __stcs(d + 1, make_float4(f[4], f[5], f[6], f[7]));
  }
};

// Eight f32 values in one 32-byte store (sm_100): two 16-byte stores of a thread cover half of every 32-byte sector each.
__device__ __forceinline__ void store32(float* p, const float* f) {
  asm volatile("st.global.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]),
               "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7])
               : "memory");
}
// p[0 .. 8) += f without reading p back: one addition per element and launch (every row has one writer), performed at L2,
// so the result does not depend on any order. Additions at L2 flush values below 2^-126 to zero.
__device__ __forceinline__ void add32(float* p, const float* f) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p), "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]) : "memory");
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + 4), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]) : "memory");
}
using nm::ptx::after_previous;
using nm::ptx::release_next;

// ------------------------------------------------------------------------------------------------ forward
// G threads side by side on a row (eight elements each); a row group takes `batches` times kFwdRows consecutive rows, the
// loads of a batch in flight while the one before it is stored. Bound by HBM: the output is written once, past the L2 (the
// frequent rows of the table are read from there again and again). 131072 x 2048 bf16, ids falling as 1 / rank (32 thousand
// distinct rows): 117 us, 5.7 TB/s; batches of three rows 118 us, of four 122 us, one batch of four rows per group 128 us.
constexpr int kFwdRows = 2, kFwdMaxBatches = 8;
template <bool BF16>
__global__ void __launch_bounds__(kThreads, BF16 ? 6 : 4) k_embed_fwd(const void* __restrict__ table, const int32_t* __restrict__ tokens,
                                                        void* __restrict__ out, float scale, int64_t T, int D, int V, int G,
                                                        int batches) {
  __shared__ int32_t tok_s[kThreads / 32 * kFwdRows * kFwdMaxBatches];
  const int groups = kThreads / G, pieces = D / 8, g = threadIdx.x / G, tg = threadIdx.x % G;
  const int rows = kFwdRows * batches;                       // per group
  const int64_t row0 = (int64_t(blockIdx.x) * groups + g) * rows;
  int32_t* const tok = tok_s + g * rows;
  for (int u = tg; u < rows; u += G) {
    const int32_t t = row0 + u < T ? __ldg(tokens + row0 + u) : -1;
    tok[u] = uint32_t(t) < uint32_t(V) ? t : -1;
  }
  __syncthreads();
  for (int pc = tg; pc < pieces; pc += G) {
    Eight<BF16> e[kFwdRows], next[kFwdRows];
    auto fetch = [&](Eight<BF16>(&to)[kFwdRows], int at) {
#pragma unroll
      for (int u = 0; u < kFwdRows; ++u) {
        const int32_t t = tok[at + u];
        if (t >= 0) to[u].load(table, int64_t(t) * D + pc * 8);
      }
    };
    fetch(e, 0);
    for (int at = 0; at < rows; at += kFwdRows) {
      if (at + kFwdRows < rows) fetch(next, at + kFwdRows);
#pragma unroll
      for (int u = 0; u < kFwdRows; ++u) {
        if (row0 + at + u >= T) break;
        float f[8] = {};
        if (tok[at + u] >= 0) {
          e[u].get(f);
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] *= scale;
        }
        Eight<BF16>::stream(out, (row0 + at + u) * D + pc * 8, f);
      }
#pragma unroll
      for (int u = 0; u < kFwdRows; ++u) e[u] = next[u];
    }
  }
}

// ------------------------------------------------------------------------------------------------ sort
// One cluster of up to sixteen CTAs sorts the positions of a section by token: a least-significant-digit radix sort, nine
// bits a pass, whose items never leave shared memory between passes (a pass scatters them into the other CTAs' shared
// memory). CTA r holds the items [r * per, (r + 1) * per). Within a pass a warp ranks its items of equal digit, 32
// consecutive items at a time, which keeps the sort stable; equal lanes are found by nine votes. Bound by latency (scans, two
// cluster barriers a pass, random 4-byte accesses): 131072 tokens of 17 bits 36 us on 16 CTAs, with match.any 43 us, that on 8
// CTAs 75 us; beside the zeroing it costs nothing.
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32, kDigitBits = 9, kDigits = 1 << kDigitBits;
constexpr int kMaxCluster = 16, kMaxPerThread = 8, kPosBits = 17;
constexpr int64_t kSection = int64_t(kMaxCluster) * kSortThreads * kMaxPerThread;   // 131072 tokens
static_assert(kSection <= (int64_t(1) << kPosBits), "a position and its rank within a warp share one register");

struct SortParams {
  const int32_t* tokens;
  int n, V, D, per, passes;
  int32_t* keys;        // [n] sorted tokens (V for one outside [0, V))
  int32_t* pos;         // [n] their positions
  int32_t* chains;      // word 0: how many long runs the reduction has listed (zeroed here)
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

// The lanes that hold the same digit (kDigits and beyond mean nothing; -1 only matches -1): one vote per bit.
__device__ __forceinline__ uint32_t lanes_with(int digit) {
  uint32_t same = __ballot_sync(0xffffffffu, digit >= 0);
  if (digit < 0) same = ~same;
#pragma unroll
  for (int b = 0; b < kDigitBits; ++b) {
    const bool set = (digit >> b) & 1;
    const uint32_t votes = __ballot_sync(0xffffffffu, set);
    same &= set ? votes : ~votes;
  }
  return same;
}

inline __host__ __device__ uint32_t sort_smem_bytes(int per) {
  return uint32_t(per) * 8u + kSortWarps * kDigits * 2u + 3u * kDigits * 4u + 128u;
}

// A short section (at most kRankMax tokens) needs no radix passes: the place of a token in the sorted order is the number
// of tokens that are smaller, or equal and earlier (2125 tokens: a few us of latency against 12 us for the radix sort).
// 32 positions per CTA, one per lane; warp w counts over the w-th eighth
// of the tokens, which lie in shared memory.
constexpr int kRankMax = 4096, kRankWarps = kThreads / 32;
__global__ void __launch_bounds__(kThreads) k_embed_rank(const SortParams p) {
  __shared__ __align__(16) int32_t key[kRankMax];
  __shared__ int partial[kRankWarps][32];
  release_next();
  if (blockIdx.x == 0 && threadIdx.x == 0) p.chains[0] = 0;
  const int n4 = (p.n + 3) / 4;
  for (int t = threadIdx.x; t < 4 * n4; t += kThreads) key[t] = t < p.n ? key_of(p, t) : INT_MAX;
  __syncthreads();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t = int(blockIdx.x) * 32 + lane;
  const int k = t < p.n ? key[t] : 0;
  int count = 0;
#pragma unroll 4
  for (int q = n4 * warp / kRankWarps; q < n4 * (warp + 1) / kRankWarps; ++q) {
    const int4 v = reinterpret_cast<const int4*>(key)[q];
    const int j = 4 * q;
    count += (v.x < k || (v.x == k && j < t)) + (v.y < k || (v.y == k && j + 1 < t)) +
             (v.z < k || (v.z == k && j + 2 < t)) + (v.w < k || (v.w == k && j + 3 < t));
  }
  partial[warp][lane] = count;
  __syncthreads();
  if (warp == 0 && t < p.n) {
    int rank = 0;
#pragma unroll
    for (int w = 0; w < kRankWarps; ++w) rank += partial[w][lane];
    p.keys[rank] = k;
    p.pos[rank] = t;
  }
}

// Zeroes the rows that no token of the section names (the larger part of the writes of an overwriting call whose
// vocabulary is larger than the section). It needs the tokens, not their order, so it runs beside the sort: it does not wait
// for the launch before it until it has done its work. The vocabulary is dealt to the CTAs (a power of two of them) in
// blocks of eight rows, because frequent ids lie together; a CTA marks the tokens of its share (10 us for 131072 tokens), then
// writes. Bound by HBM: 786 MB in 137 us; dealt in contiguous ranges 148 us.
constexpr int kZeroThreads = 1024, kZeroSlab = 65536;   // rows whose presence a CTA marks at a time (8 KiB of bits)
struct ZeroParams {
  const int32_t* tokens;
  float* dtable;
  int n, V, D, log_ctas, wide;
};
__global__ void __launch_bounds__(kZeroThreads) k_embed_zero_absent(const ZeroParams p) {
  __shared__ uint32_t bits[kZeroSlab / 32];
  release_next();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t me = blockIdx.x, mask = gridDim.x - 1u;
  // id v: block v >> 3 belongs to CTA (v >> 3) & mask, where it is row ((v >> 3) >> log_ctas) * 8 + (v & 7)
  const int64_t slab_ids = int64_t(kZeroSlab) << p.log_ctas;
  for (int64_t v0 = 0; v0 < p.V; v0 += slab_ids) {
    const int ids = int(min(slab_ids, int64_t(p.V) - v0));
    const int rows = (((ids + 7) >> 3) + int(mask) >> p.log_ctas) * 8;
    __syncthreads();
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += kZeroThreads) bits[i] = 0u;
    __syncthreads();
#pragma unroll 16
    for (int t = threadIdx.x; t < p.n; t += kZeroThreads) {
      const int64_t v = int64_t(__ldg(p.tokens + t)) - v0;
      if (v < 0 || v >= ids || ((uint32_t(v) >> 3) & mask) != me) continue;
      const uint32_t at = (uint32_t(v) >> (3 + p.log_ctas)) * 8u + (uint32_t(v) & 7u), bit = 1u << (at & 31);
      if (!(bits[at >> 5] & bit)) atomicOr(&bits[at >> 5], bit);   // a frequent token finds its bit set already
    }
    __syncthreads();
    for (int r = warp; r < rows; r += kZeroThreads / 32) {
      const int64_t v = v0 + ((int64_t(r >> 3) << p.log_ctas) + me) * 8 + (r & 7);
      if (v >= p.V || ((bits[r >> 5] >> (r & 31)) & 1u)) continue;
      float* row = p.dtable + v * p.D;
      const float none[8] = {};
      if (p.wide) {
        for (int c = lane * 8; c < p.D; c += 256) store32(row + c, none);
      } else {
        for (int c = lane * 8; c < p.D; c += 256) Eight<false>::store(row, c, none);
      }
    }
  }
  after_previous();
}

template <int R>   // items per thread
__global__ void __launch_bounds__(kSortThreads, 1) k_embed_sort(const SortParams p) {
  extern __shared__ __align__(16) uint8_t sort_smem[];
  release_next();
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
    int item[R], key[R];   // item: position, later with the rank among the warp's items of equal digit above it
    uint32_t on = 0;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int at = warp * (32 * R) + j * 32 + lane;
      if (base + at < p.n) on |= 1u << j;
      item[j] = !((on >> j) & 1u) ? 0 : pass == 0 ? base + at : in[at];
    }
#pragma unroll
    for (int j = 0; j < R; ++j) key[j] = ((on >> j) & 1u) ? key_of(p, item[j]) : -1;
#pragma unroll
    for (int j = 0; j < R; ++j) {
      const int digit = ((on >> j) & 1u) ? (key[j] >> shift) & (kDigits - 1) : -1;
      const uint32_t same = lanes_with(digit);
      if (digit >= 0) item[j] |= (mine[digit] + __popc(same & ((1u << lane) - 1u))) << kPosBits;
      __syncwarp();
      if (digit >= 0 && lane == __ffs(same) - 1) mine[digit] = uint16_t(mine[digit] + __popc(same));
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
      int c[kMaxCluster];
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) c[r] = r < p.cluster ? ld_cluster(mapa_shared(a, uint32_t(r))) : 0;
#pragma unroll
      for (int r = 0; r < kMaxCluster; ++r) {
        total += c[r];
        if (r < rank) before += c[r];
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
      if (!((on >> j) & 1u)) continue;
      const int digit = (key[j] >> shift) & (kDigits - 1), at = item[j] & ((1 << kPosBits) - 1);
      const int dest = start[digit] + mine[digit] + (item[j] >> kPosBits);
      if (last) {
        p.pos[dest] = at;
        p.keys[dest] = key[j];
      } else {
        st_cluster(mapa_shared(out + 4u * uint32_t(dest & (p.per - 1)), uint32_t(dest >> log_per)), at);
      }
    }
    // the scattered items have landed; also: no CTA leaves while another may still read its counts
    cluster_sync_all();
  }
}

// ------------------------------------------------------------------------------------------------ reduction
// The sorted positions are cut into windows of `win`; G threads (eight columns each) sum the rows of a window run by run.
// A run that crosses a window's edge is finished by the window it began in, unless it extends at least win / 2 to both
// sides of the edge: then it is cut there, and each piece's sum goes to a row of its own in the workspace (slot 0 of a
// window: a piece that continues a run; slot 1: a piece that begins one), to be joined afterwards in order. So short
// runs are never cut, no window has more than 2.5 win rows to read, and a cut costs 8 bytes of f32 traffic per column
// for at least win / 2 rows read.
constexpr int kNoKey = INT_MAX;
// Rows per window: many windows keep every SM busy and no CTA waits long, few of them cut fewer runs (8 bytes per column and
// cut). Whole calls of 16 / 32 / 64 rows in us, ids falling as 1 / rank, replayed from a graph:
//   2000 x 512 bf16, added 17 / 21 / 30     8000 x 64 bf16, added 23 / 26 / 34       16384 x 256 bf16 43 / 50 / 56
//   4000 x 512 bf16, added 26 / 32 / 33     16000 x 64 bf16, added 26 / 28 / 36      16000 x 768 f32, added 50 / 44 / 47
//   32768 x 2048 bf16 218 / 217 / 222       48000 x 512 bf16, added 52 / 49 / 58     65536 x 2048 bf16 257 / 244 / 246
//   64000 x 768 f32, added 116 / 120 / 142  98304 x 1024 f32 234 / 230 / 237         98304 x 2048 bf16 294 / 273 / 271
//   131072 x 512 bf16 120 / 112 / 116       131072 x 1024 f32 276 / 268 / 281        131072 x 2048 bf16 330 / 301 / 293
// and of a single id, which is cut at every edge: 16384 x 512 36 / 29 / 28, 131072 x 2048 383 / 239 / 175. So 16 rows for short
// sections, as long as the cut pieces' rows (8 D n / 16 bytes of workspace) stay under 2.5 MiB, and 64 for a nearly full one.
constexpr int64_t kMost16 = 16384, kMost16Elements = int64_t(5) << 20, kMost32 = 98304;
inline int64_t most16(int D) { return std::min(kMost16, kMost16Elements / D); }   // tokens in windows of 16 rows
inline int window_for(int64_t n, int D) { return n > kMost32 ? 64 : n > most16(D) ? 32 : 16; }
inline int64_t windows_of(int64_t n, int D) { return (n + window_for(n, D) - 1) / window_for(n, D); }
// The most windows of any section of up to n tokens: a workspace planned for the longest call serves every shorter one.
inline int64_t windows_up_to(int64_t n, int D) {
  int64_t most = windows_of(n, D);
  if (n > most16(D)) most = std::max(most, windows_of(most16(D), D));
  if (n > kMost32) most = std::max(most, windows_of(kMost32, D));
  return most;
}

struct ReduceParams {
  const void* dy;
  const int32_t* keys; const int32_t* pos;
  int32_t* chains;      // [0] count, then the windows in which a cut run begins
  float* part;          // [windows][2][D]
  float* dtable;
  float scale;
  int n, V, D, G, win, windows, accumulate, wide;   // wide: rows of dtable and part are 32-byte aligned
};

// Is the run that holds sorted index b cut at b? `key(i)` reads the sorted keys (kNoKey outside).
template <class Key>
__device__ __forceinline__ bool is_cut(const Key& key, int b, int win, int V) {
  const int k = key(b);
  return b > 0 && k < V && key(b - 1) == k && key(b - win / 2) == k && key(b + win / 2 - 1) == k;
}
// First index the window at b owns: b itself at the start of a run or at a cut, else the end of the run that b lies in
// (the window before finishes it) or the next edge when the run is cut there. Whole warps call it.
template <class Key>
__device__ __forceinline__ int first_owned(const Key& key, int b, int win, int V, int lane) {
  const int k = key(b);
  if (b == 0 || k >= V || key(b - 1) != k || is_cut(key, b, win, V)) return b;
  for (int o = 0; o < win + win / 2; o += 32) {
    const uint32_t other = __ballot_sync(0xffffffffu, key(b + o + lane) != k);
    if (other) {
      const int e = b + o + __ffs(other) - 1;
      return (e > b + win && is_cut(key, b + win, win, V)) ? b + win : e;
    }
  }
  return b + win;   // the run extends further: it is cut at the next edge
}

// A thread's pieces of the rows to come travel through its own slots of a ring in shared memory (cp.async, no barrier:
// nobody else reads them), 64 KiB in flight per CTA: what a window waits for is a few round trips, and registers do not
// limit how many rows are on their way. Bound by HBM: 131072 x 2048 bf16 into 32 thousand rows 128 us (795 MB, 6.2 TB/s);
// with loads into registers 175 us.
template <bool BF16>
struct Ring {
  static constexpr int kGroups = 4;                        // commit groups in flight
  static constexpr int kRows = BF16 ? 4 : 2;               // rows per group
  static constexpr int kPieces = BF16 ? 1 : 2;             // 16-byte pieces per row and thread
  static constexpr int kBytes = kGroups * kRows * kPieces * kThreads * 16;
};
// 16 bytes, or zeros without a read when `bytes` is 0
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Shared memory of the reduction: the ring, then per row group the keys and the rows of its window (in 16-byte units from
// dy), padded to whole ring groups.
inline __host__ __device__ int span_of(int win) { return 3 * win; }
template <bool BF16>
int reduce_smem_bytes(int groups, int win) { return Ring<BF16>::kBytes + groups * span_of(win) * 3 * 4; }

template <bool BF16>
__global__ void __launch_bounds__(kThreads, 3) k_embed_reduce(const ReduceParams p) {
  using R = Ring<BF16>;
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ int ends[kThreads / 32];
  release_next();
  const int groups = kThreads / p.G, g = threadIdx.x / p.G, tg = threadIdx.x % p.G, lane = threadIdx.x & 31;
  const int win = int(blockIdx.x) * groups + g, W = p.win, span = span_of(W);
  const int b = win * W, origin = b - W / 2;
  int32_t* const k_s = reinterpret_cast<int32_t*>(ring + R::kBytes) + g * span * 3;   // keys of the span
  int32_t* const m_s = k_s + span;      // per row: the key where a piece ends, -1 elsewhere
  uint32_t* const r_s = reinterpret_cast<uint32_t*>(m_s + span);
  after_previous();
  for (int i = tg; i < span; i += p.G) {
    const int at = origin + i;
    k_s[i] = at >= 0 && at < p.n ? __ldcg(p.keys + at) : kNoKey;
  }
  __syncthreads();
  // an index at or beyond the span is never reached by a run that is not cut before; it reads as "another key"
  auto key = [&](int i) {
    const int at = i - origin;
    return at >= 0 && at < span ? k_s[at] : kNoKey;
  };
  int begin = 0, end = 0;
  if (win < p.windows) {
    begin = first_owned(key, b, W, p.V, lane);
    end = min(p.n, first_owned(key, b + W, W, p.V, lane));
  }
  const bool work = begin < end && key(begin) < p.V;
  const bool continues = work && begin == b && is_cut(key, b, W, p.V);   // the first piece continues a run
  const bool cut_end = work && is_cut(key, end, W, p.V);                 // the last piece goes on in the next window
  if (cut_end && tg == 0 && blockIdx.y == 0 && !(continues && key(begin) == key(end - 1)))
    p.chains[1 + atomicAdd(p.chains, 1)] = win;
  const int first_key = work ? key(begin) : kNoKey, last_key = work ? key(end - 1) : kNoKey;
  if (tg == 0) ends[g] = end;
  __syncthreads();
  if (work) {
    for (int i = begin + tg; i < begin + span; i += p.G) {
      const int k = i < end ? key(i) : kNoKey;
      if (i < end && k >= p.V && key(i - 1) < p.V) ends[g] = i;   // ids outside the vocabulary sort last
      const int next = i + 1 < end ? key(i + 1) : kNoKey;
      m_s[i - begin] = k < p.V && next != k ? k : -1;
      r_s[i - begin] = k < p.V ? uint32_t(__ldcg(p.pos + i)) * uint32_t(p.D / 8 * R::kPieces) : 0u;
    }
  }
  __syncthreads();
  const int col = (blockIdx.y * p.G + tg) * 8;
  if (!work || col >= p.D) return;
  const int rows = ends[g] - begin;
  const uint32_t slots = nm::ptx::smem_u32(ring) + threadIdx.x * 16u;
  auto slot = [&](int group, int u, int piece) {
    return slots + uint32_t(((group * R::kRows + u) * R::kPieces + piece) * kThreads) * 16u;
  };
  const uint8_t* const mine = static_cast<const uint8_t*>(p.dy) + int64_t(col) * (BF16 ? 2 : 4);
  auto fetch = [&](int group, int i0) {       // rows past the end become zeros
#pragma unroll
    for (int u = 0; u < R::kRows; ++u) {
      const bool in = i0 + u < rows;
      const uint8_t* src = mine + (in ? uint64_t(r_s[i0 + u]) * 16u : 0u);
#pragma unroll
      for (int h = 0; h < R::kPieces; ++h) cp_async16(slot(group, u, h), src + 16 * h, in ? 16u : 0u);
    }
    cp_async_commit();
  };
  F2 acc[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) acc[q] = f2(0.f, 0.f);
  auto flush = [&](int k) {
    float* to;
    float f[8];
#pragma unroll
    for (int q = 0; q < 4; ++q) f2_get(acc[q], f[2 * q], f[2 * q + 1]), acc[q] = f2(0.f, 0.f);
    const bool head = continues && k == first_key, tail = cut_end && k == last_key;
    if (head || tail) {
      to = p.part + (int64_t(win) * 2 + (head ? 0 : 1)) * p.D + col;
    } else {
      to = p.dtable + int64_t(k) * p.D + col;
#pragma unroll
      for (int q = 0; q < 8; ++q) f[q] *= p.scale;
    }
    if (p.accumulate && !head && !tail) {
      add32(to, f);
    } else if (p.wide) {
      store32(to, f);
    } else {
      Eight<false>::store(to, 0, f);
    }
  };
#pragma unroll
  for (int g4 = 0; g4 < R::kGroups; ++g4) fetch(g4, g4 * R::kRows);
  for (int i0 = 0; i0 < rows;) {
#pragma unroll
    for (int group = 0; group < R::kGroups; ++group) {
      cp_async_wait<R::kGroups - 1>();
#pragma unroll
      for (int u = 0; u < R::kRows; ++u) {
        const int m = i0 + u < rows ? m_s[i0 + u] : -1;
        const uint4 q0 = nm::ptx::ld_shared_v4(slot(group, u, 0));
        if constexpr (BF16) {
          acc[0] = f2_add(acc[0], f2_of(q0.x)), acc[1] = f2_add(acc[1], f2_of(q0.y));
          acc[2] = f2_add(acc[2], f2_of(q0.z)), acc[3] = f2_add(acc[3], f2_of(q0.w));
        } else {
          const uint4 q1 = nm::ptx::ld_shared_v4(slot(group, u, 1));
          acc[0] = f2_add(acc[0], f2(__uint_as_float(q0.x), __uint_as_float(q0.y)));
          acc[1] = f2_add(acc[1], f2(__uint_as_float(q0.z), __uint_as_float(q0.w)));
          acc[2] = f2_add(acc[2], f2(__uint_as_float(q1.x), __uint_as_float(q1.y)));
          acc[3] = f2_add(acc[3], f2(__uint_as_float(q1.z), __uint_as_float(q1.w)));
        }
        if (m >= 0) flush(m);
      }
      fetch(group, i0 + R::kGroups * R::kRows);
      i0 += R::kRows;
    }
  }
  cp_async_wait<0>();
}

// Joins the pieces of the listed cut runs: slot 1 of the window the run begins in, then slot 0 of the windows after it, in
// that order. A job is 128 columns of one run and belongs to a warp; a run of more than kJoinAlone pieces is summed by all
// warps of the CTA together (pieces dealt to the warps, their sums added in warp order), so that what the launch takes is
// a few round trips whatever the longest run: 12 us for the 131072-token case, 26 us with a CTA per job.
constexpr int kJoinCols = 128, kJoinWarps = kThreads / 32, kJoinAlone = 16;
struct JoinJob {
  int win, second, pieces, col, key;
};
__device__ __forceinline__ float4 add4(float4 a, float4 b) {
  return make_float4(a.x + b.x, a.y + b.y, a.z + b.z, a.w + b.w);
}
__device__ __forceinline__ float4 join_pieces(const ReduceParams& p, const JoinJob& j, int col, int from, int step) {
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < p.D) {
#pragma unroll 8
    for (int i = from; i < j.pieces; i += step) {
      const int64_t slot = i == 0 ? int64_t(j.win) * 2 + 1 : int64_t(j.second + i - 1) * 2;
      s = add4(s, __ldcg(reinterpret_cast<const float4*>(p.part + slot * p.D + col)));
    }
  }
  return s;
}
__device__ __forceinline__ void join_write(const ReduceParams& p, int key, int col, float4 s) {
  if (col >= p.D) return;
  float4* o = reinterpret_cast<float4*>(p.dtable + int64_t(key) * p.D + col);
  const float4 r = make_float4(p.scale * s.x, p.scale * s.y, p.scale * s.z, p.scale * s.w);
  *o = p.accumulate ? add4(*o, r) : r;
}
__global__ void __launch_bounds__(kThreads) k_embed_join(const ReduceParams p) {
  __shared__ float4 red[kJoinWarps][32];
  __shared__ JoinJob long_jobs[kJoinWarps];
  __shared__ int n_long;
  after_previous();
  const int count = __ldcg(p.chains), half = p.win / 2;
  const int col_blocks = (p.D + kJoinCols - 1) / kJoinCols;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t jobs = int64_t(count) * col_blocks;
  // jobs are dealt to the CTAs first: the column blocks of one long run go to different CTAs
  for (int64_t job0 = blockIdx.x; job0 < jobs; job0 += int64_t(gridDim.x) * kJoinWarps) {
    if (threadIdx.x == 0) n_long = 0;
    __syncthreads();
    const int64_t job = job0 + int64_t(warp) * gridDim.x;
    if (job < jobs) {
      JoinJob j;
      j.win = __ldcg(p.chains + 1 + int(job / col_blocks));
      j.col = int(job % col_blocks) * kJoinCols;
      const int edge = (j.win + 1) * p.win;
      const int k = __ldcg(p.keys + edge);
      j.key = k;
      // the first cut: at this edge, or at the next one when the run has fewer than half a window on a side of this edge
      const bool here = edge >= half && __ldcg(p.keys + edge - half) == k && edge + half - 1 < p.n &&
                        __ldcg(p.keys + edge + half - 1) == k;
      j.second = here ? j.win + 1 : j.win + 2;   // the window that holds the second piece
      // the edges after it at which the run is cut too: those with half a window of it behind them
      j.pieces = 2;
      for (int w0 = j.second + 1;; w0 += 128) {
        int found = 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int64_t at = int64_t(w0 + q * 32 + lane) * p.win + half - 1;
          found += __popc(__ballot_sync(0xffffffffu, at < p.n && __ldcg(p.keys + at) == k));
        }
        j.pieces += found;
        if (found < 128) break;
      }
      const int col = j.col + lane * 4;
      if (j.pieces <= kJoinAlone) join_write(p, k, col, join_pieces(p, j, col, 0, 1));
      else if (lane == 0) long_jobs[atomicAdd(&n_long, 1)] = j;
    }
    __syncthreads();
    const int longs = n_long;
    for (int i = 0; i < longs; ++i) {            // in whatever order they were listed: they write different columns
      const JoinJob j = long_jobs[i];
      const int col = j.col + lane * 4;
      red[warp][lane] = join_pieces(p, j, col, warp, kJoinWarps);
      __syncthreads();
      if (warp == 0) {
        float4 s = red[0][lane];
        for (int w = 1; w < kJoinWarps; ++w) s = add4(s, red[w][lane]);
        join_write(p, j.key, col, s);
      }
      __syncthreads();
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
  const int64_t n = std::min(T, kSection), windows = windows_up_to(n, D);
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
  NM_REQUIRE(D <= 65536, w + ": D <= 65536");   // row offsets of a section are 32-bit counts of 16-byte pieces
  NM_REQUIRE(V > 0, w + ": the vocabulary size V must be positive");
}
void require_arch(const char* who) {
  NM_REQUIRE(ce::device_arch() >= 100, std::string(who) + ": this library holds sm_100a code only");
}

template <class Kernel, class Params>
void launch_next(Kernel kernel, dim3 grid, int threads, int smem, const Params& p, cudaStream_t st) {
  if (smem > 48 * 1024) NM_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  ce::launch_after(kernel, grid, unsigned(threads), unsigned(smem), st, p);
}

template <int R>
void launch_sort(const SortParams& p, cudaStream_t st) {
  const uint32_t smem = sort_smem_bytes(p.per);
  NM_CUDA(cudaFuncSetAttribute(k_embed_sort<R>, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
  NM_CUDA(cudaFuncSetAttribute(k_embed_sort<R>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(p.cluster));
  cfg.blockDim = dim3(kSortThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(p.cluster); attr.val.clusterDim.y = 1; attr.val.clusterDim.z = 1;
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
  // one batch where that leaves SMs without a CTA otherwise
  const int groups = kThreads / G;
  const int batches = T >= int64_t(groups) * kFwdRows * kFwdMaxBatches * ce::sm_count() * 8 ? kFwdMaxBatches : 1;
  const int64_t per_cta = int64_t(groups) * kFwdRows * batches, grid = (T + per_cta - 1) / per_cta;
  NM_REQUIRE(grid <= INT_MAX, "embed_fwd: too many rows for one launch");
  auto kern = bf16 ? k_embed_fwd<true> : k_embed_fwd<false>;
  kern<<<unsigned(grid), kThreads, 0, st>>>(table, tokens, out, scale, T, D, V, G, batches);
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
    SortParams sp{tokens + t0, n, V, D, per, (bits + kDigitBits - 1) / kDigitBits, r.keys, r.pos, r.chains, cluster};
    if (n <= kRankMax) {
      k_embed_rank<<<unsigned((n + 31) / 32), kThreads, 0, st>>>(sp);
      NM_CUDA(cudaGetLastError());
    } else {
      switch (per / kSortThreads) {
        case 1: launch_sort<1>(sp, st); break;
        case 2: launch_sort<2>(sp, st); break;
        case 4: launch_sort<4>(sp, st); break;
        default: launch_sort<8>(sp, st); break;
      }
    }
    const bool wide = reinterpret_cast<uintptr_t>(dtable) % 32 == 0;
    if (!add) {   // at most one CTA on each SM that does not sort
      int log_ctas = 0;
      while ((2 << log_ctas) <= ce::sm_count() - (n > kRankMax ? cluster : 0)) ++log_ctas;
      const ZeroParams zp{tokens + t0, dtable, n, V, D, log_ctas, wide};
      launch_next(k_embed_zero_absent, dim3(1u << log_ctas), kZeroThreads, 0, zp, st);
    }
    ReduceParams rp{};
    rp.dy = static_cast<const uint8_t*>(dy) + t0 * D * (bf16 ? 2 : 4);
    rp.keys = r.keys, rp.pos = r.pos, rp.chains = r.chains, rp.part = r.part, rp.dtable = dtable, rp.scale = scale;
    rp.n = n, rp.V = V, rp.D = D, rp.G = threads_per_row(D / 8), rp.accumulate = add;
    rp.win = window_for(n, D), rp.windows = int(windows_of(n, D));
    rp.wide = wide;
    const int groups = kThreads / rp.G;
    const dim3 rg(unsigned((rp.windows + groups - 1) / groups), unsigned((D / 8 + rp.G - 1) / rp.G));
    if (bf16) launch_next(k_embed_reduce<true>, rg, kThreads, reduce_smem_bytes<true>(groups, rp.win), rp, st);
    else launch_next(k_embed_reduce<false>, rg, kThreads, reduce_smem_bytes<false>(groups, rp.win), rp, st);
    const int64_t jobs = int64_t(rp.windows) * ((D + kJoinCols - 1) / kJoinCols);
    launch_next(k_embed_join, dim3(unsigned(std::min<int64_t>(jobs, int64_t(ce::sm_count()) * 8))), kThreads, 0, rp, st);
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
