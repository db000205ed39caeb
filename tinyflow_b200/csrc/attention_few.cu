// Attention of a few queries: tokens that are answered one by one.  Exact fp32, bound by the bytes of keys and values.
//
// 8, 16 or 32 lanes share a key, each with up to eight of its elements; up to four rows (queries of all heads that share the key-value head) have their
// queries and sums in registers, so keys and values go from memory to registers once and nothing else moves.  A running maximum and sum per group of lanes,
// joined at the end over the warp, the block and, where one block per key-value head would leave SMs idle, over blocks that take shares of the keys: the last one to finish
// adds the parts up in their order.
#include "attention.h"
#include <algorithm>
#include <atomic>
#include <type_traits>
#include "pieces.h"

namespace tf {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32, kUnroll = 2, kBlocks = 4;        // keys of a group in flight; blocks an SM

struct FewArgs {
  AttentionArgs a;
  int shares, row_blocks;
  float* part;                       // of every block: rows x (D + 2)
  uint32_t* counters;                // of every sequence, key-value head and block of rows
};

template <int kLanes> __device__ __forceinline__ float over_lanes(float v) {
#pragma unroll
  for (int o = 1; o < kLanes; o <<= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

template <int kLanes, int DL, int ROWS, int VEC, bool SHAPED>
__global__ void __launch_bounds__(kThreads, kBlocks) attention_few_kernel(const __grid_constant__ FewArgs p) {
  constexpr int kPieces = DL / VEC, kAtOnce = kThreads / kLanes;       // keys that a block takes at once
  extern __shared__ float held[];                // [kWarps][ROWS][D + 2]
  __shared__ bool last;
  const AttentionArgs& a = p.a;
  const int share = blockIdx.x % p.shares, rest = blockIdx.x / p.shares, rows_at = rest % p.row_blocks * ROWS, bg = rest / p.row_blocks, b = bg / a.G, kv = bg - b * a.G;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, piece = lane % kLanes, sub = warp * (32 / kLanes) + lane / kLanes;
  const int count = a.group * a.Tq, D = a.D;
  grid_dep_sync();
  float q[ROWS][DL], acc[ROWS][DL], most[ROWS], sum[ROWS], slope[ROWS], document[ROWS];
  Sight sight[ROWS];
  int at[ROWS];
  const int prefix = prefix_of(a, b);
  int first = a.Tk, end = prefix;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = rows_at + r, i = row / a.group, h = kv * a.group + row - i * a.group;
    const bool there = row < count;
    most[r] = -INFINITY; sum[r] = 0.f; slope[r] = 0.f; document[r] = 0.f;
    at[r] = i + a.Tk - a.Tq;
    sight[r] = there ? sight_of(a, at[r]) : Sight{1, 0};
    if (!there) at[r] = 0;
    if (there && sight[r].lo <= sight[r].hi) { first = min(first, sight[r].lo); end = max(end, min(sight[r].hi, a.Tk - 1) + 1); }
    if (there && a.slopes) slope[r] = __ldg(a.slopes + h);
    document[r] = a.documents ? (there ? document_of(a, b, at[r]) : -1.f) : 0.f;
    const float* const from = a.q + (((int64_t)b * a.Tq + (there ? i : 0)) * a.H + h) * D;
#pragma unroll
    for (int n = 0; n < kPieces; ++n) {
      const int d = (piece + kLanes * n) * VEC;
      if (there && d < D) get<VEC>(&q[r][n * VEC], from + d);
      else
#pragma unroll
        for (int k = 0; k < VEC; ++k) q[r][n * VEC + k] = 0.f;
#pragma unroll
      for (int k = 0; k < VEC; ++k) acc[r][n * VEC + k] = 0.f;
    }
  }
  if (prefix > 0) first = 0;
  // this block's share of the keys
  const int span = end > first ? end - first : 0, each = (span + p.shares - 1) / p.shares, from = first + share * each, to = min(end, from + each);
  const int64_t stride = (int64_t)a.G * D, base = (((int64_t)b * a.Tk + from + sub) * a.G + kv) * D + piece * VEC;
  const float *kp = a.k + base, *vp = a.v + base;
  // keys that every row sees, so that nothing is looked at one by one
  int all_from = 0, all_to = a.documents ? 0 : to;
#pragma unroll
  for (int r = 0; r < ROWS; ++r) { all_from = max(all_from, sight[r].lo); all_to = min(all_to, sight[r].hi + 1); }
  const float scale = SHAPED ? a.scale : a.scale * kLog2e;
  for (int j0 = from; j0 < to; j0 += kAtOnce * kUnroll, kp += kAtOnce * kUnroll * stride, vp += kAtOnce * kUnroll * stride) {
    float k[kUnroll][DL], v[kUnroll][DL];
    const bool whole = j0 >= all_from && j0 + kAtOnce * kUnroll <= all_to;
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const bool there = whole || j0 + u * kAtOnce + sub < to;
#pragma unroll
      for (int n = 0; n < kPieces; ++n) {
        if (there && (piece + kLanes * n) * VEC < D) {
          get<VEC>(&k[u][n * VEC], kp + u * kAtOnce * stride + kLanes * n * VEC);
          get<VEC>(&v[u][n * VEC], vp + u * kAtOnce * stride + kLanes * n * VEC);
        } else {
#pragma unroll
          for (int i = 0; i < VEC; ++i) k[u][n * VEC + i] = v[u][n * VEC + i] = 0.f;
        }
      }
    }
    if (VEC == 4 && piece * 32 < D) {            // the lines of the keys two passes ahead: one lane a line
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j0 + (2 * kUnroll + u) * kAtOnce + sub < to) {
          const int64_t ahead = (2 * kUnroll + u) * kAtOnce * stride + piece * (32 - VEC);
          asm volatile("prefetch.global.L2 [%0];" ::"l"(kp + ahead));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(vp + ahead));
        }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float s[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float dot = 0.f;
#pragma unroll
        for (int d = 0; d < DL; ++d) dot = fmaf(q[r][d], k[u][d], dot);
        s[u] = over_lanes<kLanes>(dot) * scale;
        if (SHAPED) {
          if (a.cap > 0.f) s[u] = a.cap * tanhf(s[u] / a.cap);
          s[u] = (s[u] - slope[r] * fabsf((float)(at[r] - j0 - u * kAtOnce - sub))) * kLog2e;
        }
      }
      bool seen[kUnroll];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) seen[u] = true;
      if (!whole) {
#pragma unroll
        for (int u = 0; u < kUnroll; ++u) {
          const int j = j0 + u * kAtOnce + sub;
          seen[u] = j < to && sees(sight[r], prefix, j) && rows_at + r < count;
          if (a.documents && seen[u]) { const float of = __ldg(a.documents + (int64_t)b * a.Tk + j); seen[u] = of == document[r] && of >= 0.f; }
          if (!seen[u]) s[u] = -INFINITY;
        }
      }
      float m = most[r];
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) m = fmaxf(m, s[u]);
      if (m > most[r]) {                         // rarely, after the first keys
        const float faded = exp2_fast(most[r] - m);
        sum[r] *= faded;
#pragma unroll
        for (int d = 0; d < DL; ++d) acc[r][d] *= faded;
        most[r] = m;
      }
      const float origin = max_of_finite_or(m);
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const float w = exp2_fast(s[u] - origin);
        sum[r] += w;
        if (whole) {
#pragma unroll
          for (int d = 0; d < DL; ++d) acc[r][d] = fmaf(w, v[u][d], acc[r][d]);
        } else if (seen[u]) {                    // what the row does not see may hold anything
#pragma unroll
          for (int d = 0; d < DL; ++d) acc[r][d] = fmaf(w, v[u][d], acc[r][d]);
        }
      }
    }
  }
  // over the groups of the warp
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1)
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float m = fmaxf(most[r], __shfl_xor_sync(0xffffffffu, most[r], o)), faded = exp2_fast(most[r] - max_of_finite_or(m));
      most[r] = m;
      sum[r] *= faded;
      sum[r] += __shfl_xor_sync(0xffffffffu, sum[r], o);
#pragma unroll
      for (int d = 0; d < DL; ++d) { acc[r][d] *= faded; acc[r][d] += __shfl_xor_sync(0xffffffffu, acc[r][d], o); }
    }
  if (lane < kLanes) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float* const mine = held + (warp * ROWS + r) * (D + 2);
      if (piece == 0) { mine[D] = most[r]; mine[D + 1] = sum[r]; }
#pragma unroll
      for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) if ((piece + kLanes * n) * VEC + i < D) mine[(piece + kLanes * n) * VEC + i] = acc[r][n * VEC + i];
    }
  }
  __syncthreads();
  // Joins `count` parts of row r, `step` floats apart; column d of it
  const auto joined = [&](const float* parts, int64_t step, int parts_count, int d, bool beyond_l1, float& m, float& total) {
    const auto read = [&](int64_t i) { return beyond_l1 ? __ldcg(parts + i) : parts[i]; };
    m = -INFINITY;
    for (int i = 0; i < parts_count; ++i) m = fmaxf(m, read(i * step + D));
    const float origin = max_of_finite_or(m);
    float s = 0.f, x = 0.f;
    for (int i = 0; i < parts_count; ++i) {
      const float faded = exp2_fast(read(i * step + D) - origin);
      s = fmaf(read(i * step + D + 1), faded, s);
      x = fmaf(read(i * step + d), faded, x);
    }
    total = s;
    return x;
  };
  const auto finish = [&](int r, int d, float x, float m, float total) {
    const int row = rows_at + r, i = row / a.group, h = kv * a.group + row - i * a.group;
    if (row >= count) return;
    const float inv = total == 0.f ? 0.f : 1.f / total;
    a.o[(((int64_t)b * a.Tq + i) * a.H + h) * D + d] = x * inv;
    if (a.stats && d == 0) {
      float* const stat = a.stats + 2 * (((int64_t)b * a.H + h) * a.Tq + i);
      stat[0] = max_of_finite_or(m); stat[1] = inv;
    }
  };
  const int64_t size = (int64_t)ROWS * (D + 2);
  float* const parts = p.part + ((int64_t)rest * p.shares) * size;
  for (int n = threadIdx.x; n < ROWS * D; n += kThreads) {
    const int r = n / D, d = n - r * D;
    float m, total;
    const float x = joined(held + r * (D + 2), ROWS * (D + 2), kWarps, d, false, m, total);
    if (p.shares == 1) { finish(r, d, x, m, total); continue; }
    float* const mine = parts + share * size + r * (D + 2);
    mine[d] = x;
    if (d == 0) { mine[D] = m; mine[D + 1] = total; }
  }
  if (p.shares == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(p.counters + rest, (unsigned)p.shares - 1) == (unsigned)p.shares - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  for (int n = threadIdx.x; n < ROWS * D; n += kThreads) {
    const int r = n / D, d = n - r * D;
    float m, total;
    const float x = joined(parts + r * (D + 2), size, p.shares, d, true, m, total);
    finish(r, d, x, m, total);
  }
}

}  // namespace

// 0: launched; -1: error; 1: short of *bytes
int attention_few(const AttentionArgs& a, size_t* bytes, cudaStream_t s, const char* what) {
  const int64_t count = (int64_t)a.group * a.Tq;
  const int rows = count > 2 ? 4 : (int)count;
  FewArgs p;
  memset(&p, 0, sizeof(p));
  p.a = a;
  p.row_blocks = (int)((count + rows - 1) / rows);
  const int64_t blocks = (int64_t)a.B * a.G * p.row_blocks;
  // One wave of blocks, shares of at least 64 keys
  p.shares = (int)std::max<int64_t>(1, std::min<int64_t>(kBlocks * device_sm_count() / blocks, a.Tk / 64));
  TF_REQUIRE(blocks * p.shares < (1ll << 31), "%s: too many blocks", what);
  StreamLease lease(s);
  if (p.shares > 1) {
    *bytes = sizeof(float) * (size_t)blocks * p.shares * rows * (a.D + 2);
    if (!(p.part = (float*)lease.scratch(kScratchAttention, *bytes)) || !(p.counters = lease.counters((int)blocks))) return 1;
  }
  uintptr_t bits = (uintptr_t)a.D * sizeof(float);
  for (const void* x : {(const void*)a.q, (const void*)a.k, (const void*)a.v}) bits |= reinterpret_cast<uintptr_t>(x);
  cudaError_t e = cudaSuccess;
  const auto launch = [&](auto lanes, auto dl, auto r, auto vec) {
    constexpr int L = decltype(lanes)::value, DL = decltype(dl)::value, R = decltype(r)::value, V = decltype(vec)::value;
    e = launch_dep(a.cap > 0.f || a.slopes ? attention_few_kernel<L, DL, R, V, true> : attention_few_kernel<L, DL, R, V, false>, dim3((unsigned)(blocks * p.shares)), dim3(kThreads), sizeof(float) * kWarps * R * (size_t)(a.D + 2), s, p);
  };
  const auto with_rows = [&](auto lanes, auto dl, auto vec) {
    if (rows == 1) launch(lanes, dl, std::integral_constant<int, 1>(), vec);
    else if (rows == 2) launch(lanes, dl, std::integral_constant<int, 2>(), vec);
    else launch(lanes, dl, std::integral_constant<int, 4>(), vec);
  };
  const auto with_width = [&](auto lanes, auto dl) { if (bits % 16 == 0) with_rows(lanes, dl, std::integral_constant<int, 4>()); else with_rows(lanes, dl, std::integral_constant<int, 1>()); };
  if (a.D <= 32) with_width(std::integral_constant<int, 8>(), std::integral_constant<int, 4>());
  else if (a.D <= 64) with_width(std::integral_constant<int, 8>(), std::integral_constant<int, 8>());
  else if (a.D <= 128) with_width(std::integral_constant<int, 16>(), std::integral_constant<int, 8>());
  else with_width(std::integral_constant<int, 32>(), std::integral_constant<int, 8>());
  TF_CUDA(e);
  TF_AFTER(s, what);
  return 0;
}

}  // namespace tf
