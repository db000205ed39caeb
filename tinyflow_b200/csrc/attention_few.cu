// Attention of a few queries: tokens that are answered one by one.  Exact fp32, bound by the bytes of keys and values.
//
// 8, 16 or 32 lanes share a key, each with up to eight of its elements; up to four rows (queries of all heads that share the key-value head) have their
// queries and sums in registers, so keys and values go from memory to registers once and nothing else moves.  Of the scores of a step (rows x 2 keys) a lane looks after one:
// the dots are added up by an exchange that leaves each lane its own, which then takes cap, bias, mask and exponential once and hands the weight round (58 us against 62 with
// all lanes doing all scores, at 8 x 4096 keys of 8 heads with four queries each, 128 wide).  A running maximum and sum per score's lane,
// joined at the end over the warp, the block and, where one block per key-value head would leave SMs idle, over blocks that take shares of the keys: the last one to finish
// adds the parts up in their order, its warps taking turns at them (52.6 us; a thread for an element took 58, and at 74 shares 108 instead of 78).
// That size, 268 MB, takes 50.5 us = 5.3 TB/s, bound by bytes in flight and the latency of a step; keys copied asynchronously through shared memory three steps
// ahead took 63, one block a share more (two waves) 60.
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
  float* part;                       // of every block: part_floats(rows, D)
  uint32_t* counters;                // of every sequence, key-value head and block of rows
};

// Sums N numbers over kLanes lanes; lane l is left with that of number l / (kLanes / N).  A lane gives half of what it has to the lane that keeps it, so N - 1 exchanges
// stand for log2(kLanes) * N.
template <int kLanes, int N> __device__ __forceinline__ float over_lanes(float* v) {
  int o = kLanes / 2;
#pragma unroll
  for (int n = N / 2; n > 0; n >>= 1, o >>= 1) {
    const bool upper = threadIdx.x & o;
#pragma unroll
    for (int i = 0; i < n; ++i) {
      const float keep = upper ? v[i + n] : v[i], give = upper ? v[i] : v[i + n];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, give, o);
    }
  }
#pragma unroll
  for (o = kLanes / N / 2; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
  return v[0];
}

// A part: sums [rows][D], then the rows' maxima and the sums of their weights
__host__ __device__ constexpr int part_floats(int rows, int D) { return (rows * (D + 2) + 3) / 4 * 4; }

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
  // A lane looks after the score of one row and one key of a step
  constexpr int kScores = ROWS * kUnroll, kShare = kLanes / kScores;
  static_assert(kShare > 0, "a lane has one score at most");
  const int score = piece / kShare, my_row = rows_at + score / kUnroll, my_u = score % kUnroll, lane0 = lane / kLanes * kLanes;
  const bool my_row_there = my_row < count;
  const int my_at = (my_row_there ? my_row / a.group : 0) + a.Tk - a.Tq;
  const Sight my_sight = my_row_there ? sight_of(a, my_at) : Sight{1, 0};
  const float my_slope = my_row_there && a.slopes ? __ldg(a.slopes + kv * a.group + my_row % a.group) : 0.f;
  const float my_document = a.documents ? (my_row_there ? document_of(a, b, my_at) : -1.f) : 0.f;
  float q[ROWS][DL], acc[ROWS][DL], most = -INFINITY, sum = 0.f;
  const int prefix = prefix_of(a, b);
  int first = a.Tk, end = prefix, all_from = 0, all_to = a.documents ? 0 : a.Tk;       // keys that some row may see, and that every row sees, so that nothing is looked at one by one
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    const int row = rows_at + r, i = row / a.group, h = kv * a.group + row - i * a.group;
    const bool there = row < count;
    const Sight sight = there ? sight_of(a, i + a.Tk - a.Tq) : Sight{1, 0};
    if (sight.lo <= sight.hi) { first = min(first, sight.lo); end = max(end, min(sight.hi, a.Tk - 1) + 1); }
    all_from = max(all_from, sight.lo); all_to = min(all_to, sight.hi + 1);
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
  all_to = min(all_to, to);
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
    if (VEC == 4 && piece * 32 < D) {            // the lines of the next step's keys: one lane a line (two steps ahead took 52.6 us)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u)
        if (j0 + (kUnroll + u) * kAtOnce + sub < to) {
          const int64_t ahead = (kUnroll + u) * kAtOnce * stride + piece * (32 - VEC);
          asm volatile("prefetch.global.L2 [%0];" ::"l"(kp + ahead));
          asm volatile("prefetch.global.L2 [%0];" ::"l"(vp + ahead));
        }
    }
    float dots[kScores];
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        float2 dot = mul2(at2(q[r], 0), at2(k[u], 0));
#pragma unroll
        for (int d = 2; d < DL; d += 2) dot = fma2(at2(q[r], d), at2(k[u], d), dot);
        dots[r * kUnroll + u] = dot.x + dot.y;
      }
    float s = __fmul_rn(over_lanes<kLanes, kScores>(dots), scale);   // rounded before the maximum is taken off, however large it is
    if (!(fabsf(s) < INFINITY)) s = NAN;         // a cap or a weight of zero would hide what is not finite
    const int j = j0 + my_u * kAtOnce + sub;
    if (SHAPED) {
      if (a.cap > 0.f) s = a.cap * tanhf(s / a.cap);
      s = __fmul_rn(fmaf(-my_slope, fabsf((float)(my_at - j)), s), kLog2e);
    }
    unsigned seen_by = 0xffffffffu;
    if (!whole) {
      bool seen = j < to && sees(my_sight, prefix, j) && my_row_there;
      if (a.documents && seen) { const float of = __ldg(a.documents + (int64_t)b * a.Tk + j); seen = of == my_document && of >= 0.f; }
      if (!seen) s = -INFINITY;
      seen_by = __ballot_sync(0xffffffffu, seen);
    }
    float m = fmaxf(most, s);
#pragma unroll
    for (int o = kShare; o < kShare * kUnroll; o <<= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (__any_sync(0xffffffffu, m > most)) {     // rarely, after the first keys
      const float faded = exp2_fast(most - max_of_finite_or(m));
      sum *= faded;
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float f = __shfl_sync(0xffffffffu, faded, lane0 + r * kUnroll * kShare);
#pragma unroll
        for (int d = 0; d < DL; d += 2) put2(acc[r], d, mul2(at2(acc[r], d), both(f)));
      }
      most = m;
    }
    const float weight = exp2_fast(s - max_of_finite_or(m));
    sum += weight;
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
      for (int u = 0; u < kUnroll; ++u) {
        const int of = lane0 + (r * kUnroll + u) * kShare;
        const float w = __shfl_sync(0xffffffffu, weight, of);
        if (whole || (seen_by >> of & 1)) {      // what the row does not see may hold anything
#pragma unroll
          for (int d = 0; d < DL; d += 2) put2(acc[r], d, fma2(both(w), at2(v[u], d), at2(acc[r], d)));
        }
      }
  }
  // over the groups of the warp
#pragma unroll
  for (int o = kShare; o < kShare * kUnroll; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
  for (int o = kLanes; o < 32; o <<= 1) {
    const float m = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o)), faded = exp2_fast(most - max_of_finite_or(m));
    most = m;
    sum *= faded;
    sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float f = __shfl_sync(0xffffffffu, faded, lane0 + r * kUnroll * kShare);
#pragma unroll
      for (int d = 0; d < DL; ++d) { acc[r][d] *= f; acc[r][d] += __shfl_xor_sync(0xffffffffu, acc[r][d], o); }
    }
  }
  if (lane < kLanes) {
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      float* const mine = held + (warp * ROWS + r) * (D + 2);
      if (piece == r * kUnroll * kShare) { mine[D] = most; mine[D + 1] = sum; }
#pragma unroll
      for (int n = 0; n < kPieces; ++n)
#pragma unroll
        for (int i = 0; i < VEC; ++i) if ((piece + kLanes * n) * VEC + i < D) mine[(piece + kLanes * n) * VEC + i] = acc[r][n * VEC + i];
    }
  }
  __syncthreads();
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
  float* const parts = p.part + (int64_t)rest * p.shares * part_floats(ROWS, D);
  for (int n = threadIdx.x; n < ROWS * D; n += kThreads) {
    const int r = n / D, d = n - r * D;
    const float* const from_warps = held + r * (D + 2);
    float m = -INFINITY, total = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) m = fmaxf(m, from_warps[w * ROWS * (D + 2) + D]);
    const float origin = max_of_finite_or(m);
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float* const of = from_warps + w * ROWS * (D + 2);
      const float faded = exp2_fast(of[D] - origin);
      total = fmaf(of[D + 1], faded, total);
      x = fmaf(of[d], faded, x);
    }
    if (p.shares == 1) { finish(r, d, x, m, total); continue; }
    float* const mine = parts + (int64_t)share * part_floats(ROWS, D);
    mine[n] = x;
    if (d == 0) { mine[ROWS * D + r] = m; mine[ROWS * D + ROWS + r] = total; }
  }
  if (p.shares == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(p.counters + rest, (unsigned)p.shares - 1) == (unsigned)p.shares - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // The last block: every warp takes every fourth part, with the factors of 32 parts in its lanes
  constexpr int kWide = kLanes * DL > 32 * VEC ? kLanes * DL / (32 * VEC) : 1;
  const float* const stats = parts + ROWS * D;
  float top[ROWS], total[ROWS], x[ROWS][kWide * VEC];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    top[r] = -INFINITY; total[r] = 0.f;
#pragma unroll
    for (int n = 0; n < kWide * VEC; ++n) x[r][n] = 0.f;
  }
  for (int i0 = 0; i0 < p.shares; i0 += 32) {
    float faded[ROWS];
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const float* const of = stats + (int64_t)(i0 + lane) * part_floats(ROWS, D) + r;
      const bool there = i0 + lane < p.shares;
      const float most_of = there ? __ldcg(of) : -INFINITY, sum_of = there ? __ldcg(of + ROWS) : 0.f;
      float m = fmaxf(top[r], most_of);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
      const float origin = max_of_finite_or(m), before = exp2_fast(top[r] - origin);
      faded[r] = exp2_fast(most_of - origin);
      total[r] = fmaf(total[r], before, sum_of * faded[r]);
      if (i0 > 0)
#pragma unroll
        for (int n = 0; n < kWide * VEC; ++n) x[r][n] *= before;
      top[r] = m;
    }
#pragma unroll 2
    for (int i = warp; i < min(32, p.shares - i0); i += kWarps) {
      const float* const of = parts + (int64_t)(i0 + i) * part_floats(ROWS, D);
#pragma unroll
      for (int r = 0; r < ROWS; ++r) {
        const float f = __shfl_sync(0xffffffffu, faded[r], i);
#pragma unroll
        for (int n = 0; n < kWide; ++n) {
          const int d = (lane + 32 * n) * VEC;
          if (d < D) {
            float v[VEC];
            get_beyond_l1<VEC>(v, of + r * D + d);
#pragma unroll
            for (int k = 0; k < VEC; ++k) x[r][n * VEC + k] = fmaf(f, v[k], x[r][n * VEC + k]);
          }
        }
      }
    }
  }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) total[r] += __shfl_xor_sync(0xffffffffu, total[r], o);
#pragma unroll
    for (int n = 0; n < kWide * VEC; ++n) {
      const int d = (lane + 32 * (n / VEC)) * VEC + n % VEC;
      if (d < D) held[(warp * ROWS + r) * D + d] = x[r][n];
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
    for (int d = threadIdx.x; d < D; d += kThreads) {
      float sum_of_warps = 0.f;
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum_of_warps += held[(w * ROWS + r) * D + d];
      finish(r, d, sum_of_warps, top[r], total[r]);
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
    *bytes = sizeof(float) * (size_t)blocks * p.shares * part_floats(rows, a.D);
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
