// Layer normalisation over the last axis, alone and behind the residual sum of a dropped-out branch, forward and backward.
//
//   s = residual + keep * branch / (1 - p)                    (the second form only; without it s is the input)
//   y = gamma * xh + beta,  xh = (s - mean) * inv,  inv = (mean((s - mean)^2) + eps)^(-1/2)
//   g = gamma * dy,  ds = inv * (g - mean(g) - xh * mean(g * xh)) [+ the gradient that reaches s behind the block]
//   dgamma = sum over rows of dy * xh,  dbeta = sum over rows of dy,  dbranch = keep * ds / (1 - p)
//
// HBM-bound: every tensor is read once and written once.  A row stays in the registers of one group of threads, so the mean is
// known before the squares are summed, so squares of far numbers never cancel, and the backward pass forms the statistics again instead of
// reading them.  What an offset does cost is the rounding of the mean, one fp32 number: up to n 2^-24 mean|s| (n additions, 64 and D / 512) shifts
// every s - mean alike, 1e-3 of a spread at 1e4 spreads from zero.  (Adding up s - mean as well and taking its mean off would end that, and costs 3 to
// 10 % of every call, or 1 to 11 where only far rows do it.)  keep is drawn from (seed, element index) again, nothing of it is stored.
#include "common.h"
#include <math.h>
#include <algorithm>
#include <initializer_list>
#include <cooperative_groups.h>
#include <type_traits>
#include "operands.h"
#include "pieces.h"

namespace cg = cooperative_groups;

namespace tf {

struct NormArgs {
  const float* x;            // forward: the input, or the branch; backward: the tensor that was normalised
  const float* residual;     // forward with a residual
  const float* gamma;
  const float* beta;
  const float* dy;
  const float* dsum;         // backward with a residual: the gradient that s has from elsewhere, or null
  float* sum;                // forward with a residual
  float* y;                  // may be null with a residual
  float* dx;                 // may be null
  float* dbranch;            // may be null
  float* part;               // [block][2 * D] sums of dy * xh and of dy, or null
  float *dgamma, *dbeta;     // where a grid of one cluster leaves them itself (either may be null)
  float2* stats;             // per row: mean and inv (rows that do not fit the registers)
  int64_t rows;
  int D;
  float eps, p, scale;
  uint32_t threshold;        // of the upper word of the mixed number: below it an element is dropped
  unsigned long long seed;
  const uint32_t* seed_word;
  AmaxOut am;
};

// Sums over the G threads that share a row, the same in all of them.  Two buffers in turn: a thread that writes one for the next sum
// has passed the barrier behind which every thread had read the one before.
template <int G> struct RowSum {
  static constexpr int kWarps = G / 32;
  float (*held)[2][3][kWarps];
  int group, turn = 0;
  __device__ __forceinline__ void barrier() const {
    if (G == 32) __syncwarp();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(G) : "memory");
  }
  template <int N> __device__ __forceinline__ void operator()(float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    if (G == 32) return;
    const int lane = threadIdx.x & 31, w = (threadIdx.x >> 5) % kWarps;
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < N; ++i) held[group][turn][i][w] = v[i];
    }
    barrier();
#pragma unroll
    for (int i = 0; i < N; ++i) {
      v[i] = held[group][turn][i][0];
#pragma unroll
      for (int k = 1; k < kWarps; ++k) v[i] += held[group][turn][i][k];
    }
    turn ^= 1;
  }
};

__device__ __forceinline__ unsigned long long seed_of(const NormArgs& a) { return a.seed_word ? (unsigned long long)__ldg(a.seed_word) : a.seed; }
// What uniform01(seed, i) >= p says, from z = (i + 1) * step + seed * key: its 24 bits are compared as a whole number, and only the
// upper word of the mix decides.  z of the elements of a thread differ by constants.
constexpr unsigned long long kMixStep = 0x9E3779B97F4A7C15ull, kMixKey = 0xD1342543DE82EF95ull;
__device__ __forceinline__ float dropped(const NormArgs& a, unsigned long long z, float v) {
  if (a.p == 0.f) return v * a.scale;
  z = (z ^ (z >> 30)) * 0xBF58476D1CE4E5B9ull;
  z = (z ^ (z >> 27)) * 0x94D049BB133111EBull;
  const uint32_t upper = (uint32_t)(z >> 32);
  return (upper ^ upper >> 31) >= a.threshold ? v * a.scale : 0.f;
}
__device__ __forceinline__ unsigned long long mix_start(unsigned long long seed, int64_t i) { return (unsigned long long)(i + 1) * kMixStep + seed * kMixKey; }

// A row of D elements is dealt to G threads, NV pieces of VEC elements each: piece v of thread t begins at element (v * G + t) * VEC.
// The shape of a launch (with_shape) is the smallest that fits, in steps of four elements a thread, so only the last of them need a look
// at D; the rest are there at compile time.  (With pieces of 4 to 16 elements and a look at every one, scalar rows of 2050 elements took
// 234 instructions an element in the backward kernel.)
template <int VEC, int G, int NV> struct Row {
  static constexpr int kStep = 4 / VEC;
  int D, t;
  __device__ __forceinline__ int at(int v) const { return (v * G + t) * VEC; }
  __device__ __forceinline__ bool has(int v) const { return v < NV - kStep || at(v) < D; }
  // whether the row has any of the pair that piece v begins or ends: what has none is skipped, not computed on zeros
  __device__ __forceinline__ bool begins(int v) const { return has(VEC == 1 ? v & ~1 : v); }
  // pair i of the thread's elements: v where the row has it, else 0 (a pair may lie in two pieces of one element)
  __device__ __forceinline__ float2 where(int i, float v) const {
    const int first = 2 * i / VEC, second = (2 * i + 1) / VEC;
    return make_float2(has(first) ? v : 0.f, has(second) ? v : 0.f);
  }
};

// Arithmetic goes two elements at a time (a packed instruction each).
template <int N> __device__ __forceinline__ float2& pair(float (&x)[N], int i) { return reinterpret_cast<float2*>(x)[i]; }
__device__ __forceinline__ float2 both(float v) { return make_float2(v, v); }
// The sum of a thread's elements, in four chains
template <int E> __device__ __forceinline__ float row_part(float (&x)[E]) {
  float2 p[2] = {both(0.f), both(0.f)};
#pragma unroll
  for (int i = 0; i < E / 2; ++i) p[i & 1] = __fadd2_rn(p[i & 1], pair(x, i));
  p[0] = __fadd2_rn(p[0], p[1]);
  return p[0].x + p[0].y;
}

// R groups, a row each.
template <int VEC, int G, int R, int NV, bool RES>
__global__ void __launch_bounds__(G * R) norm_fwd_kernel(const NormArgs a) {
  __shared__ float held[R][2][3][G / 32];
  grid_dep_sync();
  const int group = threadIdx.x / G, D = a.D;
  constexpr int E = NV * VEC;
  const Row<VEC, G, NV> r{D, (int)(threadIdx.x % G)};
  const float over_d = 1.f / (float)D;
  RowSum<G> add{held, group};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  float m = 0.f;              // a NaN does not raise it: it goes through the pack whatever the scale
  for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.rows; row += (int64_t)gridDim.x * R) {
    const int64_t base = row * D;
    const unsigned long long z = RES ? mix_start(seed, base + r.t * VEC) : 0;
    float x[E];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (r.has(v)) get<VEC>(x + v * VEC, a.x + base + r.at(v));
      else
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[v * VEC + j] = 0.f;
    }
    if (RES) {
      float old[E];
#pragma unroll
      for (int v = 0; v < NV; ++v) if (r.has(v)) get<VEC>(old + v * VEC, a.residual + base + r.at(v));
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        if (r.has(v)) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[v * VEC + j] = old[v * VEC + j] + dropped(a, z + (v * G * VEC + j) * kMixStep, x[v * VEC + j]);
          put<VEC>(a.sum + base + r.at(v), x + v * VEC);
        }
      }
      if (!a.y) continue;
    }
    float sum[1] = {row_part(x)};
    add(sum);
    const float mean = sum[0] * over_d;
    float2 sq = both(0.f);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if (r.begins(2 * i / VEC)) {
        pair(x, i) = __fadd2_rn(pair(x, i), r.where(i, -mean));
        sq = __ffma2_rn(pair(x, i), pair(x, i), sq);
      }
    }
    float squares[1] = {sq.x + sq.y};
    add(squares);
    const float2 inv = both(rsqrtf(fmaf(squares[0], over_d, a.eps)));
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (r.has(v)) {
        float w[VEC], b[VEC];
        get<VEC>(w, a.gamma + r.at(v));
        get<VEC>(b, a.beta + r.at(v));
        if (VEC > 1) {
#pragma unroll
          for (int i = 0; i < VEC / 2; ++i) pair(b, i) = __ffma2_rn(__fmul2_rn(pair(x, v * VEC / 2 + i), inv), pair(w, i), pair(b, i));
        } else {
          b[0] = fmaf(x[v] * inv.x, w[0], b[0]);
        }
#pragma unroll
        for (int j = 0; j < VEC; ++j) m = finite_max(m, b[j]);
        put<VEC>(a.y + base + r.at(v), b);
      }
    }
  }
  amax_commit(a.am, amax_key(m));
}

template <int BYTES> __device__ __forceinline__ void copy_ahead(uint32_t to, const float* from) {
  if (BYTES == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(from), "n"(BYTES) : "memory");
}

// Persistent: blockDim / G groups, each taking every (grid * groups)-th row, so a thread always has the same columns and keeps their
// parts of dgamma and dbeta in registers; the groups' parts are added in group order and left as one row of `part` per block.
// The rows ahead of the present one are copied to shared memory, `depth` of them in flight.  A thread copies what it will read itself, and
// the copies need no barrier; but rows that only 4-byte accesses fit are copied in the 16-byte pieces that they lie in, which their
// readers share (2000 x 4099: 41.0 us with copies of 4 bytes, 37.5 so; even widths are faster with copies of 8: 1000 x 2050 12.1 against 12.7).
constexpr int kBwdThreads = 512;            // most threads of a block
constexpr int kFewBlocks = 8;
constexpr int kBwdSmem = 225 * 1024;
// bytes of a row in the ring: one that begins between boundaries takes a piece more
template <int VEC, int G, int NV> constexpr uint32_t norm_pitch() { return G * NV * VEC * 4 + (VEC == 1 ? 32 : 0); }
template <int VEC, int G, int NV, bool RES>
__global__ void __launch_bounds__(kBwdThreads, 1) norm_bwd_kernel(const NormArgs a, int depth) {
  constexpr int kArrays = RES ? 3 : 2;
  constexpr uint32_t kPitch = norm_pitch<VEC, G, NV>(), kArray = kBwdThreads / G * kPitch, kStage = kArrays * kArray;      // bytes
  __shared__ float held[kBwdThreads / G][2][3][G / 32];
  extern __shared__ __align__(16) float ring[];            // [depth][array][group][kPitch], then gamma; at the end the groups' sums [group][2 * D]
  float* const gamma = ring + depth * (kStage / 4);
  const int group = threadIdx.x / G, groups = blockDim.x / G, D = a.D;
  const Row<VEC, G, NV> r{D, (int)(threadIdx.x % G)};
  const float over_d = 1.f / (float)D;
  const bool with_sum = RES && a.dsum;
  const int64_t first = (int64_t)blockIdx.x * groups + group, stride = (int64_t)gridDim.x * groups;
  const uint32_t mine = (uint32_t)__cvta_generic_to_shared(ring) + group * kPitch;
  // elements from the 16-byte boundary in front of a row to it
  auto shift_of = [&](const float* base, int64_t row) { return VEC > 1 ? 0 : (int)((reinterpret_cast<uintptr_t>(base) >> 2) + (uintptr_t)(row * D)) & 3; };
  auto fetch_row = [&](const float* base, int64_t row, uint32_t to) {
    const float* const from = base + row * D;
    if (VEC > 1) {
#pragma unroll
      for (int v = 0; v < NV; ++v) if (r.has(v)) copy_ahead<VEC * 4>(to + r.at(v) * 4, from + r.at(v));
    } else {
      const int shift = shift_of(base, row), pieces = (shift + D + 3) / 4;
      for (int i = r.t; i < pieces; i += G) {
        const float* const piece = from - shift + 4 * i;
        // a piece may hold the end of the row before and the start of the next, but nothing outside the array
        if (piece >= base && piece + 4 <= base + a.rows * D) copy_ahead<16>(to + 16 * i, piece);
        else
          for (int j = 0; j < 4; ++j) if (piece + j >= from && piece + j < from + D) copy_ahead<4>(to + 16 * i + 4 * j, piece + j);
      }
    }
  };
  auto fetch = [&](int64_t row, uint32_t stage) {          // `stage` in bytes
    if (row < a.rows) {
      fetch_row(a.x, row, mine + stage);
      fetch_row(a.dy, row, mine + stage + kArray);
      if (with_sum) fetch_row(a.dsum, row, mine + stage + 2 * kArray);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  const char* const own = reinterpret_cast<const char*>(ring) + group * kPitch;
  auto fetched = [&](float* to, uint32_t stage, int array, int shift, int v) {
    *reinterpret_cast<typename Pieces<VEC>::T*>(to) = *reinterpret_cast<const typename Pieces<VEC>::T*>(own + stage + array * kArray + (r.at(v) + shift) * 4);
  };
  // gamma of pair i of the thread's elements (what lies behind the last one meets zeros)
  auto gammas = [&](int i) -> float2 {
    if (VEC > 1) return *reinterpret_cast<const float2*>(gamma + r.at(2 * i / VEC) + 2 * i % VEC);
    return make_float2(gamma[r.at(2 * i)], gamma[r.at(2 * i + 1)]);
  };
  grid_dep_sync();
  RowSum<G> add{held, group};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  float m = 0.f;
  constexpr int E = NV * VEC;
  float dgamma[E], dbeta[E];
#pragma unroll
  for (int i = 0; i < E; ++i) dgamma[i] = dbeta[i] = 0.f;
  for (int i = 0; i < depth; ++i) fetch(first + i * stride, i * kStage);
  for (int c = threadIdx.x; c < G * E; c += blockDim.x) gamma[c] = c < D ? __ldg(a.gamma + c) : 0.f;
  __syncthreads();
  uint32_t stage = 0;
  for (int64_t row = first; row < a.rows; row += stride) {
    if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
    else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
    else asm volatile("cp.async.wait_group 3;" ::: "memory");
    if (VEC == 1) add.barrier();               // what the others of the group copied
    float x[E], dy[E], ds[RES ? E : 1];
    const int shift_x = shift_of(a.x, row), shift_dy = shift_of(a.dy, row), shift_ds = RES ? shift_of(a.dsum, row) : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (r.has(v)) {
        if (with_sum) fetched(ds + v * VEC, stage, 2, shift_ds, v);
        fetched(dy + v * VEC, stage, 1, shift_dy, v);
        fetched(x + v * VEC, stage, 0, shift_x, v);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[v * VEC + j] = dy[v * VEC + j] = 0.f;
        if (RES) ds[v * VEC] = 0.f;
      }
    }
    float sum[1] = {row_part(x)};
    add(sum);
    const float mean = sum[0] * over_d;
    float2 sq = both(0.f), sg = both(0.f), sgx = both(0.f);      // (x - mean)^2, g, g * (x - mean)
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if (r.begins(2 * i / VEC)) {
        pair(x, i) = __fadd2_rn(pair(x, i), r.where(i, -mean));
        const float2 g = __fmul2_rn(gammas(i), pair(dy, i));       // in a pair that the row ends in dy is zero
        sq = __ffma2_rn(pair(x, i), pair(x, i), sq);
        sg = __fadd2_rn(sg, g);
        sgx = __ffma2_rn(g, pair(x, i), sgx);
      }
    }
    float three[3] = {sq.x + sq.y, sg.x + sg.y, sgx.x + sgx.y};
    add(three);
    if (VEC == 1 && G == 32) __syncwarp();     // the copies of a lane may replace what another one has read (longer rows have had a barrier)
    fetch(row + depth * stride, stage);        // what was there has been read, by all: the sums had barriers, and depend on the last of it
    stage += kStage;
    if (stage == depth * kStage) stage = 0;
    const float inv = rsqrtf(fmaf(three[0], over_d, a.eps));
    // ds = inv * g - inv * mean(g) - (x - mean) * inv^2 * mean(g * xh)
    const float2 inv2 = both(inv), shift = both(-inv * (three[1] * over_d)), slope = both(-inv * (inv * (inv * (three[2] * over_d))));
    const int64_t base = row * D + r.t * VEC;
    const unsigned long long z = RES ? mix_start(seed, base) : 0;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
      if (r.begins(2 * i / VEC)) {
        const float2 g = __fmul2_rn(gammas(i), pair(dy, i));
        pair(dgamma, i) = __ffma2_rn(__fmul2_rn(pair(dy, i), inv2), pair(x, i), pair(dgamma, i));
        pair(dbeta, i) = __fadd2_rn(pair(dbeta, i), pair(dy, i));
        pair(x, i) = __ffma2_rn(g, inv2, __ffma2_rn(pair(x, i), slope, shift));
        if (with_sum) pair(x, i) = __fadd2_rn(pair(x, i), pair(ds, i));
      }
    }
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (r.has(v)) {
        float* const d = x + v * VEC;
        if (a.dx) {
          put<VEC>(a.dx + base + v * G * VEC, d);
          if (!RES || !a.dbranch)
#pragma unroll
            for (int j = 0; j < VEC; ++j) m = finite_max(m, d[j]);
        }
        if (RES && a.dbranch) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) { d[j] = dropped(a, z + (v * G * VEC + j) * kMixStep, d[j]); m = finite_max(m, d[j]); }
          put<VEC>(a.dbranch + base + v * G * VEC, d);
        }
      }
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  amax_commit(a.am, amax_key(m));
  const bool direct = a.dgamma || a.dbeta;
  if (!a.part && !direct) return;
  __syncthreads();
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (r.has(v)) {
      put<VEC>(ring + (size_t)group * 2 * D + r.at(v), dgamma + v * VEC);
      put<VEC>(ring + (size_t)group * 2 * D + D + r.at(v), dbeta + v * VEC);
    }
  }
  __syncthreads();
  float* const out = direct ? ring : a.part + (int64_t)blockIdx.x * 2 * D;
  for (int c = threadIdx.x; c < 2 * D; c += blockDim.x) {
    float total = ring[c];
    for (int g = 1; g < groups; ++g) total += ring[(size_t)g * 2 * D + c];
    out[c] = total;
  }
  if (!direct) return;
  // few rows: the grid is one cluster, and its blocks add a share of the columns each
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = (int)cluster.num_blocks();
  cluster.sync();
  for (int c = (int)cluster.block_rank() * blockDim.x + threadIdx.x; c < 2 * D; c += ranks * blockDim.x) {
    float v[kFewBlocks];
#pragma unroll
    for (int k = 0; k < kFewBlocks; ++k) v[k] = cluster.map_shared_rank(ring, min(k, ranks - 1))[c];
    float total = v[0];
#pragma unroll
    for (int k = 1; k < kFewBlocks; ++k) if (k < ranks) total += v[k];
    if (c < D) { if (a.dgamma) a.dgamma[c] = total; }
    else if (a.dbeta) a.dbeta[c - D] = total;
  }
  cluster.sync();              // nobody leaves while its shared memory is still read
}

// Rows of more than 8192 elements: their sums and the parts of dgamma and dbeta take the registers, so the row stays in shared memory, every
// piece with the thread that copied it.  Where the last pass has read a piece, the next row's is copied to its place: a row's bytes are
// under way during that pass and the barriers of the next.  gamma has room there without a residual; else it comes from L2.
// (3262 x 14712: 335 us with three passes over global memory, 158 so, 3.6 TB/s; with the residual's arrays 453 and 262, 3.7 TB/s.)
constexpr int kWideThreads = 1024;
template <int VEC, int NV, bool RES>
__global__ void __launch_bounds__(kWideThreads, 1) norm_wide_bwd_kernel(const NormArgs a) {
  constexpr int E = NV * VEC, kArray = E * kWideThreads;            // floats
  __shared__ float held[1][2][3][kWideThreads / 32];
  extern __shared__ __align__(16) float wide[];                     // x, dy, then the gradient of the sum or gamma: [piece][thread]
  grid_dep_sync();
  const int D = a.D;
  const Row<VEC, kWideThreads, NV> r{D, (int)threadIdx.x};
  const float over_d = 1.f / (float)D;
  const bool with_sum = RES && a.dsum;
  RowSum<kWideThreads> add{held, 0};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  auto slot = [&](int array, int v) { return wide + array * kArray + r.at(v); };
  auto copy = [&](const float* from, int64_t row, int array, int v) { copy_ahead<VEC * 4>((uint32_t)__cvta_generic_to_shared(slot(array, v)), from + row * D + r.at(v)); };
  auto fetch = [&](int64_t row, int v) {
    if (row >= a.rows || !r.has(v)) return;
    copy(a.x, row, 0, v);
    copy(a.dy, row, 1, v);
    if (with_sum) copy(a.dsum, row, 2, v);
  };
  auto gamma_of = [&](float* w, int v) {
    if (RES) get<VEC>(w, a.gamma + r.at(v));
    else held_at<VEC>(w, slot(2, v));
  };
  if (!RES)
    for (int v = 0; v < NV; ++v) if (r.has(v)) copy(a.gamma, 0, 2, v);
  for (int v = 0; v < NV; ++v) fetch(blockIdx.x, v);
  float dgamma[E], dbeta[E], m = 0.f;
#pragma unroll
  for (int i = 0; i < E; ++i) dgamma[i] = dbeta[i] = 0.f;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    asm volatile("cp.async.wait_all;" ::: "memory");
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!r.has(v)) continue;
      float x[VEC];
      held_at<VEC>(x, slot(0, v));
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0] += x[j];
    }
    add(sum);
    const float mean = sum[0] * over_d;
    float three[3] = {0.f, 0.f, 0.f};                               // (x - mean)^2, g, g * (x - mean)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!r.has(v)) continue;
      float x[VEC], dy[VEC], w[VEC];
      held_at<VEC>(x, slot(0, v));
      held_at<VEC>(dy, slot(1, v));
      gamma_of(w, v);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = x[j] - mean, g = w[j] * dy[j];
        three[0] = fmaf(d, d, three[0]);
        three[1] += g;
        three[2] = fmaf(g, d, three[2]);
      }
    }
    add(three);
    const float inv = rsqrtf(fmaf(three[0], over_d, a.eps));
    const float shift = -inv * (three[1] * over_d), slope = -inv * (inv * (inv * (three[2] * over_d)));
    const int64_t base = row * D;
    const unsigned long long z = RES ? mix_start(seed, base + r.t * VEC) : 0;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      if (!r.has(v)) continue;
      float x[VEC], dy[VEC], w[VEC], ds[VEC];
      held_at<VEC>(x, slot(0, v));
      held_at<VEC>(dy, slot(1, v));
      gamma_of(w, v);
      if (with_sum) held_at<VEC>(ds, slot(2, v));
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = x[j] - mean;
        dgamma[v * VEC + j] = fmaf(dy[j] * inv, d, dgamma[v * VEC + j]);
        dbeta[v * VEC + j] += dy[j];
        x[j] = fmaf(w[j] * dy[j], inv, fmaf(d, slope, shift));
        if (with_sum) x[j] += ds[j];
      }
      if (a.dx) {
        put<VEC>(a.dx + base + r.at(v), x);
        if (!RES || !a.dbranch)
#pragma unroll
          for (int j = 0; j < VEC; ++j) m = finite_max(m, x[j]);
      }
      if (RES && a.dbranch) {
#pragma unroll
        for (int j = 0; j < VEC; ++j) { x[j] = dropped(a, z + (v * kWideThreads * VEC + j) * kMixStep, x[j]); m = finite_max(m, x[j]); }
        put<VEC>(a.dbranch + base + r.at(v), x);
      }
      fetch(row + gridDim.x, v);
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
  amax_commit(a.am, amax_key(m));
  if (!a.part) return;
  float* const out = a.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll
  for (int v = 0; v < NV; ++v) {
    if (!r.has(v)) continue;
    put<VEC>(out + r.at(v), dgamma + v * VEC);
    put<VEC>(out + D + r.at(v), dbeta + v * VEC);
  }
}

// Rows of any length (forward above 16384 elements, backward too), a block each: three passes over the row, which L1 and L2 hold from the second on.
constexpr int kLongThreads = 512;
template <bool RES> __global__ void __launch_bounds__(kLongThreads) norm_long_fwd_kernel(const NormArgs a) {
  __shared__ float held[1][2][3][kLongThreads / 32];
  grid_dep_sync();
  RowSum<kLongThreads> add{held, 0};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  const int D = a.D;
  uint32_t m = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * D;
    const float* const x = RES ? a.sum + base : a.x + base;            // a thread reads what it wrote itself
    float sum[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += kLongThreads) {
      float v = a.x[base + c];
      if (RES) { v = a.residual[base + c] + dropped(a, mix_start(seed, base + c), v); a.sum[base + c] = v; }
      sum[0] += v;
    }
    if (RES && !a.y) continue;
    add(sum);
    const float mean = sum[0] / (float)D;
    float squares[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += kLongThreads) { const float v = x[c] - mean; squares[0] = fmaf(v, v, squares[0]); }
    add(squares);
    const float inv = __frsqrt_rn(squares[0] / (float)D + a.eps);
    for (int c = threadIdx.x; c < D; c += kLongThreads) {
      const float y = fmaf((x[c] - mean) * inv, a.gamma[c], a.beta[c]);
      a.y[base + c] = y;
      m = max(m, amax_key(y));
    }
  }
  amax_commit(a.am, m);
}
template <bool RES> __global__ void __launch_bounds__(kLongThreads) norm_long_bwd_kernel(const NormArgs a) {
  __shared__ float held[1][2][3][kLongThreads / 32];
  grid_dep_sync();
  RowSum<kLongThreads> add{held, 0};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  const int D = a.D;
  uint32_t m = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const float* const x = a.x + row * D;
    const float* const dy = a.dy + row * D;
    float sum[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += kLongThreads) sum[0] += x[c];
    add(sum);
    const float mean = sum[0] / (float)D;
    float three[3] = {0.f, 0.f, 0.f};
    for (int c = threadIdx.x; c < D; c += kLongThreads) {
      const float v = x[c] - mean, g = a.gamma[c] * dy[c];
      three[0] = fmaf(v, v, three[0]);
      three[1] += g;
      three[2] = fmaf(g, v, three[2]);
    }
    add(three);
    const float inv = __frsqrt_rn(three[0] / (float)D + a.eps);
    const float mean_g = three[1] / (float)D, mean_gx = three[2] * inv / (float)D;
    if (threadIdx.x == 0 && a.stats) a.stats[row] = make_float2(mean, inv);
    for (int c = threadIdx.x; c < D; c += kLongThreads) {
      float d = inv * (a.gamma[c] * dy[c] - mean_g - (x[c] - mean) * inv * mean_gx);
      if (RES && a.dsum) d += a.dsum[row * D + c];
      if (a.dx) {
        a.dx[row * D + c] = d;
        if (!RES || !a.dbranch) m = max(m, amax_key(d));
      }
      if (RES && a.dbranch) { d = dropped(a, mix_start(seed, row * D + c), d); a.dbranch[row * D + c] = d; m = max(m, amax_key(d)); }
    }
  }
  amax_commit(a.am, m);
}
// dgamma and dbeta of long rows: a thread per column, a share of the rows per blockIdx.y
__global__ void __launch_bounds__(256) norm_columns_kernel(const NormArgs a, int64_t per_block) {
  grid_dep_sync();
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.D) return;
  const int64_t r0 = blockIdx.y * per_block, r1 = min(a.rows, r0 + per_block);
  float dgamma = 0.f, dbeta = 0.f;
#pragma unroll 4
  for (int64_t r = r0; r < r1; ++r) {
    const float2 st = __ldg(a.stats + r);
    const float dy = __ldg(a.dy + r * a.D + c);
    dgamma = fmaf(dy, (__ldg(a.x + r * a.D + c) - st.x) * st.y, dgamma);
    dbeta += dy;
  }
  a.part[blockIdx.y * 2ll * a.D + c] = dgamma;
  a.part[blockIdx.y * 2ll * a.D + a.D + c] = dbeta;
}

// Adds the blocks' parts, in the order of the blocks: 32 columns a block, 32 runs of blocks.
__global__ void __launch_bounds__(1024) norm_params_kernel(const float* __restrict__ part, float* __restrict__ dgamma, float* __restrict__ dbeta, int blocks, int D) {
  __shared__ float held[32][33];
  grid_dep_sync();
  const int lane = threadIdx.x & 31, run = threadIdx.x >> 5;
  const int64_t c = (int64_t)blockIdx.x * 32 + lane;
  const int per_run = (blocks + 31) / 32, b0 = run * per_run, b1 = min(blocks, b0 + per_run);
  float sum = 0.f;
  if (c < 2ll * D) {
    for (int b = b0; b < b1; b += 8) {           // eight loads in flight
      float v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = b + i < b1 ? __ldg(part + (int64_t)(b + i) * 2 * D + c) : 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) sum += v[i];
    }
  }
  held[run][lane] = sum;
  __syncthreads();
  sum = held[lane][run];                       // 32 runs of column `run`
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  const int64_t out = (int64_t)blockIdx.x * 32 + run;
  if (lane == 0 && out < 2ll * D) {
    if (out < D) { if (dgamma) dgamma[out] = sum; }
    else if (dbeta) dbeta[out - D] = sum;
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
// Threads of a row, rows of a block (forward) and pieces of a row per thread: calls f with them as constants, or returns false where the
// row is too long for MOST threads.
template <int VEC, int MOST, class F> static bool with_shape(int D, F&& f) {
#define TF_NORM_SHAPE(G, R, E) if constexpr (G <= MOST) if (D <= G * E) { f(std::integral_constant<int, G>(), std::integral_constant<int, R>(), std::integral_constant<int, E / VEC>()); return true; }
  TF_NORM_SHAPE(32, 8, 4)
  TF_NORM_SHAPE(32, 8, 8)
  TF_NORM_SHAPE(32, 8, 12)
  TF_NORM_SHAPE(32, 8, 16)
  TF_NORM_SHAPE(64, 4, 12)
  TF_NORM_SHAPE(64, 4, 16)
  TF_NORM_SHAPE(128, 2, 12)
  TF_NORM_SHAPE(128, 2, 16)
  TF_NORM_SHAPE(256, 1, 12)
  TF_NORM_SHAPE(256, 1, 16)
  TF_NORM_SHAPE(512, 1, 12)
  TF_NORM_SHAPE(512, 1, 16)
  TF_NORM_SHAPE(1024, 1, 12)
  TF_NORM_SHAPE(1024, 1, 16)
#undef TF_NORM_SHAPE
  return false;
}
// Elements that one access takes: f(4), f(2) or f(1) as a constant
template <class F> static bool with_width(int D, std::initializer_list<const void*> all, F&& f) {
  uintptr_t bits = (uintptr_t)D * 4;
  for (const void* p : all) bits |= reinterpret_cast<uintptr_t>(p);         // a null pointer counts as aligned
  return bits % 16 == 0 ? f(std::integral_constant<int, 4>()) : bits % 8 == 0 ? f(std::integral_constant<int, 2>()) : f(std::integral_constant<int, 1>());
}
template <bool RES> static cudaError_t launch_norm_fwd(const NormArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  auto run = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    return with_shape<VEC, 1024>(a.D, [&](auto g, auto r, auto nv) {
      constexpr int G = decltype(g)::value, R = decltype(r)::value, NV = decltype(nv)::value;
      const int64_t blocks = (a.rows + R - 1) / R;
      e = launch_dep(norm_fwd_kernel<VEC, G, R, NV, RES>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(G * R), 0, s, a);
    });
  };
  if (!with_width(a.D, {a.x, a.residual, a.gamma, a.beta, a.sum, a.y}, run))
    e = launch_dep(norm_long_fwd_kernel<RES>, dim3((unsigned)std::min<int64_t>(a.rows, 4 * device_sm_count())), dim3(kLongThreads), 0, s, a);
  return e;
}
template <bool RES> static int run_norm_bwd(NormArgs a, float* dgamma, float* dbeta, int* memorytoSaving, cudaStream_t s, const char* what) {
  const bool sums = dgamma || dbeta;
  const float* const tracked = a.dbranch ? a.dbranch : a.dx;
  auto track = [&] { if (tracked && a.rows) a.am = amax_track_begin(tracked); };              // once nothing is short: a launch writes the word
  StreamLease lease(s);
  auto shortage = [&](size_t bytes) { if (memorytoSaving) *memorytoSaving = bytes > 0x7fffffffu ? 0x7fffffff : (int)bytes; return 0; };
  int blocks = 0, out_of_memory = 0;
  bool few = false;
  cudaError_t e = cudaSuccess;
  auto run = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    return with_shape<VEC, kBwdThreads>(a.D, [&](auto g, auto, auto nv) {
      constexpr int G = decltype(g)::value, NV = decltype(nv)::value;
      constexpr int kMost = kBwdThreads / G;           // groups of a block
      const int sms = device_sm_count(), stage = kMost * (int)norm_pitch<VEC, G, NV>() * (RES ? 3 : 2), depth = std::min(4, (kBwdSmem - G * NV * VEC * (int)sizeof(float)) / stage);
      static_assert(kMost * norm_pitch<VEC, G, NV>() * 3 * 2 + G * NV * VEC * 4 <= kBwdSmem, "two rows ahead and gamma always fit");
      // Up to two rows a group in one cluster: the sums of its blocks go through shared memory, and there is no second launch (64 x 256:
      // 4.3 us, 7.1 with one).
      // Else one block per SM, with as many groups as there are rows for.
      few = sums && a.rows > 0 && a.rows <= 2 * kFewBlocks * kMost;
      const int groups = few ? (int)std::min<int64_t>(kMost, (a.rows + kFewBlocks - 1) / kFewBlocks) : (int)std::max<int64_t>(1, std::min<int64_t>(kMost, (a.rows + sms - 1) / sms));
      blocks = (int)std::min<int64_t>((a.rows + groups - 1) / groups, few ? kFewBlocks : sms);
      const size_t bytes = sizeof(float) * 2 * (size_t)a.D * blocks, smem = (size_t)stage * depth + sizeof(float) * G * NV * VEC;
      if (few) { a.dgamma = dgamma; a.dbeta = dbeta; }
      else if (sums && blocks && !(a.part = (float*)lease.scratch(kScratchNorm, bytes))) { out_of_memory = 1; shortage(bytes); return; }
      static std::atomic<uint64_t> ready{0};
      const auto kernel = norm_bwd_kernel<VEC, G, NV, RES>;
      e = once_per_device(ready, [kernel] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBwdSmem); });
      if (!blocks || e != cudaSuccess) return;
      track();
      if (few) e = launch_cluster(norm_bwd_kernel<VEC, G, NV, RES>, blocks, dim3(blocks), dim3(groups * G), smem, s, a, depth);
      else e = launch_dep(norm_bwd_kernel<VEC, G, NV, RES>, dim3(blocks), dim3(groups * G), smem, s, a, depth);
    });
  };
  auto run_wide = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    auto launch = [&](auto elements) {
      constexpr int E = decltype(elements)::value;
      blocks = (int)std::min<int64_t>(a.rows, device_sm_count());
      const size_t bytes = sizeof(float) * 2 * (size_t)a.D * blocks, smem = sizeof(float) * 3 * E * kWideThreads;
      if (sums && blocks && !(a.part = (float*)lease.scratch(kScratchNorm, bytes))) { out_of_memory = 1; shortage(bytes); return; }
      static std::atomic<uint64_t> ready{0};
      const auto kernel = norm_wide_bwd_kernel<VEC, E / VEC, RES>;
      e = once_per_device(ready, [kernel] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBwdSmem); });
      if (!blocks || e != cudaSuccess) return;
      track();
      e = launch_dep(kernel, dim3(blocks), dim3(kWideThreads), smem, s, a);
    };
    if (a.D <= 12 * kWideThreads) launch(std::integral_constant<int, 12>());
    else if (a.D <= 16 * kWideThreads) launch(std::integral_constant<int, 16>());
    else return false;
    return true;
  };
  auto aligned = [&](auto&& f) { return with_width(a.D, {a.x, a.gamma, a.dy, a.dsum, a.dx, a.dbranch}, f); };
  if (!aligned(run) && !aligned(run_wide)) {
    const unsigned across = (unsigned)((a.D + 255) / 256);
    const int64_t shares = std::max<int64_t>(1, std::min<int64_t>(std::min<int64_t>(a.rows, 65535), 4 * device_sm_count() / across));
    const int64_t per_block = (a.rows + shares - 1) / shares;
    blocks = a.rows ? (int)((a.rows + per_block - 1) / per_block) : 0;
    const size_t part = sizeof(float) * 2 * (size_t)a.D * blocks, stats = sizeof(float2) * (size_t)a.rows;
    if (sums && blocks) {
      char* const scratch = (char*)lease.scratch(kScratchNorm, part + stats);
      if (!scratch) return shortage(part + stats);
      a.part = (float*)scratch; a.stats = (float2*)(scratch + part);
    }
    track();
    if (a.rows) e = launch_dep(norm_long_bwd_kernel<RES>, dim3((unsigned)std::min<int64_t>(a.rows, 4 * device_sm_count())), dim3(kLongThreads), 0, s, a);
    if (e == cudaSuccess && sums && blocks) {
      e = launch_dep(norm_columns_kernel, dim3(across, (unsigned)blocks), dim3(256), 0, s, a, per_block);
      TF_AFTER(s, what);
    }
  }
  if (out_of_memory) return 0;
  TF_CUDA(e);
  TF_AFTER(s, what);
  if (sums && !few) {
    TF_CUDA(launch_dep(norm_params_kernel, dim3((unsigned)((2ll * a.D + 31) / 32)), dim3(1024), 0, s, (const float*)a.part, dgamma, dbeta, blocks, a.D));
    TF_AFTER(s, what);
  }
  return 0;
}

}  // namespace tf

using namespace tf;

namespace {

int check_norm(const char* what, const DLArray* x, float eps, int64_t* rows, int* D) {
  TF_REQUIRE(x && x->ndim >= 1, "%s: the array to normalise needs an axis", what);
  const int64_t last = x->shape[x->ndim - 1], size = numel(x);
  TF_REQUIRE(size >= 0 && last >= 0 && last < (1ll << 30), "%s: rows of %lld elements", what, (long long)last);
  TF_REQUIRE(eps >= 0.f && eps < INFINITY, "%s: eps has to be finite and not negative", what);
  int64_t r = 1;
  for (int i = 0; i + 1 < x->ndim; ++i) r *= x->shape[i];
  *rows = r; *D = (int)last;
  return 0;
}
void set_dropout(NormArgs& a, const ResidualDropoutState* st) {
  a.p = st->p; a.scale = 1.f / (1.f - st->p); a.seed = st->seed;
  a.threshold = (uint32_t)ceil((double)st->p * 16777216.0) << 8;          // k * 2^-24 >= p is k >= p * 2^24, and a rate below one has 24 bits at most
}
float* opt_out(DLArrayHandle a) { return a ? out_f32(a) : nullptr; }

}  // namespace

extern "C" {

int TfLayerNormForward(const DLArrayHandle input, const DLArrayHandle gamma, const DLArrayHandle beta, DLArrayHandle output, float eps, void** cudaStream) {
  const char* const what = "TfLayerNormForward";
  NormArgs a;
  memset(&a, 0, sizeof(a));
  if (check_norm(what, input, eps, &a.rows, &a.D)) return -1;
  Operands o(what);
  o.add(input, "input", -1, false); o.add(gamma, "gamma", a.D, false); o.add(beta, "beta", a.D, false); o.add(output, "output", numel(input), true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.x = (const float*)input->data; a.gamma = (const float*)gamma->data; a.beta = (const float*)beta->data; a.y = out_f32(output); a.eps = eps;
  if (numel(input) == 0) return 0;
  a.am = amax_track_begin(a.y);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 8.0 * numel(input));
  TF_CUDA(launch_norm_fwd<false>(a, s));
  TF_AFTER(s, what);
  return 0;
}

int TfLayerNormBackward(const DLArrayHandle input, const DLArrayHandle gamma, const DLArrayHandle doutput, DLArrayHandle dinput, DLArrayHandle dgamma,
                        DLArrayHandle dbeta, float eps, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfLayerNormBackward";
  NormArgs a;
  memset(&a, 0, sizeof(a));
  if (check_norm(what, input, eps, &a.rows, &a.D)) return -1;
  Operands o(what);
  o.add(input, "input", -1, false); o.add(gamma, "gamma", a.D, false); o.add(doutput, "doutput", numel(input), false);
  o.add(dinput, "dinput", numel(input), true, true); o.add(dgamma, "dgamma", a.D, true, true); o.add(dbeta, "dbeta", a.D, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.x = (const float*)input->data; a.gamma = (const float*)gamma->data; a.dy = (const float*)doutput->data; a.eps = eps;
  a.dx = opt_out(dinput);
  float *dg = opt_out(dgamma), *db = opt_out(dbeta);
  if (a.D == 0 || !(a.dx || dg || db)) return 0;
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 12.0 * numel(input));
  return run_norm_bwd<false>(a, dg, db, memorytoSaving, s, what);
}

int TfDropoutState(float dropout, int seed, void*** state) {
  TF_REQUIRE(state, "TfDropoutState: null cell");
  TF_REQUIRE(dropout >= 0.f && dropout < 1.f, "TfDropoutState: rate must be in [0,1)");
  ResidualDropoutState* st = plan_of<ResidualDropoutState>(state, kPlanResidualDropout);
  TF_REQUIRE(st || !holds_plan(state), "TfDropoutState: the cell holds another descriptor");
  if (!st) st = new_plan<ResidualDropoutState>(state, kPlanResidualDropout, 1);
  st->p = dropout; st->seed = (unsigned long long)(unsigned)seed;
  return 0;
}

int TfDropoutAddLayerNormForward(const DLArrayHandle input, const DLArrayHandle residual, const DLArrayHandle gamma, const DLArrayHandle beta, DLArrayHandle sum,
                                 DLArrayHandle output, float eps, void*** state, void** cudaStream) {
  const char* const what = "TfDropoutAddLayerNormForward";
  NormArgs a;
  memset(&a, 0, sizeof(a));
  if (check_norm(what, input, eps, &a.rows, &a.D)) return -1;
  ResidualDropoutState* st = plan_of<ResidualDropoutState>(state, kPlanResidualDropout);
  TF_REQUIRE(st, "%s: the state was not made by TfDropoutState", what);
  const int64_t n = numel(input);
  Operands o(what);
  o.add(input, "input", -1, false); o.add(residual, "residual", n, false); o.add(gamma, "gamma", a.D, false); o.add(beta, "beta", a.D, false);
  o.add(sum, "sum", n, true); o.add(output, "output", n, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.x = (const float*)input->data; a.residual = (const float*)residual->data; a.gamma = (const float*)gamma->data; a.beta = (const float*)beta->data;
  a.sum = out_f32(sum); a.y = opt_out(output); a.eps = eps;
  st->seed_word = t_recording ? recording_seed((unsigned)st->seed) : nullptr;
  st->recording = recording_id();
  set_dropout(a, st); a.seed_word = st->seed_word;
  if (n == 0) return 0;
  if (a.y) a.am = amax_track_begin(a.y);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 16.0 * n);
  TF_CUDA(launch_norm_fwd<true>(a, s));
  TF_AFTER(s, what);
  return 0;
}

int TfDropoutAddLayerNormBackward(const DLArrayHandle sum, const DLArrayHandle gamma, const DLArrayHandle doutput, const DLArrayHandle dsum, DLArrayHandle dinput,
                                  DLArrayHandle dresidual, DLArrayHandle dgamma, DLArrayHandle dbeta, float eps, void*** state, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfDropoutAddLayerNormBackward";
  NormArgs a;
  memset(&a, 0, sizeof(a));
  if (check_norm(what, sum, eps, &a.rows, &a.D)) return -1;
  ResidualDropoutState* st = plan_of<ResidualDropoutState>(state, kPlanResidualDropout);
  TF_REQUIRE(st, "%s: the state was not made by TfDropoutState", what);
  const int64_t n = numel(sum);
  Operands o(what);
  o.add(sum, "sum", -1, false); o.add(gamma, "gamma", a.D, false); o.add(doutput, "doutput", n, false); o.add(dsum, "dsum", n, false, true);
  o.add(dinput, "dinput", n, true, true); o.add(dresidual, "dresidual", n, true, true); o.add(dgamma, "dgamma", a.D, true, true); o.add(dbeta, "dbeta", a.D, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.x = (const float*)sum->data; a.gamma = (const float*)gamma->data; a.dy = (const float*)doutput->data; a.dsum = dsum ? (const float*)dsum->data : nullptr; a.eps = eps;
  a.dx = opt_out(dresidual); a.dbranch = opt_out(dinput);
  float *dg = opt_out(dgamma), *db = opt_out(dbeta);
  set_dropout(a, st);
  a.seed_word = st->recording && st->recording == recording_id() ? st->seed_word : nullptr;
  if (a.D == 0 || !(a.dx || a.dbranch || dg || db)) return 0;
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 20.0 * n);
  return run_norm_bwd<true>(a, dg, db, memorytoSaving, s, what);
}

}  // extern "C"
