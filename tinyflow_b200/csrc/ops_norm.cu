// Layer normalisation over the last axis, alone and behind the residual sum of a dropped-out branch, forward and backward.
//
//   s = residual + keep * branch / (1 - p)                    (the second form only; without it s is the input)
//   y = gamma * xh + beta,  xh = (s - mean) * inv,  inv = (mean((s - mean)^2) + eps)^(-1/2)
//   g = gamma * dy,  ds = inv * (g - mean(g) - xh * mean(g * xh)) [+ the gradient that reaches s behind the block]
//   dgamma = sum over rows of dy * xh,  dbeta = sum over rows of dy,  dbranch = keep * ds / (1 - p)
//
// HBM-bound: every tensor is read once and written once.  A row stays in the registers of one group of threads, so the mean is
// known before the squares are summed (no cancellation, whatever the offset) and the backward pass forms the statistics again
// instead of reading them.  keep is drawn from (seed, element index) again, nothing of it is stored.
#include "common.h"
#include <math.h>
#include <algorithm>
#include <initializer_list>
#include <type_traits>
#include "operands.h"

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
  float2* stats;             // per row: mean and inv (rows that do not fit the registers)
  int64_t rows;
  int D;
  float eps, p, scale;
  unsigned long long seed;
  const uint32_t* seed_word;
  AmaxOut am;
};

template <int VEC> struct Pieces;
template <> struct Pieces<4> { typedef float4 T; };
template <> struct Pieces<1> { typedef float T; };
template <int VEC> __device__ __forceinline__ void get(float* v, const float* __restrict__ p) { *reinterpret_cast<typename Pieces<VEC>::T*>(v) = __ldg(reinterpret_cast<const typename Pieces<VEC>::T*>(p)); }
template <int VEC> __device__ __forceinline__ void put(float* p, const float* v) { *reinterpret_cast<typename Pieces<VEC>::T*>(p) = *reinterpret_cast<const typename Pieces<VEC>::T*>(v); }

// Sums over the G threads that share a row, the same in all of them.  Two buffers in turn: a thread that writes one for the next sum
// has passed the barrier behind which every thread had read the one before.
template <int G, int R> struct RowSum {
  static constexpr int kWarps = G / 32;
  float (*held)[2][3][kWarps];
  int group, turn = 0;
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
    if (R == 1) __syncthreads();
    else asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "r"(G) : "memory");
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
__device__ __forceinline__ float dropped(const NormArgs& a, unsigned long long seed, int64_t i, float v) {
  return a.p == 0.f || uniform01(seed, (unsigned long long)i) >= a.p ? v * a.scale : 0.f;
}

// R groups of G threads, a row each, NV * VEC elements of it per thread.
template <int VEC, int G, int R, int NV, bool RES>
__global__ void __launch_bounds__(G * R) norm_fwd_kernel(const NormArgs a) {
  __shared__ float held[R][2][3][G / 32];
  grid_dep_sync();
  const int t = threadIdx.x % G, group = threadIdx.x / G, D = a.D;
  RowSum<G, R> add{held, group};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  uint32_t m = 0;
  for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.rows; row += (int64_t)gridDim.x * R) {
    const int64_t base = row * D;
    float x[NV][VEC];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) get<VEC>(x[v], a.x + base + c);
      else
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[v][j] = 0.f;
    }
    if (RES) {
      float r[NV][VEC];
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * G + t) * VEC;
        if (c < D) get<VEC>(r[v], a.residual + base + c);
      }
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = (v * G + t) * VEC;
        if (c < D) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) x[v][j] = r[v][j] + dropped(a, seed, base + c + j, x[v][j]);
          put<VEC>(a.sum + base + c, x[v]);
        }
      }
      if (!a.y) continue;
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0] += x[v][j];
    add(sum);
    const float mean = sum[0] / (float)D;
    float squares[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const bool there = (v * G + t) * VEC < D;
#pragma unroll
      for (int j = 0; j < VEC; ++j) { x[v][j] = there ? x[v][j] - mean : 0.f; squares[0] = fmaf(x[v][j], x[v][j], squares[0]); }
    }
    add(squares);
    const float inv = __frsqrt_rn(squares[0] / (float)D + a.eps);
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) {
        float w[VEC], b[VEC];
        get<VEC>(w, a.gamma + c);
        get<VEC>(b, a.beta + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) { b[j] = fmaf(x[v][j] * inv, w[j], b[j]); m = max(m, amax_bits(b[j])); }
        put<VEC>(a.y + base + c, b);
      }
    }
  }
  amax_commit(a.am, m);
}

// Persistent: a group takes every (grid * R)-th row, so a thread always has the same columns and keeps their parts of dgamma and dbeta
// in registers; the groups' parts are added in group order and left as one row of `part` per block.
template <int VEC, int G, int R, int NV, bool RES>
__global__ void __launch_bounds__(G * R) norm_bwd_kernel(const NormArgs a) {
  __shared__ float held[R][2][3][G / 32];
  extern __shared__ float sums[];              // [2 * D], with more than one group
  grid_dep_sync();
  const int t = threadIdx.x % G, group = threadIdx.x / G, D = a.D;
  RowSum<G, R> add{held, group};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  uint32_t m = 0;
  float dgamma[NV][VEC], dbeta[NV][VEC];
#pragma unroll
  for (int v = 0; v < NV; ++v)
#pragma unroll
    for (int j = 0; j < VEC; ++j) dgamma[v][j] = dbeta[v][j] = 0.f;
  for (int64_t row = (int64_t)blockIdx.x * R + group; row < a.rows; row += (int64_t)gridDim.x * R) {
    const int64_t base = row * D;
    float x[NV][VEC], dy[NV][VEC];
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) { get<VEC>(x[v], a.x + base + c); get<VEC>(dy[v], a.dy + base + c); }
      else
#pragma unroll
        for (int j = 0; j < VEC; ++j) x[v][j] = dy[v][j] = 0.f;
    }
    float sum[1] = {0.f};
#pragma unroll
    for (int v = 0; v < NV; ++v)
#pragma unroll
      for (int j = 0; j < VEC; ++j) sum[0] += x[v][j];
    add(sum);
    const float mean = sum[0] / (float)D;
    float three[3] = {0.f, 0.f, 0.f};          // (x - mean)^2, g, g * (x - mean)
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) {
        float w[VEC];
        get<VEC>(w, a.gamma + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[v][j] -= mean;
          const float g = w[j] * dy[v][j];
          three[0] = fmaf(x[v][j], x[v][j], three[0]);
          three[1] += g;
          three[2] = fmaf(g, x[v][j], three[2]);
        }
      }
    }
    add(three);
    const float inv = __frsqrt_rn(three[0] / (float)D + a.eps);
    const float mean_g = three[1] / (float)D, mean_gx = three[2] * inv / (float)D;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) {
        float w[VEC], ds[VEC];
        get<VEC>(w, a.gamma + c);
        if (RES && a.dsum) get<VEC>(ds, a.dsum + base + c);
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          const float xh = x[v][j] * inv;
          dgamma[v][j] = fmaf(dy[v][j], xh, dgamma[v][j]);
          dbeta[v][j] += dy[v][j];
          const float d = inv * (w[j] * dy[v][j] - mean_g - xh * mean_gx);
          ds[j] = RES && a.dsum ? ds[j] + d : d;
        }
        if (a.dx) {
          put<VEC>(a.dx + base + c, ds);
          if (!RES || !a.dbranch)
#pragma unroll
            for (int j = 0; j < VEC; ++j) m = max(m, amax_bits(ds[j]));
        }
        if (RES && a.dbranch) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) { ds[j] = dropped(a, seed, base + c + j, ds[j]); m = max(m, amax_bits(ds[j])); }
          put<VEC>(a.dbranch + base + c, ds);
        }
      }
    }
  }
  amax_commit(a.am, m);
  if (!a.part) return;
  float* const out = a.part + (int64_t)blockIdx.x * 2 * D;
#pragma unroll 1
  for (int r = 0; r < R; ++r) {
    if (R > 1) __syncthreads();
    if (group != r) continue;
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = (v * G + t) * VEC;
      if (c < D) {
        if (r) {
#pragma unroll
          for (int j = 0; j < VEC; ++j) { dgamma[v][j] += sums[c + j]; dbeta[v][j] += sums[D + c + j]; }
        }
        float* const to = R > 1 && r + 1 < R ? sums : out;
#pragma unroll
        for (int j = 0; j < VEC; ++j) { to[c + j] = dgamma[v][j]; to[D + c + j] = dbeta[v][j]; }
      }
    }
  }
}

// Rows of any length, a block each: three passes over the row, which L1 and L2 hold from the second on.
constexpr int kLongThreads = 512;
template <bool RES> __global__ void __launch_bounds__(kLongThreads) norm_long_fwd_kernel(const NormArgs a) {
  __shared__ float held[1][2][3][kLongThreads / 32];
  grid_dep_sync();
  RowSum<kLongThreads, 1> add{held, 0};
  const unsigned long long seed = RES ? seed_of(a) : 0;
  const int D = a.D;
  uint32_t m = 0;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t base = row * D;
    const float* const x = RES ? a.sum + base : a.x + base;            // a thread reads what it wrote itself
    float sum[1] = {0.f};
    for (int c = threadIdx.x; c < D; c += kLongThreads) {
      float v = a.x[base + c];
      if (RES) { v = a.residual[base + c] + dropped(a, seed, base + c, v); a.sum[base + c] = v; }
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
      m = max(m, amax_bits(y));
    }
  }
  amax_commit(a.am, m);
}
template <bool RES> __global__ void __launch_bounds__(kLongThreads) norm_long_bwd_kernel(const NormArgs a) {
  __shared__ float held[1][2][3][kLongThreads / 32];
  grid_dep_sync();
  RowSum<kLongThreads, 1> add{held, 0};
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
        if (!RES || !a.dbranch) m = max(m, amax_bits(d));
      }
      if (RES && a.dbranch) { d = dropped(a, seed, row * D + c, d); a.dbranch[row * D + c] = d; m = max(m, amax_bits(d)); }
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
#pragma unroll 8
    for (int b = b0; b < b1; ++b) sum += __ldg(part + (int64_t)b * 2 * D + c);
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
// Threads of a row and elements of it per thread; calls f(G, R, NV as constants), or returns false where the row is too long.
template <int VEC, int MOST, class F> static bool with_shape(int D, F&& f) {
#define TF_NORM_SHAPE(G, R, E) if constexpr (E <= MOST) if (D <= G * E) { f(std::integral_constant<int, G>(), std::integral_constant<int, R>(), std::integral_constant<int, E / VEC>()); return true; }
  TF_NORM_SHAPE(32, 8, 4)
  TF_NORM_SHAPE(32, 8, 8)
  TF_NORM_SHAPE(32, 8, 16)
  TF_NORM_SHAPE(64, 4, 16)
  TF_NORM_SHAPE(128, 2, 16)
  TF_NORM_SHAPE(256, 1, 16)
  TF_NORM_SHAPE(512, 1, 16)
  TF_NORM_SHAPE(512, 1, 32)
#undef TF_NORM_SHAPE
  return false;
}
static bool vectors(int D, std::initializer_list<const void*> all) {
  if (D % 4) return false;
  for (const void* p : all) if (!aligned16(p)) return false;         // a null pointer counts as aligned
  return true;
}
template <bool RES> static cudaError_t launch_norm_fwd(const NormArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  auto run = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    return with_shape<VEC, 32>(a.D, [&](auto g, auto r, auto nv) {
      constexpr int G = decltype(g)::value, R = decltype(r)::value, NV = decltype(nv)::value;
      const int64_t blocks = (a.rows + R - 1) / R;
      e = launch_dep(norm_fwd_kernel<VEC, G, R, NV, RES>, dim3((unsigned)std::min<int64_t>(blocks, 1 << 20)), dim3(G * R), 0, s, a);
    });
  };
  const bool vec = vectors(a.D, {a.x, a.residual, a.gamma, a.beta, a.sum, a.y});
  if (!(vec ? run(std::integral_constant<int, 4>()) : run(std::integral_constant<int, 1>())))
    e = launch_dep(norm_long_fwd_kernel<RES>, dim3((unsigned)std::min<int64_t>(a.rows, 4 * device_sm_count())), dim3(kLongThreads), 0, s, a);
  return e;
}
constexpr int kBwdRegs = 16;             // elements per thread of the backward kernel
static int norm_bwd_blocks(int64_t rows, int R, int threads) {
  return (int)std::min<int64_t>((rows + R - 1) / R, (int64_t)device_sm_count() * std::max(1, 512 / threads));
}
template <bool RES> static int run_norm_bwd(NormArgs a, float* dgamma, float* dbeta, int* memorytoSaving, cudaStream_t s, const char* what) {
  const bool sums = dgamma || dbeta;
  StreamLease lease(s);
  auto shortage = [&](size_t bytes) { if (memorytoSaving) *memorytoSaving = bytes > 0x7fffffffu ? 0x7fffffff : (int)bytes; return 0; };
  int blocks = 0, out_of_memory = 0;
  cudaError_t e = cudaSuccess;
  auto run = [&](auto vec) {
    constexpr int VEC = decltype(vec)::value;
    return with_shape<VEC, kBwdRegs>(a.D, [&](auto g, auto r, auto nv) {
      constexpr int G = decltype(g)::value, R = decltype(r)::value, NV = decltype(nv)::value;
      blocks = norm_bwd_blocks(a.rows, R, G * R);
      const size_t bytes = sizeof(float) * 2 * (size_t)a.D * blocks;
      if (sums && blocks && !(a.part = (float*)lease.scratch(kScratchNorm, bytes))) { out_of_memory = 1; shortage(bytes); return; }
      if (blocks) e = launch_dep(norm_bwd_kernel<VEC, G, R, NV, RES>, dim3(blocks), dim3(G * R), R > 1 && sums ? sizeof(float) * 2 * a.D : 0, s, a);
    });
  };
  const bool vec = vectors(a.D, {a.x, a.gamma, a.dy, a.dsum, a.dx, a.dbranch});
  if (!(vec ? run(std::integral_constant<int, 4>()) : run(std::integral_constant<int, 1>()))) {
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
    if (a.rows) e = launch_dep(norm_long_bwd_kernel<RES>, dim3((unsigned)std::min<int64_t>(a.rows, 4 * device_sm_count())), dim3(kLongThreads), 0, s, a);
    if (e == cudaSuccess && sums && blocks) {
      e = launch_dep(norm_columns_kernel, dim3(across, (unsigned)blocks), dim3(256), 0, s, a, per_block);
      TF_AFTER(s, what);
    }
  }
  if (out_of_memory) return 0;
  TF_CUDA(e);
  TF_AFTER(s, what);
  if (sums) {
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
  if (a.dx && a.rows) a.am = amax_track_begin(a.dx);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 12.0 * numel(input));
  return run_norm_bwd<false>(a, dg, db, memorytoSaving, s, what);
}

int TfDropoutState(float dropout, int seed, void*** state) {
  TF_REQUIRE(state, "TfDropoutState: null cell");
  TF_REQUIRE(dropout >= 0.f && dropout < 1.f, "TfDropoutState: rate must be in [0,1)");
  ResidualDropoutState* st = plan_of<ResidualDropoutState>(state, kPlanResidualDropout);
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
  a.p = st->p; a.scale = 1.f / (1.f - st->p); a.seed = st->seed; a.seed_word = st->seed_word;
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
  a.p = st->p; a.scale = 1.f / (1.f - st->p); a.seed = st->seed;
  a.seed_word = st->recording && st->recording == recording_id() ? st->seed_word : nullptr;
  if (a.D == 0 || !(a.dx || a.dbranch || dg || db)) return 0;
  if (a.rows && (a.dx || a.dbranch)) a.am = amax_track_begin(a.dbranch ? a.dbranch : a.dx);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 20.0 * n);
  return run_norm_bwd<true>(a, dg, db, memorytoSaving, s, what);
}

}  // extern "C"
