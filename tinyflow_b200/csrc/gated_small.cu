// Gated dense layers of the sizes that the tensor path is too long a road for, in exact fp32: one launch forward, one backward.
//
// Latency is the bound (launches, and one chain of loads and sums per block), so everything that can be formed on the way is: the forward
// kernel computes the gate columns and the value columns that they meet in the same block and finishes them; the backward kernel holds the
// tiles of dx and of dW, and forms dz from the projections while it loads, once per tile that reads it.  Long reductions are cut over the
// CTAs of a cluster and added in rank order through distributed shared memory, as in the plain products.
// 64 x 784 x 256, forward and backward: products and elementwise kernels one by one 30 us, so 20.4.
#include "common.h"
#include <algorithm>
#include <type_traits>
#include <cooperative_groups.h>
#include "gated.h"
#include "simt.h"

namespace cg = cooperative_groups;

namespace tf {

namespace {

constexpr int kTile = 32, kDepth = 32, kThreads = 128, kPitch = kTile + 4;
struct Small {
  const float *x, *w, *z, *dout;
  float *gates, *out, *dx, *dw;
  int M, K, F;
  int per_cta;              // of the reduction that is cut (forward: K, a multiple of 32; dx: F, a multiple of 16)
  int rows_per_cta;         // dW: of the batch, a multiple of 32
  int dx_ranks, dw_ranks;   // CTAs of a cluster that share a tile: 1 up to its size
  int dx_clusters;          // the first so many, the others are dW's
  int x_vec, w_vec, z_vec;  // 16-byte accesses allowed
  int dx_tiles, dw_tiles, dx_across, dw_across;
  AmaxOut am;
};

typedef float Block[kDepth][kPitch];
// thread (ty, tx) of 8 x 16: 4 rows x 2 columns
__device__ __forceinline__ void multiply(const Block& a, const Block& b, int ty, int tx, float (&acc)[4][2]) {
#pragma unroll
  for (int k = 0; k < kDepth; ++k) {
    const float4 r = *reinterpret_cast<const float4*>(&a[k][ty * 4]);
    const float2 c = *reinterpret_cast<const float2*>(&b[k][tx * 2]);
    acc[0][0] = fmaf(r.x, c.x, acc[0][0]); acc[0][1] = fmaf(r.x, c.y, acc[0][1]);
    acc[1][0] = fmaf(r.y, c.x, acc[1][0]); acc[1][1] = fmaf(r.y, c.y, acc[1][1]);
    acc[2][0] = fmaf(r.z, c.x, acc[2][0]); acc[2][1] = fmaf(r.z, c.y, acc[2][1]);
    acc[3][0] = fmaf(r.w, c.x, acc[3][0]); acc[3][1] = fmaf(r.w, c.y, acc[3][1]);
  }
}
// (16 CTAs are more than every GPU's clusters may have; this one's may)
constexpr int kMostRanks = 16;
// Stores a tile: straight from the registers, or the sum over `ranks` CTAs of the cluster from `first` on, in order, each a slice of it
template <class Store> __device__ __forceinline__ void finish_tile(int ranks, int first, float* part, const float (&acc)[4][2], int ty, int tx, Store&& store) {
  if (ranks == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) store(ty * 4 + i, tx * 2 + j, acc[i][j]);
    return;
  }
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank() - first;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) part[(ty * 4 + i) * kTile + tx * 2 + j] = acc[i][j];
  cluster.sync();
  const int slice = (kTile * kTile + ranks - 1) / ranks, end = min(kTile * kTile, (rank + 1) * slice);
  for (int e = rank * slice + threadIdx.x; e < end; e += kThreads) {
    float a[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) a[r] = cluster.map_shared_rank(part, first + min(r, ranks - 1))[e];
    float total = a[0];
#pragma unroll
    for (int r = 1; r < 8; ++r) if (r < ranks) total += a[r];
    for (int r = 8; r < ranks; ++r) total += cluster.map_shared_rank(part, first + r)[e];
    store(e / kTile, e % kTile, total);
  }
  cluster.sync();           // nobody leaves while its shared memory is still read
}
// four elements of a row from column c on, zeros from `cols` on
__device__ __forceinline__ float4 four(const float* __restrict__ row, int c, int cols, bool vec) {
  if (vec && c + 4 <= cols) return __ldg(reinterpret_cast<const float4*>(row + c));
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (c < cols) v.x = __ldg(row + c);
  if (c + 1 < cols) v.y = __ldg(row + c + 1);
  if (c + 2 < cols) v.z = __ldg(row + c + 2);
  if (c + 3 < cols) v.w = __ldg(row + c + 3);
  return v;
}
// dz of four columns of one row: loaded, then formed
template <int ACT> struct GateGradient {
  float4 g, v, d;
  __device__ __forceinline__ void fetch(const Small& p, int m, int f) {
    g = v = d = make_float4(0.f, 0.f, 0.f, 0.f);
    if (m >= p.M) return;
    const float* const z = p.z + (long long)m * 2 * p.F;
    g = four(z, f, p.F, p.z_vec);
    v = four(z + p.F, f, p.F, p.z_vec);
    d = four(p.dout + (long long)m * p.F, f, p.F, p.z_vec);            // zeros past the end: so is dz
  }
  __device__ __forceinline__ void form(float (&dg)[4], float (&dv)[4]) const {
    const float gg[4] = {g.x, g.y, g.z, g.w}, vv[4] = {v.x, v.y, v.z, v.w}, dd[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float value, slope;
      gate_slope<ACT>(gg[i], value, slope);
      dg[i] = dd[i] * vv[i] * slope;
      dv[i] = dd[i] * value;
    }
  }
};

// grid (ranks * ceil(F / 32), ceil(M / 32)), clusters of `ranks` along x.  Steps of 32 of K come by asynchronous copies, kAhead of them in
// flight: a CTA of a cut reduction has them all under way at once.
constexpr int kAhead = 4;
struct FwdStep { float x[kTile][kPitch]; float g[kDepth][kTile], v[kDepth][kTile]; };      // x by rows, 16-byte aligned ones
template <int ACT> __global__ void __launch_bounds__(kThreads) gated_small_fwd_kernel(const Small p) {
  extern __shared__ __align__(16) unsigned char small_smem[];
  FwdStep* const ring = reinterpret_cast<FwdStep*>(small_smem);
  cg::cluster_group cluster = cg::this_cluster();
  const int rank = (int)cluster.block_rank(), ranks = (int)cluster.num_blocks();
  grid_dep_sync();
  const int m0 = blockIdx.y * kTile, f0 = (int)(blockIdx.x / ranks) * kTile, tx = threadIdx.x % 16, ty = threadIdx.x / 16;
  const int kbeg = rank * p.per_cta, kend = min(p.K, kbeg + p.per_cta), steps = max(0, (kend - kbeg + kDepth - 1) / kDepth);
  float g[4][2] = {}, v[4][2] = {};
  // `there` of the four elements at `from`, zeros for the rest
  auto copy4 = [](float* to, const float* from, int there, bool vec) {
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(to);
    if (vec) {
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(from), "r"(max(0, min(4, there)) * 4) : "memory");
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i)
        asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst + 4 * i), "l"(i < there ? from + i : from), "r"(i < there ? 4 : 0) : "memory");
    }
  };
  auto fetch = [&](int step) {
    if (step < steps) {
      FwdStep& st = ring[step % kAhead];
      const int k0 = kbeg + step * kDepth;
#pragma unroll
      for (int i = 0; i < kTile * kDepth / 4 / kThreads; ++i) {
        const int e = threadIdx.x + i * kThreads, line = e / 8, quad = e % 8 * 4;
        const bool row = m0 + line < p.M, deep = k0 + line < kend;
        const int xs = row ? kend - k0 - quad : 0, ws = deep ? p.F - f0 - quad : 0;
        copy4(&st.x[line][quad], xs > 0 ? p.x + (long long)(m0 + line) * p.K + k0 + quad : p.x, xs, p.x_vec);
        const float* const w = ws > 0 ? p.w + (long long)(k0 + line) * 2 * p.F + f0 + quad : p.w;
        copy4(&st.g[line][quad], w, ws, p.w_vec);
        copy4(&st.v[line][quad], ws > 0 ? w + p.F : p.w, ws, p.w_vec);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAhead; ++i) fetch(i);
  for (int step = 0; step < steps; ++step) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    __syncthreads();
    const FwdStep& st = ring[step % kAhead];
#pragma unroll
    for (int k = 0; k < kDepth; k += 4) {
      float x[4][4];
#pragma unroll
      for (int i = 0; i < 4; ++i) *reinterpret_cast<float4*>(x[i]) = *reinterpret_cast<const float4*>(&st.x[ty * 4 + i][k]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float2 a = *reinterpret_cast<const float2*>(&st.g[k + j][tx * 2]), b = *reinterpret_cast<const float2*>(&st.v[k + j][tx * 2]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          g[i][0] = fmaf(x[i][j], a.x, g[i][0]); g[i][1] = fmaf(x[i][j], a.y, g[i][1]);
          v[i][0] = fmaf(x[i][j], b.x, v[i][0]); v[i][1] = fmaf(x[i][j], b.y, v[i][1]);
        }
      }
    }
    if (step + kAhead < steps) __syncthreads();                // nobody reads what comes next into its place
    fetch(step + kAhead);
  }
  __syncthreads();
  uint32_t top = 0;
  auto finish = [&](int row, int col, float gate, float value) {
    const int m = m0 + row, f = f0 + col;
    if (m >= p.M || f >= p.F) return;
    if (p.gates) { p.gates[(long long)m * 2 * p.F + f] = gate; p.gates[(long long)m * 2 * p.F + p.F + f] = value; }
    value *= gate_value<ACT, false>(gate);
    p.out[(long long)m * p.F + f] = value;
    top = max(top, amax_key(value));
  };
  if (ranks == 1) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) finish(ty * 4 + i, tx * 2 + j, g[i][j], v[i][j]);
  } else {
    float* const part = reinterpret_cast<float*>(small_smem);            // gates, then values, 32 x 32 each, where the first step was
    static_assert(sizeof(FwdStep) >= 2 * kTile * kTile * sizeof(float), "a tile's partial sums fit there");
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j) { part[(ty * 4 + i) * kTile + tx * 2 + j] = g[i][j]; part[kTile * kTile + (ty * 4 + i) * kTile + tx * 2 + j] = v[i][j]; }
    cluster.sync();
    const int slice = (kTile * kTile + ranks - 1) / ranks, end = min(kTile * kTile, (rank + 1) * slice);
    for (int e = rank * slice + threadIdx.x; e < end; e += kThreads) {
      float a[8], b[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        const float* const from = cluster.map_shared_rank(part, min(r, ranks - 1));
        a[r] = from[e]; b[r] = from[kTile * kTile + e];
      }
      float gate = a[0], value = b[0];
#pragma unroll
      for (int r = 1; r < 8; ++r) if (r < ranks) { gate += a[r]; value += b[r]; }
      finish(e / kTile, e % kTile, gate, value);
    }
    cluster.sync();           // nobody leaves while its shared memory is still read
  }
  amax_commit(p.am, top);
}

// dx: cut over the columns; dW: cut over the rows of the batch where they are long and the weights few.
// A step of 32 of the reduction is 16 columns of each half for dx, 32 rows for dW; a tile of dW is 32 rows x 16 columns of each half.
// Five CTAs an SM with two steps' loads in flight; four with four steps' are faster where gradients follow gradients, slower where they follow the
// forward call (256 x 256 x 256: 12.2 us against 14.0 alone, a step of both 23.3 against 19.9; 14 sizes on average 7 % and 5 %).
constexpr int kLoads = 2;           // steps of dx whose loads are in flight at once
template <int ACT> __global__ void __launch_bounds__(kThreads, 5) gated_small_bwd_kernel(const Small p) {
  __shared__ __align__(16) Block as[2], bs[2];
  cg::cluster_group cluster = cg::this_cluster();
  const int size = (int)cluster.num_blocks(), at_rank = (int)cluster.block_rank(), id = (int)blockIdx.x / size;
  grid_dep_sync();
  const bool for_dx = id < p.dx_clusters;
  const int ranks = for_dx ? p.dx_ranks : p.dw_ranks, rank = at_rank % ranks, first = at_rank - rank;
  const int tile = (for_dx ? id : id - p.dx_clusters) * (size / ranks) + at_rank / ranks;
  if (tile >= (for_dx ? p.dx_tiles : p.dw_tiles)) {
    if (ranks > 1) { cluster.sync(); cluster.sync(); }             // those of the tiles that are cut
    return;
  }
  const int tx = threadIdx.x % 16, ty = threadIdx.x / 16, line = threadIdx.x / 4, quad = threadIdx.x % 4 * 4;
  float acc[4][2] = {};
  GateGradient<ACT> dz[kLoads];
  if (for_dx) {
    const int m0 = tile / p.dx_across * kTile, n0 = tile % p.dx_across * kTile, fbeg = rank * p.per_cta, fend = min(p.F, fbeg + p.per_cta);
    float4 wg[kLoads], wv[kLoads];
    auto fetch = [&](int f, int at) {
      dz[at].fetch(p, f < fend ? m0 + line : p.M, f + quad);
      wg[at] = wv[at] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (n0 + line < p.K && f < fend) {
        const float* const row = p.w + (long long)(n0 + line) * 2 * p.F;
        wg[at] = four(row, f + quad, p.F, p.w_vec);
        wv[at] = four(row + p.F, f + quad, p.F, p.w_vec);
      }
    };
    auto put = [&](int at, int to) {
      float dg[4], dv[4];
      dz[at].form(dg, dv);
      const float g[4] = {wg[at].x, wg[at].y, wg[at].z, wg[at].w}, v[4] = {wv[at].x, wv[at].y, wv[at].z, wv[at].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        as[to][quad + i][line] = dg[i]; as[to][16 + quad + i][line] = dv[i];
        bs[to][quad + i][line] = g[i]; bs[to][16 + quad + i][line] = v[i];
      }
    };
    for (int f = fbeg; f < fend; f += kLoads * 16) {
#pragma unroll
      for (int at = 0; at < kLoads; ++at) fetch(f + at * 16, at);
#pragma unroll
      for (int at = 0; at < kLoads; ++at) {
        if (f + at * 16 < fend) {                // the same for the whole block
          put(at, at & 1);
          __syncthreads();
          multiply(as[at & 1], bs[at & 1], ty, tx, acc);
        }
      }
      __syncthreads();
    }
    finish_tile(ranks, first, &as[0][0][0], acc, ty, tx, [&](int row, int col, float v) {
      if (m0 + row < p.M && n0 + col < p.K) p.dx[(long long)(m0 + row) * p.K + n0 + col] = v;
    });
    return;
  }
  const int k0 = tile / p.dw_across * kTile, f0 = tile % p.dw_across * 16;
  const int mbeg = rank * p.rows_per_cta, mend = min(p.M, mbeg + p.rows_per_cta);
  BlockLoader<kTile, kDepth, kThreads, false> lx[2];
  auto fetch = [&](int m, int at) {
    lx[at].fetch(p.x, p.K, k0, p.K, m, mend, p.x_vec);
    dz[at].fetch(p, m + line < mend ? m + line : p.M, f0 + quad);
  };
  auto put = [&](int at) {
    float dg[4], dv[4];
    lx[at].put(as[at]);
    dz[at].form(dg, dv);
    *reinterpret_cast<float4*>(&bs[at][line][quad]) = make_float4(dg[0], dg[1], dg[2], dg[3]);
    *reinterpret_cast<float4*>(&bs[at][line][16 + quad]) = make_float4(dv[0], dv[1], dv[2], dv[3]);
  };
  if (mbeg < mend) { fetch(mbeg, 0); fetch(mbeg + kDepth, 1); }
  for (int m = mbeg; m < mend; m += 2 * kDepth) {
#pragma unroll
    for (int at = 0; at < 2; ++at) {
      if (m + at * kDepth < mend) {              // the same for the whole block
        put(at);
        __syncthreads();
        fetch(m + (at + 2) * kDepth, at);
        multiply(as[at], bs[at], ty, tx, acc);
      }
    }
  }
  __syncthreads();
  finish_tile(ranks, first, &as[0][0][0], acc, ty, tx, [&](int row, int col, float v) {
    const int k = k0 + row, f = f0 + (col & 15);
    if (k < p.K && f < p.F) p.dw[(long long)k * 2 * p.F + (col < 16 ? 0 : p.F) + f] = v;
  });
}

// Blocks of 64 x 64 would leave SMs idle: above that the plain products with their larger tiles are faster (backward, where dz is formed again for
// every tile: 100 x 2000 x 500 73 us against 52)
bool small_product(int64_t M, int64_t N) { return ((M + 63) / 64) * ((N + 63) / 64) < device_sm_count(); }
int cluster_for(long long tiles, long long steps, int want, int most) {
  int c = 1;
  while (c < most && tiles * c < want && steps >= 4 * c) c *= 2;
  return c;
}

}  // namespace

// 1: done, 0: too large, -1: error
int gated_small_fwd(const float* x, const float* w, float* gates, float* out, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s, const char* what) {
  if (2.0 * M * F * K > 5e8) return 0;               // 64 x 64 tiles of the plain products (8000 x 64 x 64: 8.3 us against 18.1; 512 x 512 x 512: 24.6 for both)
  if (M > 65535ll * kTile) return 0;                 // the grid's rows
  Small p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.w = w; p.gates = gates; p.out = out; p.M = (int)M; p.K = (int)K; p.F = (int)F;
  p.x_vec = K % 4 == 0 && aligned16(x); p.w_vec = F % 4 == 0 && aligned16(w);
  const unsigned across = (unsigned)((F + kTile - 1) / kTile), down = (unsigned)((M + kTile - 1) / kTile);
  const int cluster = cluster_for((long long)across * down, (K + kDepth - 1) / kDepth, 3 * device_sm_count(), 8);
  p.per_cta = (int)(((K + cluster - 1) / cluster + kDepth - 1) / kDepth * kDepth);
  p.am = amax_track_begin(out);
  note_compute_stream(s);
  KernelTimer kt("gated_small_fwd", s, 4.0 * M * F * K, 0, 1);
  cudaError_t e = cudaSuccess;
  with_gate(activation, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    static std::atomic<uint64_t> ready{0};
    e = once_per_device(ready, [] {
      const cudaError_t set = cudaFuncSetAttribute(gated_small_fwd_kernel<ACT>, cudaFuncAttributeMaxDynamicSharedMemorySize, sizeof(FwdStep) * kAhead);
      return set != cudaSuccess ? set : cudaFuncSetAttribute(gated_small_fwd_kernel<ACT>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    });
    if (e == cudaSuccess) e = cluster > 1 ? launch_cluster(gated_small_fwd_kernel<ACT>, cluster, dim3(across * cluster, down), dim3(kThreads), sizeof(FwdStep) * kAhead, s, p)
                                          : launch_dep(gated_small_fwd_kernel<ACT>, dim3(across, down), dim3(kThreads), sizeof(FwdStep) * kAhead, s, p);
  });
  TF_CUDA(e);
  TF_AFTER(s, what);
  return 1;
}
// Of both products, so that one gradient alone has the bits that it has beside the other.
bool gated_small_bwd_takes(int64_t M, int64_t F, int64_t K) { return small_product(M, K) && small_product(K, 2 * F); }
int gated_small_bwd(const float* x, const float* w, const float* z, const float* dout, float* dx, float* dw, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s,
                    const char* what) {
  if (!gated_small_bwd_takes(M, F, K)) return 0;
  Small p;
  memset(&p, 0, sizeof(p));
  p.x = x; p.w = w; p.z = z; p.dout = dout; p.dx = dx; p.dw = dw; p.M = (int)M; p.K = (int)K; p.F = (int)F;
  p.x_vec = K % 4 == 0 && aligned16(x); p.w_vec = F % 4 == 0 && aligned16(w); p.z_vec = F % 4 == 0 && aligned16(z) && aligned16(dout);
  p.dx_across = (int)((K + kTile - 1) / kTile);
  p.dw_across = (int)((F + 15) / 16);
  p.dx_tiles = dx ? p.dx_across * (int)((M + kTile - 1) / kTile) : 0;
  p.dw_tiles = dw ? p.dw_across * (int)((K + kTile - 1) / kTile) : 0;
  const int sms = device_sm_count();
  p.dx_ranks = dx ? cluster_for(p.dx_tiles, (F + 15) / 16, sms, kMostRanks) : 1;
  p.dw_ranks = dw ? cluster_for(p.dw_tiles, (M + kDepth - 1) / kDepth, sms, kMostRanks) : 1;
  p.per_cta = (int)(((F + p.dx_ranks - 1) / p.dx_ranks + 15) / 16 * 16);
  p.rows_per_cta = (int)(((M + p.dw_ranks - 1) / p.dw_ranks + kDepth - 1) / kDepth * kDepth);
  const int cluster = std::max(p.dx_ranks, p.dw_ranks), dx_each = cluster / p.dx_ranks, dw_each = cluster / p.dw_ranks;
  p.dx_clusters = (p.dx_tiles + dx_each - 1) / dx_each;
  const int clusters = p.dx_clusters + (p.dw_tiles + dw_each - 1) / dw_each;
  if (clusters == 0) return 1;
  note_compute_stream(s);
  KernelTimer kt("gated_small_bwd", s, 4.0 * M * F * K * ((dx != nullptr) + (dw != nullptr)), 0, 1);
  cudaError_t e = cudaSuccess;
  with_gate(activation, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    // as the forward kernel's: an SM that changes the split between the two waits to be empty
    static std::atomic<uint64_t> ready{0};
    e = once_per_device(ready, [] {
      const cudaError_t set = cudaFuncSetAttribute(gated_small_bwd_kernel<ACT>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
      return set != cudaSuccess ? set : cudaFuncSetAttribute(gated_small_bwd_kernel<ACT>, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    });
    if (e == cudaSuccess) e = launch_cluster(gated_small_bwd_kernel<ACT>, cluster, dim3((unsigned)(clusters * cluster)), dim3(kThreads), 0, s, p);
  });
  TF_CUDA(e);
  TF_AFTER(s, what);
  return 1;
}

}  // namespace tf
