// Attention and its gradients: entries, the choice of the path, and the exact-fp32 kernels of small calls.
//
// The kernels here hold a tile of 16 rows (queries of all heads that share a key-value head; backward also keys) and stream the other side
// through shared memory, 64 rows at a time.  Scores live in registers and shared memory only.  One launch forward, one backward: the blocks of
// dq and those of dk and dv form the probabilities again from the row maxima and sums that the forward call left.
#include "attention.h"
#include <math.h>
#include <algorithm>
#include <cmath>
#include "operands.h"

namespace tf {

bool attention_tc_takes(const AttentionArgs& a);
int attention_few(const AttentionArgs& a, size_t* bytes, cudaStream_t s, const char* what);
int attention_tc(const AttentionArgs& a, bool backward, size_t* bytes, cudaStream_t s, const char* what);
void note_contraction_path(int path);

namespace {

constexpr int kThreads = 128;
constexpr int kRows = 16, kStream = 64, kPitchW = kStream + 4;
constexpr int kMostDim = 256;

struct AttentionState {
  int kind;
  int64_t length;
  int heads, kv_heads, causal, window;
  float scale, cap;
};

// Row r of a key-value head: query r / group of head kv * group + r % group
struct Rows {
  const AttentionArgs& a;
  int b, kv;
  __device__ __forceinline__ int64_t at(int r) const { const int i = r / a.group; return (((int64_t)b * a.Tq + i) * a.H + kv * a.group + (r - i * a.group)) * a.D; }
  __device__ __forceinline__ int64_t stat(int r) const { const int i = r / a.group; return ((int64_t)b * a.H + kv * a.group + (r - i * a.group)) * a.Tq + i; }
  __device__ __forceinline__ int head(int r) const { return kv * a.group + r % a.group; }
  __device__ __forceinline__ int position(int r) const { return r / a.group + a.Tk - a.Tq; }
};
struct Keys {
  const AttentionArgs& a;
  int b, kv;
  __device__ __forceinline__ int64_t at(int j) const { return (((int64_t)b * a.Tk + j) * a.G + kv) * a.D; }
};

// Copies rows [first, first + COUNT) of `from`, zero behind the last one and behind the head's end.  A value that is not finite becomes zero, too,
// and marks its row: a product with a weight of zero must not make others NaN.
template <int DP, int COUNT, bool WIDE, class Where>
__device__ __forceinline__ void load_rows(float* to, const float* __restrict__ from, const Where& where, int first, int rows, int D, int* bad) {
  constexpr int kPer = WIDE ? 4 : 1, kAcross = DP / kPer;
#pragma unroll 4
  for (int n = threadIdx.x; n < COUNT * kAcross; n += kThreads) {
    const int r = n / kAcross, c = (n - r * kAcross) * kPer;
    float v[4] = {0.f, 0.f, 0.f, 0.f};
    if (first + r < rows && c < D) {
      const float* const p = from + where.at(first + r) + c;
      if (WIDE) { const float4 w = __ldg(reinterpret_cast<const float4*>(p)); v[0] = w.x; v[1] = w.y; v[2] = w.z; v[3] = w.w; }
      else v[0] = __ldg(p);
      if (bad) {
        bool fine = true;
#pragma unroll
        for (int i = 0; i < kPer; ++i) if (!(fabsf(v[i]) < INFINITY)) { v[i] = 0.f; fine = false; }
        if (!fine) bad[r] = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) to[r * (DP + 4) + c + i] = v[i];
  }
}
// x[2][4]: products of rows 2 ty, 2 ty + 1 of A with rows tx + 16 c of B
template <int DP> __device__ __forceinline__ void products(const float* __restrict__ A, const float* __restrict__ B, int ty, int tx, float x[2][4]) {
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int c = 0; c < 4; ++c) x[i][c] = 0.f;
#pragma unroll 4
  for (int d = 0; d < DP; d += 4) {
    float4 u[2], w[4];
#pragma unroll
    for (int i = 0; i < 2; ++i) u[i] = *reinterpret_cast<const float4*>(A + (2 * ty + i) * (DP + 4) + d);
#pragma unroll
    for (int c = 0; c < 4; ++c) w[c] = *reinterpret_cast<const float4*>(B + (tx + 16 * c) * (DP + 4) + d);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[i][c] = fmaf(u[i].x, w[c].x, x[i][c]); x[i][c] = fmaf(u[i].y, w[c].y, x[i][c]);
        x[i][c] = fmaf(u[i].z, w[c].z, x[i][c]); x[i][c] = fmaf(u[i].w, w[c].w, x[i][c]);
      }
  }
}
// acc[2][DP / 64]: adds rows 2 ty, 2 ty + 1 of W (16 x 64) times B (64 x DP), columns 4 tx + 64 n
template <int DP> __device__ __forceinline__ void add_product(const float* __restrict__ W, const float* __restrict__ B, int ty, int tx, float4 acc[2][DP / 64]) {
#pragma unroll 2
  for (int j = 0; j < kStream; j += 4) {
    float w[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) *reinterpret_cast<float4*>(w[i]) = *reinterpret_cast<const float4*>(W + (2 * ty + i) * kPitchW + j);
#pragma unroll
    for (int k = 0; k < 4; ++k)
#pragma unroll
      for (int n = 0; n < DP / 64; ++n) {
        const float4 v = *reinterpret_cast<const float4*>(B + (j + k) * (DP + 4) + 4 * tx + 64 * n);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          acc[i][n].x = fmaf(w[i][k], v.x, acc[i][n].x); acc[i][n].y = fmaf(w[i][k], v.y, acc[i][n].y);
          acc[i][n].z = fmaf(w[i][k], v.z, acc[i][n].z); acc[i][n].w = fmaf(w[i][k], v.w, acc[i][n].w);
        }
      }
  }
}
template <int DP, class Where>
__device__ __forceinline__ void store_rows(float* to, const Where& where, int first, int rows, int D, int ty, int tx, const float4 acc[2][DP / 64]) {
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (first + 2 * ty + i >= rows) continue;
    float* const p = to + where.at(first + 2 * ty + i);
#pragma unroll
    for (int n = 0; n < DP / 64; ++n) {
      const float v[4] = {acc[i][n].x, acc[i][n].y, acc[i][n].z, acc[i][n].w};
#pragma unroll
      for (int k = 0; k < 4; ++k) if (4 * tx + 64 * n + k < D) p[4 * tx + 64 * n + k] = v[k];
    }
  }
}
// The score of a product that the query sees, in units of log 2, and the derivative of the cap.  NaN where the product is not finite: a cap or a weight of zero would hide that.
__device__ __forceinline__ float score(const AttentionArgs& a, float product, float slope, int away, float& inner) {
  float c = product * a.scale;
  if (!(fabsf(c) < INFINITY)) c = NAN;
  inner = 1.f;
  if (a.cap > 0.f) {
    const float t = tanhf(c / a.cap);
    c = a.cap * t;
    inner = 1.f - t * t;
  }
  return __fmul_rn(fmaf(-slope, fabsf((float)away), c), kLog2e);     // rounded before a maximum is taken off, in both directions alike: the largest is 0 then, however large the scores are
}
// 2^(score - most) for the gradients: at most 1, also where another kernel's forward call rounded the score otherwise and it is above the largest
__device__ __forceinline__ float weight(float score, float most) {
  const float x = score - most;
  return exp2f(x > 0.f ? 0.f : x);               // NaN stays
}
__device__ __forceinline__ float half_warp_max(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}
__device__ __forceinline__ float half_warp_sum(float v) {
#pragma unroll
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// What a block knows of one row of queries
struct RowSight { Sight sight; int at, there; float document, slope; };
__device__ __forceinline__ RowSight row_sight(const AttentionArgs& a, const Rows& rows, int r, int count) {
  RowSight s;
  s.there = r < count;
  s.at = s.there ? rows.position(r) : 0;
  s.sight = sight_of(a, s.at);
  s.document = a.documents && s.there ? document_of(a, rows.b, s.at) : 0.f;
  s.slope = a.slopes && s.there ? __ldg(a.slopes + rows.head(r)) : 0.f;
  return s;
}
__device__ __forceinline__ bool row_sees(const AttentionArgs& a, const RowSight& s, int prefix, int j, float document) {
  return s.there && j < a.Tk && sees(s.sight, prefix, j) && (!a.documents || (s.document == document && document >= 0.f));
}
// Whether any key of [j0, j1) may be seen by a query at positions [p0, p1]
__device__ __forceinline__ bool tile_seen(const AttentionArgs& a, int p0, int p1, int prefix, int j0, int j1) {
  return j0 < prefix || (j0 <= sight_of(a, p1).hi && j1 > sight_of(a, p0).lo);
}

template <int DP> struct TileSmem {
  float A[2][kRows * (DP + 4)];
  float B[2][kStream * (DP + 4)];
  float W[2][kRows * kPitchW];
  float document[kStream];
  float stat[kStream][3];
  float delta[kRows];
  int bad[kStream];
};

// Latency-bound at the sizes that take it.
template <int DP, bool WIDE>
__global__ void __launch_bounds__(kThreads) attention_tile_fwd_kernel(const __grid_constant__ AttentionArgs a, int row_blocks) {
  extern __shared__ __align__(16) char raw[];
  TileSmem<DP>& sm = *reinterpret_cast<TileSmem<DP>*>(raw);
  grid_dep_sync();
  const int bg = blockIdx.x / row_blocks, block = blockIdx.x - bg * row_blocks, b = bg / a.G, kv = bg - b * a.G;
  const Rows rows{a, b, kv};
  const Keys keys{a, b, kv};
  const int count = a.group * a.Tq, first = (row_blocks - 1 - block) * kRows;       // the rows that see most go first
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int prefix = prefix_of(a, b);
  RowSight rs[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) rs[i] = row_sight(a, rows, first + 2 * ty + i, count);
  const int p0 = rows.position(first), p1 = rows.position(min(first + kRows, count) - 1);
  load_rows<DP, kRows, WIDE>(sm.A[0], a.q, rows, first, count, a.D, nullptr);
  float4 acc[2][DP / 64];
  float most[2] = {-INFINITY, -INFINITY}, sum[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < DP / 64; ++n) acc[i][n] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int j0 = 0; j0 < a.Tk; j0 += kStream) {
    if (!tile_seen(a, p0, p1, prefix, j0, j0 + kStream)) continue;
    __syncthreads();
    if (threadIdx.x < kStream) {
      sm.bad[threadIdx.x] = 0;
      if (a.documents) sm.document[threadIdx.x] = document_of(a, b, j0 + threadIdx.x);
    }
    __syncthreads();
    load_rows<DP, kStream, WIDE>(sm.B[0], a.k, keys, j0, a.Tk, a.D, sm.bad);
    load_rows<DP, kStream, WIDE>(sm.B[1], a.v, keys, j0, a.Tk, a.D, sm.bad);
    __syncthreads();
    float x[2][4];
    products<DP>(sm.A[0], sm.B[0], ty, tx, x);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float m = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int j = tx + 16 * c;
        float inner;
        x[i][c] = row_sees(a, rs[i], prefix, j0 + j, a.documents ? sm.document[j] : 0.f) ? (sm.bad[j] ? NAN : score(a, x[i][c], rs[i].slope, rs[i].at - j0 - j, inner)) : -INFINITY;
        m = fmaxf(m, x[i][c]);
      }
      m = fmaxf(most[i], half_warp_max(m));
      const float base = max_of_finite_or(m), alpha = exp2f(most[i] - base);             // 0 at the first key
      float s = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[i][c] = exp2f(x[i][c] - base);
        s += x[i][c];
        sm.W[0][(2 * ty + i) * kPitchW + tx + 16 * c] = x[i][c];
      }
      sum[i] = sum[i] * alpha + half_warp_sum(s);
      most[i] = m;
#pragma unroll
      for (int n = 0; n < DP / 64; ++n) { acc[i][n].x *= alpha; acc[i][n].y *= alpha; acc[i][n].z *= alpha; acc[i][n].w *= alpha; }
    }
    __syncwarp();                                // a row of W is written and read by one half of a warp
    add_product<DP>(sm.W[0], sm.B[1], ty, tx, acc);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float inv = sum[i] == 0.f ? 0.f : 1.f / sum[i];
#pragma unroll
    for (int n = 0; n < DP / 64; ++n) { acc[i][n].x *= inv; acc[i][n].y *= inv; acc[i][n].z *= inv; acc[i][n].w *= inv; }
    const int r = first + 2 * ty + i;
    if (a.stats && tx == 0 && r < count) {
      const int64_t at = rows.stat(r);
      a.stats[2 * at] = max_of_finite_or(most[i]);
      a.stats[2 * at + 1] = inv;
    }
  }
  store_rows<DP>(a.o, rows, first, count, a.D, ty, tx, acc);
}

// Of a key-value head's blocks the first make dq of their rows, the others dk and dv of their keys.
template <int DP, bool WIDE>
__global__ void __launch_bounds__(kThreads) attention_tile_bwd_kernel(const __grid_constant__ AttentionArgs a, int row_blocks, int blocks) {
  extern __shared__ __align__(16) char raw[];
  TileSmem<DP>& sm = *reinterpret_cast<TileSmem<DP>*>(raw);
  grid_dep_sync();
  const int bg = blockIdx.x / blocks, block = blockIdx.x - bg * blocks, b = bg / a.G, kv = bg - b * a.G;
  const Rows rows{a, b, kv};
  const Keys keys{a, b, kv};
  const int count = a.group * a.Tq;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int prefix = prefix_of(a, b);
  float4 one[2][DP / 64], two[2][DP / 64];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int n = 0; n < DP / 64; ++n) one[i][n] = two[i][n] = make_float4(0.f, 0.f, 0.f, 0.f);
  auto delta_of = [&](int r) {                   // dout * out of a row, by a warp
    float d = 0.f;
    const int64_t at = rows.at(r);
    for (int c = lane; c < a.D; c += 32) d = fmaf(__ldg(a.dout + at + c), __ldg(a.out + at + c), d);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) d += __shfl_xor_sync(0xffffffffu, d, o);
    return d;
  };
  if (block < row_blocks) {
    const int first = (row_blocks - 1 - block) * kRows;
    RowSight rs[2];
    float most[2], inv[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = first + 2 * ty + i;
      rs[i] = row_sight(a, rows, r, count);
      most[i] = r < count ? a.stats[2 * rows.stat(r)] : 0.f;
      inv[i] = r < count ? a.stats[2 * rows.stat(r) + 1] : 0.f;
    }
    const int p0 = rows.position(first), p1 = rows.position(min(first + kRows, count) - 1);
    load_rows<DP, kRows, WIDE>(sm.A[0], a.q, rows, first, count, a.D, nullptr);
    load_rows<DP, kRows, WIDE>(sm.A[1], a.dout, rows, first, count, a.D, nullptr);
    for (int r = warp; r < kRows; r += kThreads / 32) {
      const float d = first + r < count ? delta_of(first + r) : 0.f;
      if (lane == 0) sm.delta[r] = d;
    }
    for (int j0 = 0; j0 < a.Tk; j0 += kStream) {
      if (!tile_seen(a, p0, p1, prefix, j0, j0 + kStream)) continue;
      __syncthreads();
      if (threadIdx.x < kStream) {
        sm.bad[threadIdx.x] = 0;
        if (a.documents) sm.document[threadIdx.x] = document_of(a, b, j0 + threadIdx.x);
      }
      __syncthreads();
      load_rows<DP, kStream, WIDE>(sm.B[0], a.k, keys, j0, a.Tk, a.D, sm.bad);
      load_rows<DP, kStream, WIDE>(sm.B[1], a.v, keys, j0, a.Tk, a.D, sm.bad);
      __syncthreads();
      float x[2][4], y[2][4];
      products<DP>(sm.A[0], sm.B[0], ty, tx, x);
      products<DP>(sm.A[1], sm.B[1], ty, tx, y);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const int j = tx + 16 * c;
          float w = 0.f, inner;
          if (row_sees(a, rs[i], prefix, j0 + j, a.documents ? sm.document[j] : 0.f)) {
            w = weight(score(a, x[i][c], rs[i].slope, rs[i].at - j0 - j, inner), most[i]) * inv[i];
            w = sm.bad[j] ? NAN : w * (y[i][c] - sm.delta[2 * ty + i]) * inner * a.scale;
          }
          sm.W[0][(2 * ty + i) * kPitchW + j] = w;
        }
      __syncwarp();
      add_product<DP>(sm.W[0], sm.B[0], ty, tx, one);
    }
    if (a.dq) store_rows<DP>(a.dq, rows, first, count, a.D, ty, tx, one);
    return;
  }
  const int first = (block - row_blocks) * kRows;
  load_rows<DP, kRows, WIDE>(sm.A[0], a.k, keys, first, a.Tk, a.D, nullptr);
  load_rows<DP, kRows, WIDE>(sm.A[1], a.v, keys, first, a.Tk, a.D, nullptr);
  float document[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) document[i] = a.documents ? document_of(a, b, first + 2 * ty + i) : 0.f;
  for (int r0 = 0; r0 < count; r0 += kStream) {
    if (!tile_seen(a, rows.position(r0), rows.position(min(r0 + kStream, count) - 1), prefix, first, first + kRows)) continue;
    __syncthreads();
    if (threadIdx.x < kStream) {
      const int r = r0 + threadIdx.x;
      sm.bad[threadIdx.x] = 0;
      sm.stat[threadIdx.x][0] = r < count ? a.stats[2 * rows.stat(r)] : 0.f;
      sm.stat[threadIdx.x][1] = r < count ? a.stats[2 * rows.stat(r) + 1] : 0.f;
    }
    __syncthreads();
    load_rows<DP, kStream, WIDE>(sm.B[0], a.q, rows, r0, count, a.D, sm.bad);
    load_rows<DP, kStream, WIDE>(sm.B[1], a.dout, rows, r0, count, a.D, sm.bad);
    for (int r = warp; r < kStream; r += kThreads / 32) {
      const float d = r0 + r < count ? delta_of(r0 + r) : 0.f;
      if (lane == 0) sm.stat[r][2] = d;
    }
    __syncthreads();
    float x[2][4], y[2][4];
    products<DP>(sm.A[0], sm.B[0], ty, tx, x);
    products<DP>(sm.A[1], sm.B[1], ty, tx, y);
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int r = tx + 16 * c;
      const RowSight rs = row_sight(a, rows, r0 + r, count);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = first + 2 * ty + i;
        float p = 0.f, w = 0.f, inner;
        if (row_sees(a, rs, prefix, j, document[i])) {
          p = sm.bad[r] ? NAN : weight(score(a, x[i][c], rs.slope, rs.at - j, inner), sm.stat[r][0]) * sm.stat[r][1];
          w = sm.bad[r] ? NAN : p * (y[i][c] - sm.stat[r][2]) * inner * a.scale;
        }
        sm.W[0][(2 * ty + i) * kPitchW + r] = w;
        sm.W[1][(2 * ty + i) * kPitchW + r] = p;
      }
    }
    __syncwarp();
    add_product<DP>(sm.W[0], sm.B[0], ty, tx, one);
    add_product<DP>(sm.W[1], sm.B[1], ty, tx, two);
  }
  if (a.dk) store_rows<DP>(a.dk, keys, first, a.Tk, a.D, ty, tx, one);
  if (a.dv) store_rows<DP>(a.dv, keys, first, a.Tk, a.D, ty, tx, two);
}

// ---- host side ------------------------------------------------------------------------------------------------------------
template <class F> void with_dim(int D, F&& f) {
  if (D <= 64) f(std::integral_constant<int, 64>());
  else if (D <= 128) f(std::integral_constant<int, 128>());
  else f(std::integral_constant<int, 256>());
}
bool wide(const AttentionArgs& a) {
  uintptr_t bits = (uintptr_t)a.D * sizeof(float);
  for (const void* p : {(const void*)a.q, (const void*)a.k, (const void*)a.v, (const void*)a.dout}) bits |= reinterpret_cast<uintptr_t>(p);
  return bits % 16 == 0;
}
cudaError_t tile_fwd(const AttentionArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  with_dim(a.D, [&](auto dim) {
    auto run = [&](auto w) {
      constexpr int DP = decltype(dim)::value;
      static std::atomic<uint64_t> ready{0};
      const auto kernel = attention_tile_fwd_kernel<DP, decltype(w)::value>;
      const int bytes = (int)sizeof(TileSmem<DP>);
      e = once_per_device(ready, [kernel, bytes] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
      const int row_blocks = (int)(((int64_t)a.group * a.Tq + kRows - 1) / kRows);
      if (e == cudaSuccess) e = launch_dep(kernel, dim3((unsigned)(row_blocks * a.B * a.G)), dim3(kThreads), (size_t)bytes, s, a, row_blocks);
    };
    if (wide(a)) run(std::true_type()); else run(std::false_type());
  });
  return e;
}
cudaError_t tile_bwd(const AttentionArgs& a, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  with_dim(a.D, [&](auto dim) {
    auto run = [&](auto w) {
      constexpr int DP = decltype(dim)::value;
      static std::atomic<uint64_t> ready{0};
      const auto kernel = attention_tile_bwd_kernel<DP, decltype(w)::value>;
      const int bytes = (int)sizeof(TileSmem<DP>);
      e = once_per_device(ready, [kernel, bytes] { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); });
      const int row_blocks = a.dq ? (int)(((int64_t)a.group * a.Tq + kRows - 1) / kRows) : 0, key_blocks = a.dk || a.dv ? (a.Tk + kRows - 1) / kRows : 0;
      if (e == cudaSuccess && row_blocks + key_blocks) e = launch_dep(kernel, dim3((unsigned)((row_blocks + key_blocks) * a.B * a.G)), dim3(kThreads), (size_t)bytes, s, a, row_blocks, row_blocks + key_blocks);
    };
    if (wide(a)) run(std::true_type()); else run(std::false_type());
  });
  return e;
}

int check_attention(const char* what, const AttentionState* st, const DLArray* q, const DLArray* k, const DLArray* v, const DLArray* documents, AttentionArgs* a) {
  TF_REQUIRE(st, "%s: the state was not made by TfAttentionState", what);
  TF_REQUIRE(q && q->ndim == 2 && k && k->ndim == 2 && v && v->ndim == 2, "%s: query, key and value have to be matrices of tokens by heads", what);
  TF_REQUIRE(q->shape[0] >= 0 && q->shape[1] >= 0 && q->shape[1] % st->heads == 0, "%s: the query's columns are not %d heads", what, st->heads);
  const int64_t D = q->shape[1] / st->heads, B = q->shape[0] / st->length;
  TF_REQUIRE(D >= 1 && D <= kMostDim, "%s: heads of 1 to %d elements, not %lld", what, kMostDim, (long long)D);
  TF_REQUIRE(q->shape[0] == B * st->length, "%s: %lld queries are not sequences of %lld", what, (long long)q->shape[0], (long long)st->length);
  TF_REQUIRE(k->shape[1] == D * st->kv_heads && v->shape[1] == D * st->kv_heads, "%s: key and value have to have %d heads of %lld elements", what, st->kv_heads, (long long)D);
  TF_REQUIRE(k->shape[0] == v->shape[0], "%s: key and value are of different tokens", what);
  TF_REQUIRE(B > 0 ? k->shape[0] >= 0 && k->shape[0] % B == 0 : k->shape[0] == 0, "%s: the keys are not those of %lld sequences", what, (long long)B);
  const int64_t Tk = B ? k->shape[0] / B : 0;
  TF_REQUIRE(st->length <= (1 << 24) && Tk <= (1 << 24) && st->length * (st->heads / st->kv_heads) <= (1ll << 28), "%s: sequences are too long", what);
  TF_REQUIRE(B * (st->heads * (st->length / kRows + 1) + st->kv_heads * (Tk / kRows + 1)) < (1ll << 31), "%s: more blocks than a launch has", what);
  TF_REQUIRE(!documents || Tk >= st->length, "%s: documents need a key for every query", what);
  memset(a, 0, sizeof(*a));
  a->B = (int)B; a->H = st->heads; a->G = st->kv_heads; a->group = st->heads / st->kv_heads; a->Tq = (int)st->length; a->Tk = (int)Tk; a->D = (int)D;
  a->causal = st->causal; a->window = std::min(st->window, 1 << 25); a->scale = st->scale; a->cap = st->cap;
  return 0;
}
// Up to 16 rows a key-value head, whose keys the kernel of few queries reads once for every four
bool few_queries(const AttentionArgs& a) { return (int64_t)a.group * a.Tq <= 16 && a.Tk > 0; }
// Whether the tensor path is the shorter road, in us: launches and a CTA's start and end, then what each further wave of CTAs and each further tile of the longest one
// takes.  Measured, exact against tensor path: 1 x 4 heads of 64, causal, 16 queries forward 6.8 and 11.0, backward 12.6 and 12.1; 64 queries 10.3 and 10.5, 21.3 and
// 12.6; 512 queries 60 and 16, 168 and 21; 16 x 16 heads, 16 queries 11.5 and 24.8, 21.1 and 54.3; 64 queries 26.9 and 25.8, 88 and 57.  Where the directions are near each other they
// go the same road: scores that both round alike leave the gradients of 4 x 64 tokens 4e-7 off, otherwise 6e-7.
bool tensor_path_pays(const AttentionArgs& a, bool backward) {
  const auto over = [](double n, double of) { return std::ceil(n / of); };
  const double sms = device_sm_count(), rows = (double)a.group * a.Tq, sequences = (double)a.B * a.G;
  const double per_sm = a.D <= 64 ? 4 : a.D <= 128 ? 2 : 1, row_blocks = over(rows, kRows), key_blocks = over(a.Tk, kRows);
  const double q_tiles = over(a.Tq, 128), k_tiles = over(a.Tk, 128), more = a.D <= 64 ? 1.0 : 1.6;
  if (!backward) {
    const double exact = 4.0 + std::max(1.0, sequences * row_blocks / (per_sm * sms)) * (a.D <= 64 ? 0.1 : 0.2) * std::max(24.0, (double)a.Tk);
    const double waves = std::max(1.0, (double)a.B * a.H * q_tiles / sms);
    return more * (6.2 + 4.0 + (waves - 1) * 11.0 + waves * (k_tiles - 1) * 2.0) < exact;
  }
  const double exact = 8.0 + std::max(1.0, sequences * (row_blocks + key_blocks) / (per_sm * sms)) * (a.D <= 64 ? 0.25 : 0.4) * std::max((double)a.Tk, rows);
  const double waves = std::max(1.0, (2 * sequences * k_tiles + (double)a.B * a.H * q_tiles) / sms);
  return more * (12.0 + (waves - 1) * 10.0 + std::max(waves * (k_tiles - 1), a.group * q_tiles - 1) * 2.5) < exact;
}
// 0: the exact kernels are to run, 1: launched, or short of memory; -1: error
int run_tensor_path(const AttentionArgs& a, bool backward, int* memorytoSaving, cudaStream_t s, const char* what) {
  if (contraction_path() == 1) return 0;
  const bool takes = attention_tc_takes(a);
  TF_REQUIRE(contraction_path() != 2 || takes, "%s: the tensor path takes heads of up to 128 elements and at least one key", what);
  if (!takes || (contraction_path() == 0 && !tensor_path_pays(a, backward))) return 0;
  size_t bytes = 0;
  const int r = attention_tc(a, backward, &bytes, s, what);
  if (r > 0 && memorytoSaving) *memorytoSaving = bytes > 0x7fffffffu ? 0x7fffffff : (int)bytes;
  if (r >= 0) note_contraction_path(2);
  return r < 0 ? -1 : 1;
}
const float* opt_in(const DLArray* a) { return a ? (const float*)a->data : nullptr; }

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" {

int TfAttentionState(int64_t length, int heads, int kv_heads, int causal, int window, float scale, float cap, void*** state) {
  const char* const what = "TfAttentionState";
  TF_REQUIRE(state, "%s: null cell", what);
  TF_REQUIRE(length >= 1, "%s: sequences have at least one query", what);
  TF_REQUIRE(heads >= 1 && kv_heads >= 1 && heads % kv_heads == 0, "%s: %d query heads do not share %d key-value heads", what, heads, kv_heads);
  TF_REQUIRE(causal == 0 || causal == 1, "%s: causal is 0 or 1", what);
  TF_REQUIRE(window >= 0, "%s: a window is positive, or 0 for none", what);
  TF_REQUIRE(std::isfinite(scale), "%s: the scale has to be finite", what);
  TF_REQUIRE(std::isfinite(cap) && cap >= 0.f, "%s: a cap is positive and finite, or 0 for none", what);
  AttentionState* st = plan_of<AttentionState>(state, kPlanAttention);
  TF_REQUIRE(st || !holds_plan(state), "%s: the cell holds another descriptor", what);
  if (!st) st = new_plan<AttentionState>(state, kPlanAttention, 1);
  st->length = length; st->heads = heads; st->kv_heads = kv_heads; st->causal = causal; st->window = window; st->scale = scale; st->cap = cap;
  return 0;
}

int TfAttentionForward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle value, const DLArrayHandle documents, const DLArrayHandle prefix,
                       const DLArrayHandle slopes, DLArrayHandle output, DLArrayHandle stats, void*** state, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfAttentionForward";
  const AttentionState* st = plan_of<AttentionState>(state, kPlanAttention);
  AttentionArgs a;
  if (check_attention(what, st, query, key, value, documents, &a)) return -1;
  Operands o(what);
  o.add(query, "query", -1, false); o.add(key, "key", -1, false); o.add(value, "value", -1, false); o.add(documents, "documents", (int64_t)a.B * a.Tk, false, true);
  o.add(prefix, "prefix", a.B, false, true); o.add(slopes, "slopes", a.H, false, true); o.add(output, "output", numel(query), true);
  o.add(stats, "stats", 2ll * a.B * a.H * a.Tq, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.q = (const float*)query->data; a.k = (const float*)key->data; a.v = (const float*)value->data;
  a.documents = opt_in(documents); a.prefix = opt_in(prefix); a.slopes = opt_in(slopes);
  a.o = out_f32(output); a.stats = stats ? out_f32(stats) : nullptr;
  if (a.B == 0) return 0;
  note_compute_stream(s);
  KernelTimer kt(what, s, 4.0 * a.B * a.H * (double)a.Tq * a.Tk * a.D, 4.0 * (2.0 * numel(query) + 2.0 * numel(key)));
  const bool few = few_queries(a) && contraction_path() != 2;
  if (!few) {
    if (const int r = run_tensor_path(a, false, memorytoSaving, s, what)) return r < 0 ? -1 : 0;
  }
  note_contraction_path(1);
  if (few) {
    size_t bytes = 0;
    const int r = attention_few(a, &bytes, s, what);
    if (r > 0 && memorytoSaving) *memorytoSaving = bytes > 0x7fffffffu ? 0x7fffffff : (int)bytes;
    return r < 0 ? -1 : 0;
  }
  TF_CUDA(tile_fwd(a, s));
  TF_AFTER(s, what);
  return 0;
}

int TfAttentionBackward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle value, const DLArrayHandle documents, const DLArrayHandle prefix,
                        const DLArrayHandle slopes, const DLArrayHandle output, const DLArrayHandle stats, const DLArrayHandle doutput, DLArrayHandle dquery, DLArrayHandle dkey,
                        DLArrayHandle dvalue, void*** state, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfAttentionBackward";
  const AttentionState* st = plan_of<AttentionState>(state, kPlanAttention);
  AttentionArgs a;
  if (check_attention(what, st, query, key, value, documents, &a)) return -1;
  Operands o(what);
  const int64_t nq = numel(query), nk = numel(key);
  o.add(query, "query", -1, false); o.add(key, "key", -1, false); o.add(value, "value", -1, false); o.add(documents, "documents", (int64_t)a.B * a.Tk, false, true);
  o.add(prefix, "prefix", a.B, false, true); o.add(slopes, "slopes", a.H, false, true); o.add(output, "output", nq, false); o.add(stats, "stats", 2ll * a.B * a.H * a.Tq, false);
  o.add(doutput, "doutput", nq, false); o.add(dquery, "dquery", nq, true, true); o.add(dkey, "dkey", nk, true, true); o.add(dvalue, "dvalue", nk, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  a.q = (const float*)query->data; a.k = (const float*)key->data; a.v = (const float*)value->data;
  a.documents = opt_in(documents); a.prefix = opt_in(prefix); a.slopes = opt_in(slopes);
  a.out = (const float*)output->data; a.stats = (float*)stats->data; a.dout = (const float*)doutput->data;
  a.dq = dquery ? out_f32(dquery) : nullptr; a.dk = dkey ? out_f32(dkey) : nullptr; a.dv = dvalue ? out_f32(dvalue) : nullptr;
  if (a.B == 0 || !(a.dq || a.dk || a.dv)) return 0;
  note_compute_stream(s);
  KernelTimer kt(what, s, 10.0 * a.B * a.H * (double)a.Tq * a.Tk * a.D, 4.0 * (4.0 * nq + 4.0 * nk));
  if (const int r = run_tensor_path(a, true, memorytoSaving, s, what)) return r < 0 ? -1 : 0;
  note_contraction_path(1);
  TF_CUDA(tile_bwd(a, s));
  TF_AFTER(s, what);
  return 0;
}

}  // extern "C"
