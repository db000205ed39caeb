// Rotary positions of heads, alone and behind a root-mean-square norm of each head, with their gradients.
//
//   rotation   a pair (a, b) of a head's elements at position t, f_i turns (radians) a position:
//              (a, b) -> A (a cos(t f_i) - b sin(t f_i), a sin(t f_i) + b cos(t f_i)); elements behind the rotated part stay.
//              Its gradient is the rotation by the opposite angle, with the same A.
//   norm       n = x / sqrt(mean(x^2) + eps), y = rotation(gamma * n) over each head of head_dim elements.
//              u = rotation back of dy, g = gamma * u, dx = inv * (g - n mean(g n)), dgamma = sum over tokens and heads of u * n.
//
// HBM-bound: 8 bytes an element, 12 the norm's gradients.  Rotation of 2 x 8192 tokens, 16 heads of 128: 42 us, 6.3 TB/s.  A block takes a run of heads and makes the sines of their tokens once, for all
// heads of a token, while its loads are in flight.  Angles are formed and reduced to an eighth of a turn in 64 bits: in 32 a position of
// 10^5 would be off by 0.004 radians.
#include "common.h"
#include <math.h>
#include <algorithm>
#include <cmath>
#include <limits>
#include <type_traits>
#include "operands.h"
#include "pieces.h"

namespace tf {
namespace {

constexpr int kThreads = 256;
constexpr int kNormBlocks = 4;       // blocks of the norm's gradients that an SM holds
constexpr int kMostPairs = 128, kMostDim = 2 * kMostPairs;

struct RotaryState {
  int kind;
  int D, pairs, interleaved;
  float amplitude;
  double quarters[kMostPairs];       // quarter turns per position
};
struct Quarters { double of[kMostPairs]; };

struct HeadArgs {
  const float* x;
  const float* gamma;
  const float* dy;
  float* y;                          // backward: dx
  float* dgamma;
  float* part;                       // dgamma's sums of each block
  uint32_t* count;
  AmaxOut am;
  int64_t rows;                      // tokens x heads
  int heads;
};
struct RotaryArgs {
  const float* positions;
  int64_t length, start;
  float eps, amplitude;
  int D, pairs, chunks;              // chunks of 2 VEC elements a head has
  int interleaved, back;
  int per_block;                     // heads of a block's pass
  int blocks[2];                     // of each of the two arrays
  HeadArgs h[2];
};

// cos and sin of q quarter turns: whole quarters swap and negate them, the rest, an eighth of a turn at most, goes into the series, whose next terms are 2^-29 of the values
__device__ __forceinline__ float2 turn(double q, float amplitude) {
  const double n = rint(q);
  const float x = (float)((q - n) * 1.5707963267948966), y = x * x;
  float s = fmaf(fmaf(fmaf(1.f / 362880.f, y, -1.f / 5040.f), y, 1.f / 120.f), y, -1.f / 6.f);
  float c = fmaf(fmaf(fmaf(fmaf(-1.f / 3628800.f, y, 1.f / 40320.f), y, -1.f / 720.f), y, 1.f / 24.f), y, -0.5f);
  s = fmaf(s * y, x, x);
  c = fmaf(c, y, 1.f);
  const int k = (int)((long long)n & 3);
  const float cs = k & 1 ? s : c, sn = k & 1 ? c : s;
  return make_float2(amplitude * (k == 1 || k == 2 ? -cs : cs), amplitude * (k & 2 ? -sn : sn));
}

// Where chunk c of a head lies: elements [a, a + VEC) and [b, b + VEC).  With pairs of halves the two pieces of a rotated chunk are half the
// rotated part apart, so that a thread holds whole pairs in both layouts.
template <int VEC> __device__ __forceinline__ void place(const RotaryArgs& p, int c, int& a, int& b) {
  const int turned = p.pairs / VEC;
  if (c >= turned) { a = 2 * p.pairs + 2 * VEC * (c - turned); b = a + VEC; }
  else if (p.interleaved) { a = 2 * VEC * c; b = a + VEC; }
  else { a = VEC * c; b = p.pairs + VEC * c; }
}
__device__ __forceinline__ void turn_pair(float2 t, float s, float& a, float& b) {
  const float x = a * t.x - b * s;
  b = a * s + b * t.x;
  a = x;
}
// v: 2 VEC elements; cs: cosines and sines of the chunk's VEC pairs
template <int VEC> __device__ __forceinline__ void rotate(const RotaryArgs& p, const float2* __restrict__ cs, float* v, bool back) {
  if (p.interleaved) {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { const float2 t = cs[i]; turn_pair(t, back ? -t.y : t.y, v[2 * i], v[2 * i + 1]); }
  } else {
#pragma unroll
    for (int i = 0; i < VEC; ++i) { const float2 t = cs[i]; turn_pair(t, back ? -t.y : t.y, v[i], v[VEC + i]); }
  }
}
template <int VEC> __device__ __forceinline__ void load_chunk(const RotaryArgs& p, const float* __restrict__ row, int c, float* v) {
  int a, b;
  place<VEC>(p, c, a, b);
  get<VEC>(v, row + a);
  if (VEC > 1 || b < p.D) get<VEC>(v + VEC, row + b); else v[VEC] = 0.f;          // the last element of an odd width has no partner
}
template <int VEC> __device__ __forceinline__ void store_chunk(const RotaryArgs& p, float* __restrict__ row, int c, const float* v) {
  int a, b;
  place<VEC>(p, c, a, b);
  put<VEC>(row + a, v);
  if (VEC > 1 || b < p.D) put<VEC>(row + b, v + VEC);
}
// The angles of the tokens that heads [r0, r1) belong to
__device__ __forceinline__ void make_turns(const RotaryArgs& p, const Quarters& f, float2* cs, int64_t r0, int64_t r1, int heads) {
  const unsigned t0 = (unsigned)r0 / (unsigned)heads, n = ((unsigned)(r1 - 1) / (unsigned)heads - t0 + 1) * (unsigned)p.pairs;       // rows are fewer than 2^31
  for (unsigned i = threadIdx.x; i < n; i += kThreads) {
    const unsigned t = i / (unsigned)p.pairs, pair = i - t * (unsigned)p.pairs, token = t0 + t;
    const double at = p.positions ? (double)__ldg(p.positions + token) : (double)(p.start + token % (unsigned)p.length);
    cs[i] = turn(at * f.of[pair], p.amplitude);
  }
}
template <int L> __device__ __forceinline__ float sum_of(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// The largest magnitude of what the block wrote.  Each of the two arrays has words of its own, which its first block clears for the next call.
__device__ __forceinline__ void commit_max(const AmaxOut& am, uint32_t m, bool first) {
  amax_commit(AmaxOut{am.word, nullptr}, m);
  if (first && threadIdx.x == 0 && am.clear) *am.clear = 0u;
}

// L threads a head, N chunks of 2 VEC elements each, U heads a thread.  NORM: the norm in front of the rotation.
template <int VEC, int L, int N, int U, bool NORM>
__global__ void __launch_bounds__(kThreads) heads_kernel(const __grid_constant__ RotaryArgs p, const __grid_constant__ Quarters f) {
  extern __shared__ __align__(16) float2 cs[];
  constexpr int kGroups = kThreads / L;
  grid_dep_sync();
  const int which = (int)blockIdx.x >= p.blocks[0];
  const HeadArgs& h = p.h[which];
  const int64_t r0 = (int64_t)((int)blockIdx.x - (which ? p.blocks[0] : 0)) * p.per_block, r1 = min(h.rows, r0 + p.per_block);
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  float v[U][N][2 * VEC];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * kGroups + group;
#pragma unroll
    for (int n = 0; n < N; ++n)
      if (r < r1 && lane + L * n < p.chunks) load_chunk<VEC>(p, h.x + r * p.D, lane + L * n, v[u][n]);
      else
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) v[u][n][j] = 0.f;
  }
  make_turns(p, f, cs, r0, r1, h.heads);
  __syncthreads();
  const unsigned in_token = (unsigned)r0 % (unsigned)h.heads;
  uint32_t m = 0;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t r = r0 + u * kGroups + group;
    float inv = 1.f;
    if (NORM) {
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(v[u][n][j], v[u][n][j], ss);
      inv = 1.f / sqrtf(sum_of<L>(ss) / (float)p.D + p.eps);
    }
    if (r >= r1) continue;
    const unsigned token = (in_token + (unsigned)(u * kGroups + group)) / (unsigned)h.heads;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int c = lane + L * n;
      if (c >= p.chunks) continue;
      float* const w = v[u][n];
      if (NORM) {
        float g[2 * VEC];
        load_chunk<VEC>(p, h.gamma, c, g);
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) w[j] = w[j] * inv * g[j];
      }
      if (c < p.pairs / VEC) rotate<VEC>(p, cs + token * p.pairs + c * VEC, w, p.back);
#pragma unroll
      for (int j = 0; j < 2 * VEC; ++j) m = max(m, amax_key(w[j]));
      store_chunk<VEC>(p, h.y + r * p.D, c, w);
    }
  }
  commit_max(h.am, m, (int)blockIdx.x == (which ? p.blocks[0] : 0));
}

// Gradients of the norm and the rotation.  A block works through every gridDim-th pass of its array, adds up dgamma in registers, then over
// its groups of threads and, in the block that comes last, over the blocks: always in the same order, in one launch.
template <int VEC, int L, int N, int U>
__global__ void __launch_bounds__(kThreads, kNormBlocks) head_norm_bwd_kernel(const __grid_constant__ RotaryArgs p, const __grid_constant__ Quarters f) {
  extern __shared__ __align__(16) float2 cs[];
  __shared__ bool last;
  __shared__ unsigned short token_of[U * kThreads / L];
  constexpr int kGroups = kThreads / L, kPart = VEC == 4 ? 4 : 1;
  grid_dep_sync();
  const int which = (int)blockIdx.x >= p.blocks[0], block = (int)blockIdx.x - (which ? p.blocks[0] : 0), blocks = p.blocks[which];
  const HeadArgs& h = p.h[which];
  const int lane = threadIdx.x % L, group = threadIdx.x / L;
  float gamma[N][2 * VEC], sums[N][2 * VEC];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int j = 0; j < 2 * VEC; ++j) { gamma[n][j] = 0.f; sums[n][j] = 0.f; }
    if (lane + L * n < p.chunks) load_chunk<VEC>(p, h.gamma, lane + L * n, gamma[n]);
  }
  uint32_t m = 0;
  for (int64_t r0 = (int64_t)block * p.per_block; r0 < h.rows; r0 += (int64_t)blocks * p.per_block) {
    const int64_t r1 = min(h.rows, r0 + p.per_block);
    float x[U][N][2 * VEC], d[U][N][2 * VEC];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * kGroups + group;
#pragma unroll
      for (int n = 0; n < N; ++n)
        if (r < r1 && lane + L * n < p.chunks) { load_chunk<VEC>(p, h.x + r * p.D, lane + L * n, x[u][n]); load_chunk<VEC>(p, h.dy + r * p.D, lane + L * n, d[u][n]); }
        else
#pragma unroll
          for (int j = 0; j < 2 * VEC; ++j) x[u][n][j] = d[u][n][j] = 0.f;
    }
    __syncthreads();                             // the pass before is done with the angles
    if (threadIdx.x < U * kGroups) token_of[threadIdx.x] = (unsigned short)(((unsigned)r0 % (unsigned)h.heads + threadIdx.x) / (unsigned)h.heads);
    make_turns(p, f, cs, r0, r1, h.heads);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t r = r0 + u * kGroups + group;
      const bool there = r < r1;
      const unsigned token = token_of[u * kGroups + group];
      float ss = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int c = lane + L * n;
        if (there && c < p.pairs / VEC) rotate<VEC>(p, cs + token * p.pairs + c * VEC, d[u][n], true);
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) ss = fmaf(x[u][n][j], x[u][n][j], ss);
      }
      const float inv = 1.f / sqrtf(sum_of<L>(ss) / (float)p.D + p.eps);
      float dot = 0.f;
#pragma unroll
      for (int n = 0; n < N; ++n)
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) {
          x[u][n][j] *= inv;
          if (there) sums[n][j] = fmaf(d[u][n][j], x[u][n][j], sums[n][j]);
          d[u][n][j] *= gamma[n][j];
          dot = fmaf(d[u][n][j], x[u][n][j], dot);
        }
      dot = sum_of<L>(dot) / (float)p.D;
      if (!there || !h.y) continue;
#pragma unroll
      for (int n = 0; n < N; ++n) {
        if (lane + L * n >= p.chunks) continue;
#pragma unroll
        for (int j = 0; j < 2 * VEC; ++j) { d[u][n][j] = inv * (d[u][n][j] - x[u][n][j] * dot); m = max(m, amax_key(d[u][n][j])); }
        store_chunk<VEC>(p, h.y + r * p.D, lane + L * n, d[u][n]);
      }
    }
  }
  commit_max(h.am, m, block == 0);
  if (!h.dgamma) return;
  float* const held = reinterpret_cast<float*>(cs);            // [groups][D]
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int c = lane + L * n;
    if (c >= p.chunks) continue;
    int a, b;
    place<VEC>(p, c, a, b);
#pragma unroll
    for (int j = 0; j < VEC; ++j) {
      held[group * p.D + a + j] = sums[n][j];
      if (b + j < p.D) held[group * p.D + b + j] = sums[n][VEC + j];
    }
  }
  __syncthreads();
  for (int e = threadIdx.x; e < p.D; e += kThreads) {
    float s = 0.f;
#pragma unroll
    for (int g = 0; g < kGroups; ++g) s += held[g * p.D + e];
    if (blocks == 1) h.dgamma[e] = s;
    else h.part[(int64_t)block * p.D + e] = s;
  }
  if (blocks == 1) return;
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicInc(h.count, (unsigned)blocks - 1) == (unsigned)blocks - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  // Eight loads in flight, added as a tree: chains of blocks / (8 ways) sums, then the ways'
  const int wide = p.D / kPart, ways = min(kThreads / wide, 32), way = threadIdx.x / wide, e = (threadIdx.x - way * wide) * kPart;      // D <= kThreads
  if (way < ways) {
    float sum[kPart] = {};
    for (int b = way; b < blocks; b += 8 * ways) {
      float w[8][kPart];
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (b + i * ways < blocks) get_beyond_l1<kPart>(w[i], h.part + (int64_t)(b + i * ways) * p.D + e);
        else
#pragma unroll
          for (int j = 0; j < kPart; ++j) w[i][j] = 0.f;
#pragma unroll
      for (int j = 0; j < kPart; ++j) sum[j] += ((w[0][j] + w[1][j]) + (w[2][j] + w[3][j])) + ((w[4][j] + w[5][j]) + (w[6][j] + w[7][j]));
    }
#pragma unroll
    for (int j = 0; j < kPart; ++j) held[way * p.D + e + j] = sum[j];
  }
  __syncthreads();
  for (int c = threadIdx.x; c < p.D; c += kThreads) {
    float s = 0.f;
    for (int w = 0; w < ways; ++w) s += held[w * p.D + c];
    h.dgamma[c] = s;
  }
}

// ---- host side ------------------------------------------------------------------------------------------------------------
// Elements that a piece of a chunk has, threads of a head, chunks of a thread: calls f with them as constants.
template <class F> void with_shape(int D, int pairs, uintptr_t bits, F&& f) {
  const int tail = D - 2 * pairs;
  auto at = [&](auto vec, auto l, auto n) { f(vec, l, n); };
#define TF_HEAD_SHAPE(V, L, N) at(std::integral_constant<int, V>(), std::integral_constant<int, L>(), std::integral_constant<int, N>())
  if (D % 4 == 0 && pairs % 4 == 0 && tail % 8 == 0 && bits % 16 == 0) {
    if (D <= 32) TF_HEAD_SHAPE(4, 4, 1); else if (D <= 64) TF_HEAD_SHAPE(4, 8, 1); else if (D <= 128) TF_HEAD_SHAPE(4, 16, 1); else TF_HEAD_SHAPE(4, 32, 1);
  } else if (D % 2 == 0 && pairs % 2 == 0 && tail % 4 == 0 && bits % 8 == 0) {
    if (D <= 32) TF_HEAD_SHAPE(2, 8, 1); else if (D <= 64) TF_HEAD_SHAPE(2, 16, 1); else if (D <= 128) TF_HEAD_SHAPE(2, 32, 1); else TF_HEAD_SHAPE(2, 32, 2);
  } else {
    if (D <= 32) TF_HEAD_SHAPE(1, 16, 1); else if (D <= 64) TF_HEAD_SHAPE(1, 32, 1); else if (D <= 128) TF_HEAD_SHAPE(1, 32, 2); else TF_HEAD_SHAPE(1, 32, 4);
  }
#undef TF_HEAD_SHAPE
}
uintptr_t bits_of(const void* p) { return reinterpret_cast<uintptr_t>(p); }       // of a null pointer: aligned

// Heads of a block's pass: all that U a thread make, fewer where that leaves SMs without a block.
int pass_of(int groups, int u, int64_t rows) {
  const int64_t even = (rows + 2 * device_sm_count() - 1) / (2 * device_sm_count());
  return (int)std::min<int64_t>((int64_t)groups * u, std::max<int64_t>(groups, (even + groups - 1) / groups * groups));
}
size_t turns_bytes(const RotaryArgs& a) {
  int most = 1;
  for (const HeadArgs& h : a.h) if (h.rows) most = std::max<int>(most, (int)std::min<int64_t>((a.per_block + h.heads - 2) / h.heads + 1, a.per_block));
  return sizeof(float2) * std::max<size_t>((size_t)most * a.pairs, kThreads * 4);         // dgamma's sums of the groups: at most 8 a thread
}
template <bool NORM> cudaError_t launch_heads(RotaryArgs a, const Quarters& f, cudaStream_t s) {
  uintptr_t bits = 0;
  for (const HeadArgs& h : a.h) bits |= bits_of(h.x) | bits_of(h.y) | bits_of(h.gamma);
  cudaError_t e = cudaSuccess;
  with_shape(a.D, a.pairs, bits, [&](auto vec, auto l, auto n) {
    constexpr int VEC = decltype(vec)::value, L = decltype(l)::value, N = decltype(n)::value, U = 4;
    a.chunks = (a.D + 2 * VEC - 1) / (2 * VEC);
    a.per_block = pass_of(kThreads / L, U, a.h[0].rows + a.h[1].rows);
    for (int i = 0; i < 2; ++i) a.blocks[i] = (int)((a.h[i].rows + a.per_block - 1) / a.per_block);
    e = launch_dep(heads_kernel<VEC, L, N, U, NORM>, dim3(a.blocks[0] + a.blocks[1]), dim3(kThreads), turns_bytes(a), s, a, f);
  });
  return e;
}

int check_rotary(const char* what, const RotaryState* st, const DLArray* x, const char* name, int64_t length, int64_t start, int64_t* tokens, int* heads) {
  TF_REQUIRE(st, "%s: the state was not made by TfRotaryState", what);
  TF_REQUIRE(x && x->ndim == 2, "%s: %s has to be a matrix of tokens by heads", what, name);
  TF_REQUIRE(x->shape[0] >= 0 && x->shape[1] >= 0 && x->shape[1] % st->D == 0, "%s: the columns of %s are not heads of %d elements", what, name, st->D);
  TF_REQUIRE(length >= 1 && start >= 0 && start < (1ll << 52), "%s: length has to be positive and start not negative", what);
  TF_REQUIRE(x->shape[0] < (1ll << 31) && x->shape[1] < (1ll << 31) && x->shape[0] * (x->shape[1] / st->D) < (1ll << 31), "%s: too many heads", what);
  *tokens = x->shape[0]; *heads = (int)(x->shape[1] / st->D);
  return 0;
}
RotaryArgs args_of(const RotaryState* st, const DLArray* positions, int64_t length, int64_t start, Quarters* f) {
  RotaryArgs a;
  memset(&a, 0, sizeof(a));
  a.positions = positions ? (const float*)positions->data : nullptr;
  a.length = std::min<int64_t>(length, 1ll << 31);                      // there are fewer tokens than that
  a.start = start; a.amplitude = st->amplitude; a.D = st->D; a.pairs = st->pairs; a.interleaved = st->interleaved;
  memcpy(f->of, st->quarters, sizeof(f->of));
  a.h[0].heads = a.h[1].heads = 1;
  return a;
}
int run_rotary(const char* what, const DLArray* in, const char* in_name, const DLArray* positions, DLArray* out, const char* out_name, int64_t length, int64_t start, void*** state,
               bool back, void** cudaStream) {
  const RotaryState* st = plan_of<RotaryState>(state, kPlanRotary);
  int64_t tokens;
  int heads;
  if (check_rotary(what, st, in, in_name, length, start, &tokens, &heads)) return -1;
  Operands o(what);
  o.add(in, in_name, -1, false); o.add(positions, "positions", tokens, false, true); o.add(out, out_name, numel(in), true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  Quarters f;
  RotaryArgs a = args_of(st, positions, length, start, &f);
  a.back = back;
  a.h[0].x = (const float*)in->data; a.h[0].y = out_f32(out); a.h[0].heads = heads; a.h[0].rows = tokens * heads;
  if (a.h[0].rows == 0) return 0;
  a.h[0].am = amax_track_begin(a.h[0].y);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 8.0 * numel(in));
  TF_CUDA(launch_heads<false>(a, f, s));
  TF_AFTER(s, what);
  return 0;
}

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" {

int TfRotaryState(int head_dim, int pairs, int interleaved, const double* frequencies, float amplitude, void*** state) {
  const char* const what = "TfRotaryState";
  TF_REQUIRE(state, "%s: null cell", what);
  TF_REQUIRE(head_dim >= 1 && head_dim <= kMostDim, "%s: heads of 1 to %d elements, not %d", what, kMostDim, head_dim);
  TF_REQUIRE(pairs >= 0 && 2 * pairs <= head_dim && (pairs == 0 || frequencies), "%s: %d pairs do not fit a head of %d elements", what, pairs, head_dim);
  TF_REQUIRE(interleaved == 0 || interleaved == 1, "%s: unknown layout %d", what, interleaved);
  TF_REQUIRE(std::isfinite(amplitude), "%s: the amplitude has to be finite", what);
  for (int i = 0; i < pairs; ++i) TF_REQUIRE(std::isfinite(frequencies[i]) && std::fabs(frequencies[i]) <= 1e3, "%s: frequency %d is not a number of radians a position", what, i);
  RotaryState* st = plan_of<RotaryState>(state, kPlanRotary);
  TF_REQUIRE(st || !holds_plan(state), "%s: the cell holds another descriptor", what);
  if (!st) st = new_plan<RotaryState>(state, kPlanRotary, 1);
  st->D = head_dim; st->pairs = pairs; st->interleaved = interleaved; st->amplitude = amplitude;
  for (int i = 0; i < kMostPairs; ++i) st->quarters[i] = i < pairs ? frequencies[i] * 0.63661977236758134 : 0.0;
  return 0;
}

int TfRotaryForward(const DLArrayHandle input, const DLArrayHandle positions, DLArrayHandle output, int64_t length, int64_t start, void*** state, void** cudaStream) {
  return run_rotary("TfRotaryForward", input, "input", positions, output, "output", length, start, state, false, cudaStream);
}

int TfRotaryBackward(const DLArrayHandle doutput, const DLArrayHandle positions, DLArrayHandle dinput, int64_t length, int64_t start, void*** state, void** cudaStream) {
  return run_rotary("TfRotaryBackward", doutput, "doutput", positions, dinput, "dinput", length, start, state, true, cudaStream);
}

int TfHeadNormRotaryForward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle gamma_query, const DLArrayHandle gamma_key, const DLArrayHandle positions,
                            DLArrayHandle query_out, DLArrayHandle key_out, int64_t length, int64_t start, float eps, void*** state, void** cudaStream) {
  const char* const what = "TfHeadNormRotaryForward";
  const RotaryState* st = plan_of<RotaryState>(state, kPlanRotary);
  int64_t tokens, key_tokens = 0;
  int heads, key_heads = 1;
  if (check_rotary(what, st, query, "query", length, start, &tokens, &heads)) return -1;
  TF_REQUIRE(eps >= 0.f && eps < INFINITY, "%s: eps has to be finite and not negative", what);
  TF_REQUIRE(!key == !gamma_key && !key == !key_out, "%s: key, gamma_key and key_out go together", what);
  if (key && check_rotary(what, st, key, "key", length, start, &key_tokens, &key_heads)) return -1;
  TF_REQUIRE(!key || key_tokens == tokens, "%s: query and key are of different tokens", what);
  Operands o(what);
  o.add(query, "query", -1, false); o.add(key, "key", -1, false, true); o.add(gamma_query, "gamma_query", st->D, false); o.add(gamma_key, "gamma_key", st->D, false, true);
  o.add(positions, "positions", tokens, false, true); o.add(query_out, "query_out", numel(query), true); o.add(key_out, "key_out", key ? numel(key) : 0, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  Quarters f;
  RotaryArgs a = args_of(st, positions, length, start, &f);
  a.eps = eps;
  a.h[0].x = (const float*)query->data; a.h[0].gamma = (const float*)gamma_query->data; a.h[0].y = out_f32(query_out); a.h[0].heads = heads; a.h[0].rows = tokens * heads;
  if (key) { a.h[1].x = (const float*)key->data; a.h[1].gamma = (const float*)gamma_key->data; a.h[1].y = out_f32(key_out); a.h[1].heads = key_heads; a.h[1].rows = tokens * key_heads; }
  if (a.h[0].rows + a.h[1].rows == 0) return 0;
  for (HeadArgs& h : a.h) if (h.rows) h.am = amax_track_begin(h.y);
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 8.0 * (a.h[0].rows + a.h[1].rows) * a.D);
  TF_CUDA(launch_heads<true>(a, f, s));
  TF_AFTER(s, what);
  return 0;
}

int TfHeadNormRotaryBackward(const DLArrayHandle query, const DLArrayHandle key, const DLArrayHandle gamma_query, const DLArrayHandle gamma_key, const DLArrayHandle positions,
                             const DLArrayHandle dquery_out, const DLArrayHandle dkey_out, DLArrayHandle dquery, DLArrayHandle dkey, DLArrayHandle dgamma_query,
                             DLArrayHandle dgamma_key, int64_t length, int64_t start, float eps, void*** state, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfHeadNormRotaryBackward";
  const RotaryState* st = plan_of<RotaryState>(state, kPlanRotary);
  int64_t tokens, key_tokens = 0;
  int heads, key_heads = 1;
  if (check_rotary(what, st, query, "query", length, start, &tokens, &heads)) return -1;
  TF_REQUIRE(eps >= 0.f && eps < INFINITY, "%s: eps has to be finite and not negative", what);
  TF_REQUIRE(!key == !gamma_key && !key == !dkey_out && (key || (!dkey && !dgamma_key)), "%s: key, gamma_key and dkey_out go together", what);
  if (key && check_rotary(what, st, key, "key", length, start, &key_tokens, &key_heads)) return -1;
  TF_REQUIRE(!key || key_tokens == tokens, "%s: query and key are of different tokens", what);
  Operands o(what);
  const int64_t nq = numel(query), nk = key ? numel(key) : 0;
  o.add(query, "query", -1, false); o.add(key, "key", -1, false, true); o.add(gamma_query, "gamma_query", st->D, false); o.add(gamma_key, "gamma_key", st->D, false, true);
  o.add(positions, "positions", tokens, false, true); o.add(dquery_out, "dquery_out", nq, false); o.add(dkey_out, "dkey_out", nk, false, true);
  o.add(dquery, "dquery", nq, true, true); o.add(dkey, "dkey", nk, true, true); o.add(dgamma_query, "dgamma_query", st->D, true, true); o.add(dgamma_key, "dgamma_key", st->D, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  Quarters f;
  RotaryArgs a = args_of(st, positions, length, start, &f);
  a.eps = eps;
  a.h[0].x = (const float*)query->data; a.h[0].gamma = (const float*)gamma_query->data; a.h[0].dy = (const float*)dquery_out->data;
  a.h[0].y = dquery ? out_f32(dquery) : nullptr; a.h[0].dgamma = dgamma_query ? out_f32(dgamma_query) : nullptr; a.h[0].heads = heads; a.h[0].rows = tokens * heads;
  if (key) {
    a.h[1].x = (const float*)key->data; a.h[1].gamma = (const float*)gamma_key->data; a.h[1].dy = (const float*)dkey_out->data;
    a.h[1].y = dkey ? out_f32(dkey) : nullptr; a.h[1].dgamma = dgamma_key ? out_f32(dgamma_key) : nullptr; a.h[1].heads = key_heads; a.h[1].rows = tokens * key_heads;
  }
  note_compute_stream(s);
  for (HeadArgs& h : a.h) {
    if (h.rows == 0 && h.dgamma) TF_CUDA(clear_on_stream(h.dgamma, sizeof(float) * st->D, s));
    if (!h.y && !h.dgamma) h.rows = 0;
  }
  const int64_t rows = a.h[0].rows + a.h[1].rows;
  if (rows == 0) return 0;
  StreamLease lease(s);
  // Four blocks an SM with one head a thread group and pass: 94 to 100 us by box at 16384 tokens x (16 + 4) heads of 128, 5.0 to 5.3 TB/s.  More in flight is slower, reads and writes
  // get in one another's way: three or four blocks of two heads 98 and 115, five of one 106, the next pass asked for in advance 115.
  const int64_t most = kNormBlocks * device_sm_count();
  const size_t bytes = sizeof(float) * (size_t)(most + 1) * a.D;
  float* const part = (float*)lease.scratch(kScratchNorm, bytes);
  uint32_t* const count = part ? lease.counters(2) : nullptr;
  if (!count) { if (memorytoSaving) *memorytoSaving = (int)bytes; return 0; }
  uintptr_t bits = 0;
  for (const HeadArgs& h : a.h) bits |= bits_of(h.x) | bits_of(h.y) | bits_of(h.gamma) | bits_of(h.dy);
  KernelTimer kt(what, s, 0, 12.0 * rows * a.D);
  cudaError_t e = cudaSuccess;
  with_shape(a.D, a.pairs, bits, [&](auto vec, auto l, auto n) {
    constexpr int VEC = decltype(vec)::value, L = decltype(l)::value, N = decltype(n)::value, U = 1;
    a.chunks = (a.D + 2 * VEC - 1) / (2 * VEC);
    a.per_block = pass_of(kThreads / L, U, rows);
    int64_t passes[2], all = 0;
    for (int i = 0; i < 2; ++i) all += passes[i] = (a.h[i].rows + a.per_block - 1) / a.per_block;
    for (int i = 0; i < 2; ++i)                      // shares of the blocks by shares of the passes
      a.blocks[i] = !passes[i] ? 0 : all <= most ? (int)passes[i] : (int)std::max<int64_t>(1, std::min<int64_t>(passes[i], most * passes[i] / all));
    for (int i = 0; i < 2; ++i) {
      a.h[i].part = part + (i ? (size_t)a.blocks[0] * a.D : 0); a.h[i].count = count + i;
      if (a.h[i].rows && a.h[i].y) a.h[i].am = amax_track_begin(a.h[i].y);
    }
    e = launch_dep(head_norm_bwd_kernel<VEC, L, N, U>, dim3(a.blocks[0] + a.blocks[1]), dim3(kThreads), turns_bytes(a), s, a, f);
  });
  TF_CUDA(e);
  TF_AFTER(s, what);
  return 0;
}

}  // extern "C"
