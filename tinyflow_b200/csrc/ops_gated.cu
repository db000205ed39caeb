// Gated dense layer: out = act(x Wg) * (x Wv) with both weights side by side, W = [Wg | Wv] of K x 2F, and its gradients.
//
//   z = x W (M x 2F),  out = act(zg) * zv
//   dzg = dout * zv * act'(zg),  dzv = dout * act(zg),  dx = dz W^T,  dW = x^T dz
//
// Both projections are one product of 2F columns, 4 MKF operations; the gradients are two products of dz, 8 MKF.
#include "common.h"
#include <math.h>
#include <algorithm>
#include <cmath>
#include <type_traits>
#include "gated.h"
#include "operands.h"
#include "pieces.h"

namespace tf {

int matmul_any(const float* A, bool tA, const float* B, bool tB, float* C, int64_t M, int64_t N, int64_t K, cudaStream_t s, const char* what);
int tc_gated_fwd(const float* x, const float* w, float* gates, float* out, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s, const char* what);
int tc_gated_bwd(const float* x, const float* w, const float* z, const float* dout, float* dx, float* dw, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s, const char* what);
int rows_gated(const float* x, const float* w, float* gates, float* out, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s);
bool rows_gated_bwd_takes(int64_t M, int64_t F, int64_t K);
int rows_gated_bwd(const float* x, const float* w, const float* dz, float* dx, float* dw, int64_t M, int64_t F, int64_t K, cudaStream_t s);
int gated_small_fwd(const float* x, const float* w, float* gates, float* out, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s, const char* what);
bool gated_small_bwd_takes(int64_t M, int64_t F, int64_t K);
int gated_small_bwd(const float* x, const float* w, const float* z, const float* dout, float* dx, float* dw, int64_t M, int64_t F, int64_t K, int activation, cudaStream_t s, const char* what);
void note_contraction_path(int path);
bool pause_holding();                    // what follows is not to wait; returns whether it could have
void hold_products(bool on);

namespace {

constexpr int kThreads = 256;
// HBM-bound: 12 bytes per output.
template <int ACT, int VEC>
__global__ void __launch_bounds__(kThreads) gate_kernel(const float* __restrict__ z, float* __restrict__ out, int64_t rows, int F, AmaxOut am) {
  grid_dep_sync();
  uint32_t m = 0;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float* const zr = z + row * 2 * F;
    for (int c = ((int)blockIdx.x * kThreads + threadIdx.x) * VEC; c < F; c += (int)gridDim.x * kThreads * VEC) {
      float g[VEC], v[VEC];
      get<VEC>(g, zr + c);
      get<VEC>(v, zr + F + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) { v[j] *= gate_value<ACT>(g[j]); m = max(m, amax_key(v[j])); }
      put<VEC>(out + row * F + c, v);
    }
  }
  amax_commit(am, m);
}
// HBM-bound: 20 bytes per output of the layer.
template <int ACT, int VEC>
__global__ void __launch_bounds__(kThreads) gate_gradient_kernel(const float* __restrict__ z, const float* __restrict__ dout, float* __restrict__ dz, int64_t rows, int F, AmaxOut am) {
  grid_dep_sync();
  uint32_t m = 0;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const int64_t at = row * 2 * F;
    for (int c = ((int)blockIdx.x * kThreads + threadIdx.x) * VEC; c < F; c += (int)gridDim.x * kThreads * VEC) {
      float g[VEC], v[VEC], d[VEC];
      get<VEC>(g, z + at + c);
      get<VEC>(v, z + at + F + c);
      get<VEC>(d, dout + row * F + c);
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        float value, slope;
        gate_slope<ACT>(g[j], value, slope);
        g[j] = d[j] * v[j] * slope;
        v[j] = d[j] * value;
        m = max(m, max(amax_key(g[j]), amax_key(v[j])));
      }
      put<VEC>(dz + at + c, g);
      put<VEC>(dz + at + F + c, v);
    }
  }
  amax_commit(am, m);
}

dim3 gate_grid(int64_t rows, int F, int vec) {
  const int across = (F + kThreads * vec - 1) / (kThreads * vec);
  const int64_t down = std::max<int64_t>(1, (int64_t)16 * device_sm_count() / across);
  return dim3((unsigned)across, (unsigned)std::min<int64_t>(std::min<int64_t>(rows, 65535), down));
}
cudaError_t launch_gate(int activation, const float* z, float* out, int64_t rows, int F, AmaxOut am, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  with_gate(activation, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (F % 4 == 0 && aligned16(z) && aligned16(out)) e = launch_dep(gate_kernel<ACT, 4>, gate_grid(rows, F, 4), dim3(kThreads), 0, s, z, out, rows, F, am);
    else e = launch_dep(gate_kernel<ACT, 1>, gate_grid(rows, F, 1), dim3(kThreads), 0, s, z, out, rows, F, am);
  });
  return e;
}
cudaError_t launch_gate_gradient(int activation, const float* z, const float* dout, float* dz, int64_t rows, int F, AmaxOut am, cudaStream_t s) {
  cudaError_t e = cudaSuccess;
  with_gate(activation, [&](auto act) {
    constexpr int ACT = decltype(act)::value;
    if (F % 4 == 0 && aligned16(z) && aligned16(dout) && aligned16(dz)) e = launch_dep(gate_gradient_kernel<ACT, 4>, gate_grid(rows, F, 4), dim3(kThreads), 0, s, z, dout, dz, rows, F, am);
    else e = launch_dep(gate_gradient_kernel<ACT, 1>, gate_grid(rows, F, 1), dim3(kThreads), 0, s, z, dout, dz, rows, F, am);
  });
  return e;
}

// Whether the tensor path is the shorter road, in us.  It costs a chain of launches and the traffic of the packs before the first product; the
// CUDA-core kernels cost per multiply-add, more of it where rows cannot be read 16 bytes at a time, and for long reductions over few tiles a
// chain of steps.  Fitted to 600 shapes of 16 to 8192 rows and 16 to 8192 columns with up to 3e9 multiply-adds, on which the road it takes is
// on average 0.6 % slower than the better one, backward 1.2 % (at most 1.4 and 1.6 times).  Tensor path against CUDA cores: 512 x 512 x 512 forward
// 19.9 us against 24.7, backward 33.9 against 68.7; 64 x 512 x 1024 19.1 against 9.2 and 26.5 against 24.6; 4000 x 128 x 128 16.1 against 13.2 and
// 29.9 against 43.6; 437 x 28 x 5560 backward 40 against 183.
bool tensor_path_pays(int64_t rows, int64_t outputs, int64_t inputs, bool backward) {
  const double M = (double)rows, F = (double)outputs, K = (double)inputs, work = 2.0 * M * F * K, sms = device_sm_count();
  const bool odd = outputs % 4 || inputs % 4;
  const auto tiles = [](double a, double b, double of) { return std::ceil(a / 32) * std::ceil(b / of); };
  if (!backward) {
    const double whole = 2048.0 * tiles(M, F, 32) * K;                       // multiply-adds of whole tiles
    return work > 3e8 || 15.2 + 0.0026 * K + 1e-6 * (2.3 * M * K + 3.85 * K * F + 5.1 * M * F) < 5.5 + (odd ? 9.6e-8 : 8e-8) * whole;
  }
  const double tensor = 23.2 + 1.4e-8 * work + 1e-6 * (3.9 * M * K + 8.6 * K * F + 11.5 * M * F) + (odd ? 4.6 : 0.0);
  if (rows <= 16 && !odd && 2.0 * F * K >= 1e6) return tensor < 5.0 + 3.5e-7 * work;                // the products have kernels for those
  if (!gated_small_bwd_takes(rows, outputs, inputs)) return tensor < 10.0 + 0.006 * F + (odd ? 6e-7 : 4e-7) * work;
  const double cut_dw = std::min(16.0, std::max(1.0, sms / tiles(K, F, 16))), cut_dx = std::min(16.0, std::max(1.0, sms / tiles(M, K, 32)));
  return tensor < 5.0 + (odd ? 1.6 : 1.0) * std::max(3.2e-7 * work, std::max(0.02 * M / cut_dw, 0.08 * F / cut_dx));
}

// Products of scratch are launched at once, whatever the caller holds back.
struct NoHolding {
  const bool held;
  NoHolding() : held(pause_holding()) {}
  ~NoHolding() { if (held) hold_products(true); }
};
int short_of(size_t bytes, int* memorytoSaving) {
  if (memorytoSaving) *memorytoSaving = bytes > 0x7fffffffu ? 0x7fffffff : (int)bytes;
  return 0;
}
int check_gated(const char* what, const DLArray* x, const DLArray* weight, int activation, int64_t* M, int64_t* K, int64_t* F) {
  TF_REQUIRE(x && x->ndim == 2 && weight && weight->ndim == 2, "%s: input and weight have to be matrices", what);
  TF_REQUIRE(weight->shape[1] % 2 == 0, "%s: the weight holds two halves of its columns, and %lld is odd", what, (long long)weight->shape[1]);
  TF_REQUIRE(is_gate(activation), "%s: unknown activation %d", what, activation);
  *M = x->shape[0]; *K = x->shape[1]; *F = weight->shape[1] / 2;
  TF_REQUIRE(weight->shape[0] == *K, "%s: inner extents differ (%lld vs %lld)", what, (long long)*K, (long long)weight->shape[0]);
  TF_REQUIRE(*M >= 0 && *K >= 0 && *F >= 0 && *M < (1ll << 31) && *K < (1ll << 31) && *F < (1ll << 30), "%s: extent too large", what);
  return 0;
}
int check_matrix(const char* what, const char* name, const DLArray* a, int64_t rows, int64_t cols) {
  TF_REQUIRE(!a || (a->ndim == 2 && a->shape[0] == rows && a->shape[1] == cols), "%s: %s has to be %lld x %lld", what, name, (long long)rows, (long long)cols);
  return 0;
}

}  // namespace
}  // namespace tf

using namespace tf;

extern "C" {

int TfGatedLinearForward(const DLArrayHandle input, const DLArrayHandle weight, DLArrayHandle gates, DLArrayHandle output, int activation, int* memorytoSaving,
                         void** cudaStream) {
  const char* const what = "TfGatedLinearForward";
  int64_t M, K, F;
  if (check_gated(what, input, weight, activation, &M, &K, &F) || check_matrix(what, "gates", gates, M, 2 * F) || check_matrix(what, "output", output, M, F)) return -1;
  Operands o(what);
  o.add(input, "input", M * K, false); o.add(weight, "weight", K * 2 * F, false); o.add(gates, "gates", M * 2 * F, true, true); o.add(output, "output", M * F, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  float* const out = out_f32(output);
  float* z = gates ? out_f32(gates) : nullptr;
  if (M == 0 || F == 0) return 0;
  const NoHolding launched;
  if (contraction_path() == 0) {           // (up to 16 rows against large weights)
    if (const int r = rows_gated((const float*)input->data, (const float*)weight->data, z, out, M, F, K, activation, s)) { note_contraction_path(1); return r < 0 ? -1 : 0; }
  }
  if (contraction_path() == 2 || (contraction_path() == 0 && tensor_path_pays(M, F, K, false))) {
    if (const int r = tc_gated_fwd((const float*)input->data, (const float*)weight->data, z, out, M, F, K, activation, s, what)) {
      note_contraction_path(2);
      return r < 0 ? -1 : 0;
    }
  }
  if (contraction_path() != 2) {
    int r = contraction_path() == 1 ? rows_gated((const float*)input->data, (const float*)weight->data, z, out, M, F, K, activation, s) : 0;
    if (!r) r = gated_small_fwd((const float*)input->data, (const float*)weight->data, z, out, M, F, K, activation, s, what);
    if (r) { note_contraction_path(1); return r < 0 ? -1 : 0; }
  }
  StreamLease lease(s);
  const size_t bytes = sizeof(float) * (size_t)M * 2 * F;
  if (!z && !(z = (float*)lease.scratch(kScratchGates, bytes))) return short_of(bytes, memorytoSaving);
  if (matmul_any((const float*)input->data, false, (const float*)weight->data, false, z, M, 2 * F, K, s, what)) return -1;
  note_compute_stream(s);
  KernelTimer kt(what, s, 0, 12.0 * M * F);
  TF_CUDA(launch_gate(activation, z, out, M, (int)F, amax_track_begin(out), s));
  TF_AFTER(s, what);
  return 0;
}

int TfGatedLinearBackward(const DLArrayHandle input, const DLArrayHandle weight, const DLArrayHandle gates, const DLArrayHandle doutput, DLArrayHandle dinput,
                          DLArrayHandle dweight, int activation, int* memorytoSaving, void** cudaStream) {
  const char* const what = "TfGatedLinearBackward";
  int64_t M, K, F;
  if (check_gated(what, input, weight, activation, &M, &K, &F) || check_matrix(what, "gates", gates, M, 2 * F) || check_matrix(what, "doutput", doutput, M, F) ||
      check_matrix(what, "dinput", dinput, M, K) || check_matrix(what, "dweight", dweight, K, 2 * F)) return -1;
  Operands o(what);
  o.add(input, "input", M * K, false); o.add(weight, "weight", K * 2 * F, false); o.add(gates, "gates", M * 2 * F, false); o.add(doutput, "doutput", M * F, false);
  o.add(dinput, "dinput", M * K, true, true); o.add(dweight, "dweight", K * 2 * F, true, true);
  if (!o.ok) return -1;
  cudaStream_t s = stream_of(cudaStream);
  float *dx = dinput ? out_f32(dinput) : nullptr, *dw = dweight ? out_f32(dweight) : nullptr;
  if (!dx && !dw) return 0;
  const NoHolding launched;
  const bool few_rows = rows_gated_bwd_takes(M, F, K);
  if (contraction_path() == 2 || (contraction_path() == 0 && !few_rows && tensor_path_pays(M, F, K, true))) {
    if (const int r = tc_gated_bwd((const float*)input->data, (const float*)weight->data, (const float*)gates->data, (const float*)doutput->data, dx, dw, M, F, K, activation, s, what)) {
      note_contraction_path(2);
      return r < 0 ? -1 : 0;
    }
  }
  if (contraction_path() != 2 && !few_rows) {
    if (const int r = gated_small_bwd((const float*)input->data, (const float*)weight->data, (const float*)gates->data, (const float*)doutput->data, dx, dw, M, F, K, activation, s, what)) {
      note_contraction_path(1);
      return r < 0 ? -1 : 0;
    }
  }
  StreamLease lease(s);
  const size_t bytes = sizeof(float) * (size_t)std::max<int64_t>(1, M * 2 * F);
  float* const dz = (float*)lease.scratch(kScratchGates, bytes);
  if (!dz) return short_of(bytes, memorytoSaving);
  note_compute_stream(s);
  note_write(dz);                        // scratch: whatever was known of an array at this address does not hold
  if (M && F) {
    KernelTimer kt(what, s, 0, 20.0 * M * F);
    TF_CUDA(launch_gate_gradient(activation, (const float*)gates->data, (const float*)doutput->data, dz, M, (int)F, amax_track_begin(dz), s));
    TF_AFTER(s, what);
  }
  if (few_rows && contraction_path() != 2) {
    if (const int r = rows_gated_bwd((const float*)input->data, (const float*)weight->data, dz, dx, dw, M, F, K, s)) { note_contraction_path(1); note_write(dz); return r < 0 ? -1 : 0; }
  }
  if (dx && matmul_any(dz, false, (const float*)weight->data, true, dx, M, K, 2 * F, s, what)) return -1;
  if (dw && matmul_any((const float*)input->data, true, dz, false, dw, K, 2 * F, M, s, what)) return -1;
  note_write(dz);
  return 0;
}

}  // extern "C"
