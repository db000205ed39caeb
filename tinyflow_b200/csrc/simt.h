// Operands of the exact-fp32 matrix products on CUDA cores.
#pragma once
#include "common.h"

namespace tf {

struct SimtGemm {
  const float* A; const float* B; float* C;
  int M, N, K;
  long long lda, ldb, ldc;
  int k_per_cta;            // multiple of BK
  int a_vec, b_vec, c_vec;  // 16-byte accesses allowed
};

// One BMxBK (or BKxBN) block of an operand: `rows` index M (or N), `k` the reduction.  KFAST: k is contiguous in memory.
// A thread moves VPT groups of four elements along the contiguous direction.
template <int ROWS, int BK, int THREADS, bool KFAST> struct BlockLoader {
  static constexpr int kGroups = ROWS * BK / 4;
  static constexpr int VPT = (kGroups + THREADS - 1) / THREADS;
  float4 v[VPT];
  __device__ __forceinline__ void fetch(const float* __restrict__ p, long long ld, int row0, int rows, int k0, int k1, bool vec) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = threadIdx.x + i * THREADS;
      v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (kGroups % THREADS && g >= kGroups) continue;
      if (KFAST) {
        const int r = row0 + g / (BK / 4), k = k0 + (g % (BK / 4)) * 4;
        if (r >= rows || k >= k1) continue;
        const float* q = p + (long long)r * ld + k;
        if (vec && k + 4 <= k1) v[i] = __ldg(reinterpret_cast<const float4*>(q));
        else { v[i].x = __ldg(q); if (k + 1 < k1) v[i].y = __ldg(q + 1); if (k + 2 < k1) v[i].z = __ldg(q + 2); if (k + 3 < k1) v[i].w = __ldg(q + 3); }
      } else {
        const int k = k0 + g / (ROWS / 4), r = row0 + (g % (ROWS / 4)) * 4;
        if (r >= rows || k >= k1) continue;
        const float* q = p + (long long)k * ld + r;
        if (vec && r + 4 <= rows) v[i] = __ldg(reinterpret_cast<const float4*>(q));
        else { v[i].x = __ldg(q); if (r + 1 < rows) v[i].y = __ldg(q + 1); if (r + 2 < rows) v[i].z = __ldg(q + 2); if (r + 3 < rows) v[i].w = __ldg(q + 3); }
      }
    }
  }
  // into s[k][row], row pitch ROWS + 4: 16-byte aligned rows for the vector reads
  __device__ __forceinline__ void put(float (*s)[ROWS + 4]) const {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int g = threadIdx.x + i * THREADS;
      if (kGroups % THREADS && g >= kGroups) continue;
      if (KFAST) {
        const int r = g / (BK / 4), k = (g % (BK / 4)) * 4;
        s[k][r] = v[i].x; s[k + 1][r] = v[i].y; s[k + 2][r] = v[i].z; s[k + 3][r] = v[i].w;
      } else {
        *reinterpret_cast<float4*>(&s[g / (ROWS / 4)][(g % (ROWS / 4)) * 4]) = v[i];
      }
    }
  }
};

}  // namespace tf
