// Accesses of VEC elements at once.
#pragma once

namespace tf {

#ifdef __CUDACC__
template <int VEC> struct Pieces;
template <> struct Pieces<4> { typedef float4 T; };
template <> struct Pieces<2> { typedef float2 T; };
template <> struct Pieces<1> { typedef float T; };
template <int VEC> __device__ __forceinline__ void get(float* v, const float* __restrict__ p) { *reinterpret_cast<typename Pieces<VEC>::T*>(v) = __ldg(reinterpret_cast<const typename Pieces<VEC>::T*>(p)); }
template <int VEC> __device__ __forceinline__ void held_at(float* v, const float* p) { *reinterpret_cast<typename Pieces<VEC>::T*>(v) = *reinterpret_cast<const typename Pieces<VEC>::T*>(p); }
template <int VEC> __device__ __forceinline__ void put(float* p, const float* v) { *reinterpret_cast<typename Pieces<VEC>::T*>(p) = *reinterpret_cast<const typename Pieces<VEC>::T*>(v); }
#endif

}  // namespace tf
