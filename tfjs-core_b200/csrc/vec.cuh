// V consecutive float32, half or byte values of a row as float32 registers, in one access where the
// address allows it (V * the element's size <= 16 bytes; the caller sees to the alignment), and the
// sums over lanes that the row kernels share.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace {

// ---- V consecutive values as float32 -----------------------------------------------------------
template <int V>
__device__ __forceinline__ void load_vec(const float* p, float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) {
      const float4 q = *reinterpret_cast<const float4*>(p + i);
      v[i] = q.x; v[i + 1] = q.y; v[i + 2] = q.z; v[i + 3] = q.w;
    }
  } else if constexpr (V == 2) {
    const float2 q = *reinterpret_cast<const float2*>(p);
    v[0] = q.x; v[1] = q.y;
  } else {
    v[0] = *p;
  }
}
__device__ __forceinline__ void widen2(uint32_t h, float& a, float& b) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
  a = f.x; b = f.y;
}
__device__ __forceinline__ uint32_t narrow2(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
// A 4-byte word as the values it holds.
__device__ __forceinline__ void unpack_word(uint32_t q, const float*, float (&v)[1]) { v[0] = __uint_as_float(q); }
__device__ __forceinline__ void unpack_word(uint32_t q, const __half*, float (&v)[2]) { widen2(q, v[0], v[1]); }
template <int V>
__device__ __forceinline__ void load_vec(const __half* p, float (&v)[V]) {
  if constexpr (V == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    widen2(q.x, v[0], v[1]); widen2(q.y, v[2], v[3]); widen2(q.z, v[4], v[5]); widen2(q.w, v[6], v[7]);
  } else if constexpr (V == 4) {
    const uint2 q = *reinterpret_cast<const uint2*>(p);
    widen2(q.x, v[0], v[1]); widen2(q.y, v[2], v[3]);
  } else if constexpr (V == 2) {
    widen2(*reinterpret_cast<const uint32_t*>(p), v[0], v[1]);
  } else {
    v[0] = __half2float(*p);
  }
}
template <int V>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) *reinterpret_cast<float4*>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  } else if constexpr (V == 2) {
    *reinterpret_cast<float2*>(p) = make_float2(v[0], v[1]);
  } else {
    *p = v[0];
  }
}
template <int V>
__device__ __forceinline__ void store_vec(__half* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    *reinterpret_cast<uint4*>(p) = make_uint4(narrow2(v[0], v[1]), narrow2(v[2], v[3]), narrow2(v[4], v[5]), narrow2(v[6], v[7]));
  } else if constexpr (V == 4) {
    *reinterpret_cast<uint2*>(p) = make_uint2(narrow2(v[0], v[1]), narrow2(v[2], v[3]));
  } else if constexpr (V == 2) {
    *reinterpret_cast<uint32_t*>(p) = narrow2(v[0], v[1]);
  } else {
    *p = __float2half_rn(v[0]);
  }
}

// The same with an evict-first hint, for results so large (kStreamBytes and more, where L2 holds 126 MB) that
// whoever reads them next finds little of them in L2 anyway.
constexpr int64_t kStreamBytes = 96ll << 20;
template <int V>
__device__ __forceinline__ void store_vec_stream(float* p, const float (&v)[V]) {
  if constexpr (V % 4 == 0) {
#pragma unroll
    for (int i = 0; i < V; i += 4) __stcs(reinterpret_cast<float4*>(p + i), make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]));
  } else if constexpr (V == 2) {
    __stcs(reinterpret_cast<float2*>(p), make_float2(v[0], v[1]));
  } else {
    __stcs(p, v[0]);
  }
}
template <int V>
__device__ __forceinline__ void store_vec_stream(__half* p, const float (&v)[V]) {
  if constexpr (V == 8) {
    __stcs(reinterpret_cast<uint4*>(p), make_uint4(narrow2(v[0], v[1]), narrow2(v[2], v[3]), narrow2(v[4], v[5]), narrow2(v[6], v[7])));
  } else if constexpr (V == 4) {
    __stcs(reinterpret_cast<uint2*>(p), make_uint2(narrow2(v[0], v[1]), narrow2(v[2], v[3])));
  } else if constexpr (V == 2) {
    __stcs(reinterpret_cast<uint32_t*>(p), narrow2(v[0], v[1]));
  } else {
    __stcs(reinterpret_cast<unsigned short*>(p), __half_as_ushort(__float2half_rn(v[0])));
  }
}

template <int L>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace
