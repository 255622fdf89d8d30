// norm_rope.cuh — what the per-head norm + rotation and the gradients of both
// norms share: typed 16-byte loads of 8 channels, weights, and the sum of
// per-block partial rows.
#pragma once

#include <cuda_fp16.h>

#include "sa_common.cuh"

namespace sa {
namespace nr {

// 8 consecutive channels as they lie in memory: one 16-byte vector of a 16-bit
// type, two of fp32.
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i)
    r.v[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}

__device__ __forceinline__ void unpack8(const Raw8<__nv_bfloat16>& r, float (&x)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r.v[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(w[i] << 16);
    x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
  }
}
__device__ __forceinline__ void unpack8(const Raw8<__half>& r, float (&x)[8]) {
  const __half2* w = reinterpret_cast<const __half2*>(&r.v[0]);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(w[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack8(const Raw8<float>& r, float (&x)[8]) {
  const float* w = reinterpret_cast<const float*>(&r.v[0]);
#pragma unroll
  for (int i = 0; i < 8; ++i) x[i] = w[i];
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                            pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(__half* p, const float (&x)[8]) {
  uint4 o;
  __half2* w = reinterpret_cast<__half2*>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = o;
}
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

// Channels c0..c0+7 of a weight vector of any of the three types (1 without).
__device__ __forceinline__ void load_weight8(const void* w, int dtype, int c0, float (&x)[8]) {
  if (w == nullptr) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = 1.f;
  } else if (dtype == SA_DTYPE_BF16) {
    Raw8<__nv_bfloat16> r;
    r.v[0] = __ldg(reinterpret_cast<const uint4*>(w) + (c0 >> 3));
    unpack8(r, x);
  } else if (dtype == SA_DTYPE_FP16) {
    Raw8<__half> r;
    r.v[0] = __ldg(reinterpret_cast<const uint4*>(w) + (c0 >> 3));
    unpack8(r, x);
  } else {
    Raw8<float> r;
    r.v[0] = __ldg(reinterpret_cast<const uint4*>(w) + (c0 >> 2));
    r.v[1] = __ldg(reinterpret_cast<const uint4*>(w) + (c0 >> 2) + 1);
    unpack8(r, x);
  }
}

// out[c] = sum over `rows` partial rows of part[row * pitch + c], c < cols, in a
// fixed order (the same bits on every run); columns below cols0 go to out0,
// the rest to out1.
int sum_partial_rows(const float* part, int rows, int cols, int pitch, float* out0, float* out1,
                     int cols0, cudaStream_t stream);

}  // namespace nr
}  // namespace sa
