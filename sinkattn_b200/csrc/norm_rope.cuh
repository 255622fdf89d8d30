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

template <typename T>
__device__ __forceinline__ Raw8<T> shfl8(const Raw8<T>& r, int src) {
  Raw8<T> o;
#pragma unroll
  for (int i = 0; i < (int)(sizeof(T) / 2); ++i) {
    o.v[i].x = __shfl_sync(0xffffffffu, r.v[i].x, src);
    o.v[i].y = __shfl_sync(0xffffffffu, r.v[i].y, src);
    o.v[i].z = __shfl_sync(0xffffffffu, r.v[i].z, src);
    o.v[i].w = __shfl_sync(0xffffffffu, r.v[i].w, src);
  }
  return o;
}

// The 8 channels as four f32x2 values for the packed arithmetic, even and odd
// channels apart: v[0] = (0, 2), v[1] = (1, 3), v[2] = (4, 6), v[3] = (5, 7).
struct V8 {
  uint64_t v[4];
};

__device__ __forceinline__ V8 planar(const float (&x)[8]) {
  return V8{{f2_pack(x[0], x[2]), f2_pack(x[1], x[3]), f2_pack(x[4], x[6]), f2_pack(x[5], x[7])}};
}
__device__ __forceinline__ void channels(const V8& a, float (&x)[8]) {
  f2_unpack(a.v[0], x[0], x[2]);
  f2_unpack(a.v[1], x[1], x[3]);
  f2_unpack(a.v[2], x[4], x[6]);
  f2_unpack(a.v[3], x[5], x[7]);
}

__device__ __forceinline__ V8 unpack8(const Raw8<__nv_bfloat16>& r) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&r.v[0]);
  V8 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    o.v[2 * i] = f2_pack(__uint_as_float(w[2 * i] << 16), __uint_as_float(w[2 * i + 1] << 16));
    o.v[2 * i + 1] = f2_pack(__uint_as_float(w[2 * i] & 0xffff0000u),
                             __uint_as_float(w[2 * i + 1] & 0xffff0000u));
  }
  return o;
}
__device__ __forceinline__ V8 unpack8(const Raw8<__half>& r) {
  const __half2* w = reinterpret_cast<const __half2*>(&r.v[0]);
  V8 o;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float2 a = __half22float2(w[2 * i]), b = __half22float2(w[2 * i + 1]);
    o.v[2 * i] = f2_pack(a.x, b.x);
    o.v[2 * i + 1] = f2_pack(a.y, b.y);
  }
  return o;
}
__device__ __forceinline__ V8 unpack8(const Raw8<float>& r) {
  const float* w = reinterpret_cast<const float*>(&r.v[0]);
  const float x[8] = {w[0], w[1], w[2], w[3], w[4], w[5], w[6], w[7]};
  return planar(x);
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const V8& a) {
  float x[8];
  channels(a, x);
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]),
                                            pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7]));
}
__device__ __forceinline__ void store8(__half* p, const V8& a) {
  float x[8];
  channels(a, x);
  uint4 o;
  __half2* w = reinterpret_cast<__half2*>(&o);
#pragma unroll
  for (int i = 0; i < 4; ++i) w[i] = __floats2half2_rn(x[2 * i], x[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = o;
}
__device__ __forceinline__ void store8(float* p, const V8& a) {
  float x[8];
  channels(a, x);
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}

__device__ __forceinline__ V8 fill8(float x) {
  const uint64_t v = f2_pack(x, x);
  return V8{{v, v, v, v}};
}

__device__ __forceinline__ float sum2(uint64_t v) {
  float a, b;
  f2_unpack(v, a, b);
  return a + b;
}

// Channels c0..c0+7 of a weight vector of any of the three types (1 without).
__device__ __forceinline__ V8 load_weight8(const void* w, int dtype, int c0) {
  if (w == nullptr) return fill8(1.f);
  const uint4* p = reinterpret_cast<const uint4*>(w);
  if (dtype == SA_DTYPE_BF16) return unpack8(Raw8<__nv_bfloat16>{{p[c0 >> 3]}});
  if (dtype == SA_DTYPE_FP16) return unpack8(Raw8<__half>{{p[c0 >> 3]}});
  return unpack8(Raw8<float>{{p[c0 >> 2], p[(c0 >> 2) + 1]}});
}

// 1 / sqrt(v): the hardware's approximation (within 2^-22), with one Newton
// step where the result is fp32 as well.
template <typename T>
__device__ __forceinline__ float inv_sqrt(float v) {
  const float r = rsqrtf(v);
  if (sizeof(T) == 2) return r;
  const float e = fmaf(-v * r, r, 1.f);
  // v = 0 and v = inf keep the approximation's inf and 0 (e is NaN there)
  return e == e ? fmaf(0.5f * r, e, r) : r;
}

// out[c] = sum over `rows` partial rows of part[row * pitch + c], c < cols, in a
// fixed order (the same bits on every run); columns below cols0 go to out0,
// the rest to out1.
int sum_partial_rows(const float* part, int rows, int cols, int pitch, float* out0, float* out1,
                     int cols0, cudaStream_t stream);

}  // namespace nr
}  // namespace sa
