// What the 32-bit attention kernels share: a row (of queries or keys) belongs to D / 16 neighbouring lanes with sixteen of its numbers each, in pieces of four
// that alternate between the lanes, so that the lanes read one row of a tile in shared memory without bank conflicts and the rows of a warp share the read.
#pragma once
#include "sm100_common.cuh"

namespace rb {

constexpr int AF_THREADS = 128, AF_TILE = 32;

template <int D>
struct AttnF32Row {
  static constexpr int LANES = D / 16, ROWS = AF_THREADS / LANES;
  static __device__ __forceinline__ void load(const float* p, int sub, float4 (&r)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) r[c] = *reinterpret_cast<const float4*>(p + (c * LANES + sub) * 4);
  }
  static __device__ __forceinline__ void store(float* p, int sub, const float4 (&r)[4]) {
#pragma unroll
    for (int c = 0; c < 4; ++c) *reinterpret_cast<float4*>(p + (c * LANES + sub) * 4) = r[c];
  }
  static __device__ __forceinline__ float dot(const float4 (&a)[4], const float4 (&b)[4]) {
    float s = 0.f;
#pragma unroll
    for (int c = 0; c < 4; ++c) s = fmaf(a[c].x, b[c].x, fmaf(a[c].y, b[c].y, fmaf(a[c].z, b[c].z, fmaf(a[c].w, b[c].w, s))));
    return s;
  }
  static __device__ __forceinline__ float all(float s) {
#pragma unroll
    for (int o = 1; o < LANES; o <<= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    return s;
  }
};
__device__ __forceinline__ void af_axpy(float a, const float4 (&x)[4], float4 (&y)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    y[c].x = fmaf(a, x[c].x, y[c].x);
    y[c].y = fmaf(a, x[c].y, y[c].y);
    y[c].z = fmaf(a, x[c].z, y[c].z);
    y[c].w = fmaf(a, x[c].w, y[c].w);
  }
}
__device__ __forceinline__ void af_zero(float4 (&y)[4]) {
#pragma unroll
  for (int c = 0; c < 4; ++c) y[c] = make_float4(0.f, 0.f, 0.f, 0.f);
}
// rows [r0, r0 + AF_TILE) of a strided [rows, D] matrix into shared memory, zeros beyond n
template <int D>
__device__ __forceinline__ void af_tile(float* dst, const float* src, long long stride, int r0, int n) {
  for (int i = threadIdx.x; i < AF_TILE * D / 4; i += AF_THREADS) {
    const int r = i / (D / 4), c = i % (D / 4);
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    if (r0 + r < n) v = *reinterpret_cast<const float4*>(src + (long long)(r0 + r) * stride + c * 4);
    *reinterpret_cast<float4*>(dst + r * D + c * 4) = v;
  }
}

}  // namespace rb
