// Joins the results of span attention whose keys were cut into parts.
#pragma once
#include "sm100_common.cuh"

namespace rb {

// Joins the parts of rows: out = sum 2^(lse_s - lse) o_s.  Eight numbers a thread.
template <typename T>
__global__ void __launch_bounds__(256)
    span_join_kernel(const float* __restrict__ part_o, const float* __restrict__ part_lse2, T* __restrict__ o, float* __restrict__ lse2, int B, int H,
                     int Sq, int D, int splits) {
  const int pieces = D / 8;
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x, rows = static_cast<long long>(B) * Sq * H;
  if (i >= rows * pieces) return;
  const long long r = i / pieces;
  const int c = static_cast<int>(i - r * pieces) * 8;
  const int h = static_cast<int>(r % H);
  const long long bq = r / H, b = bq / Sq, at = (b * H + h) * Sq + bq % Sq;
  float top = -INFINITY;
  for (int s = 0; s < splits; ++s) top = fmaxf(top, part_lse2[s * rows + at]);
  float sum = 0.f, f[8] = {};
  for (int s = 0; s < splits; ++s) {
    const float e = part_lse2[s * rows + at];
    if (e == -INFINITY) continue;                      // no key in this part
    const float w = fast_exp2(e - top);
    const float4* from = reinterpret_cast<const float4*>(part_o + (s * rows + r) * D + c);
    const float4 x = from[0], y = from[1];
    sum += w;
    f[0] = fmaf(w, x.x, f[0]); f[1] = fmaf(w, x.y, f[1]); f[2] = fmaf(w, x.z, f[2]); f[3] = fmaf(w, x.w, f[3]);
    f[4] = fmaf(w, y.x, f[4]); f[5] = fmaf(w, y.y, f[5]); f[6] = fmaf(w, y.z, f[6]); f[7] = fmaf(w, y.w, f[7]);
  }
  const float inv = sum == 0.f ? 0.f : 1.0f / sum;
  // two stores of 8 bytes: decoding's results may begin at any such boundary
  uint2* to = reinterpret_cast<uint2*>(o + r * D + c);
  to[0] = make_uint2(pack2<T>(f[0] * inv, f[1] * inv), pack2<T>(f[2] * inv, f[3] * inv));
  to[1] = make_uint2(pack2<T>(f[4] * inv, f[5] * inv), pack2<T>(f[6] * inv, f[7] * inv));
  if (c == 0 && lse2 != nullptr) lse2[at] = sum == 0.f ? -INFINITY : top + log2f(sum);
}

// part_o [splits, B, Sq, H, D], 16-byte aligned, part_lse2 [splits, B, H, Sq] -> o [B, Sq, H, D], 8-byte aligned, lse2 [B, H, Sq] (or null)
template <typename T>
int launch_span_join(const float* part_o, const float* part_lse2, T* o, float* lse2, int B, int H, int Sq, int D, int splits, cudaStream_t st) {
  const long long pieces = static_cast<long long>(B) * Sq * H * (D / 8), blocks = (pieces + 255) / 256;
  if (blocks > 0x7fffffffll) return 20;
  span_join_kernel<T><<<(unsigned)blocks, 256, 0, st>>>(part_o, part_lse2, o, lse2, B, H, Sq, D, splits);
  const cudaError_t e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 3000 + (int)e;
}

}  // namespace rb
