// Scores of span attention: x = cap tanh(scale q.k / cap) - slope |distance| in units of log2 e, visible for keys lo <= j < hi.
// What the forward and the backward kernels share: the same arithmetic in the same order, so that the backward pass finds the weights of the forward one.
#pragma once
#include "sm100_common.cuh"

namespace rb {

struct SpanScores {
  float scale2;        // scale log2 e (no cap)
  float in, out2;      // scale / cap, cap log2 e (cap)
  const float* slopes; // [H] or null
  const int2* spans;   // [B, Sq] {lo, hi} or null
  long long span_batch;// rows from one batch's spans to the next's (0: all batches share them)
  int causal;
};

constexpr float kLog2e = 1.4426950408889634f;

// The span of query row `row` cut to what there is: keys [x, y), {0, 0} where the row sees none.
__device__ __forceinline__ int2 span_of(const SpanScores& c, int b, int row, int Sq, int Sk) {
  int2 s = make_int2(0, Sk);
  if (c.spans != nullptr) {
    s = c.spans[b * c.span_batch + row];
    s.x = max(s.x, 0);
    s.y = min(s.y, Sk);
  }
  if (c.causal) s.y = min(s.y, row + Sk - Sq + 1);
  return s.x < s.y ? s : make_int2(0, 0);
}

// tanh(u) = u P(u^2) for |u| <= 0.75, P of degree 4 fitted so that the largest error of tanh is least: 1.9e-7, what rounding to fp32 costs
// beside it.  Two values at a time on the FMA pipe, where the exponential and the reciprocal of the general form would take the
// special-function pipe, which the softmax already fills.
constexpr float kTanhReach = 0.75f;

// N products -> cap tanh(in s) log2 e in place.  Whole warp: one vote decides between the two forms.
template <int N>
__device__ __forceinline__ void span_cap(uint32_t* s, const SpanScores& c) {
  float mx = 0.f;
#pragma unroll
  for (int i = 0; i < N; ++i) mx = fmaxf(mx, fabsf(__uint_as_float(s[i])));
  if (__all_sync(0xffffffffu, mx * fabsf(c.in) <= kTanhReach)) {
    const uint64_t in = f32x2(c.in, c.in);
    const float fit[5] = {0.999997228f, -0.333230765f, 0.132260914f, -0.0492804431f, 0.0123188287f};
    uint64_t k[5];
#pragma unroll
    for (int j = 0; j < 5; ++j) k[j] = f32x2(fit[j] * c.out2, fit[j] * c.out2);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t u = mul_f32x2(f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), in), w = mul_f32x2(u, u);
      uint64_t r = fma_f32x2(k[4], w, k[3]);
      r = fma_f32x2(r, w, k[2]);
      r = fma_f32x2(r, w, k[1]);
      r = fma_f32x2(r, w, k[0]);
      const float2 x = f32x2_get(mul_f32x2(u, r));
      s[i] = __float_as_uint(x.x);
      s[i + 1] = __float_as_uint(x.y);
    }
  } else {
    const float e = 2.f * kLog2e * c.in;       // tanh u = 1 - 2 / (1 + e^2u)
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __float_as_uint(c.out2 - __fdividef(2.f * c.out2, 1.f + fast_exp2(__uint_as_float(s[i]) * e)));
  }
}

// N scores in log2 units (not shifted by distance) from products
template <bool CAP, int N>
__device__ __forceinline__ void span_scale(uint32_t* s, const SpanScores& c) {
  if constexpr (CAP) {
    span_cap<N>(s, c);
  } else {
    const uint64_t k = f32x2(c.scale2, c.scale2);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const float2 x = f32x2_get(mul_f32x2(f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])), k));
      s[i] = __float_as_uint(x.x);
      s[i + 1] = __float_as_uint(x.y);
    }
  }
}

// x_i -= slope2 |first + i|: distances that grow by one along the tile (STEP 1) or fall by one (STEP -1).  Whole numbers up to 2^24 are exact in
// fp32, so the only rounding is the sum's.  `side`: 1 all distances >= 0, -1 all <= 0, 0 both (warp-uniform).
template <int STEP, int N>
__device__ __forceinline__ void span_bias(uint32_t* s, float slope2, float first, int side) {
  if (side != 0) {
    const float k = side > 0 ? -slope2 : slope2;
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __float_as_uint(fmaf(k, first + (float)(STEP * i), __uint_as_float(s[i])));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) s[i] = __float_as_uint(fmaf(-slope2, fabsf(first + (float)(STEP * i)), __uint_as_float(s[i])));
  }
}

// bit i set: place i of 32 lies in [lo, hi)
__device__ __forceinline__ uint32_t span_bits(int lo, int hi) {
  const int a = min(max(lo, 0), 32), b = min(max(hi, 0), 32);
  const uint32_t below_b = b >= 32 ? 0xffffffffu : (1u << b) - 1, below_a = a >= 32 ? 0xffffffffu : (1u << a) - 1;
  return below_b & ~below_a;
}

// Range of keys that rows of a tile reach, over the `live` lanes of a warp: {least lo, largest hi, largest lo, least hi}; a row without keys keeps
// the tile from being whole.
__device__ __forceinline__ int4 span_range_warp(int2 s, bool live) {
  const bool sees = live && s.x < s.y;
  int4 r;
  r.x = __reduce_min_sync(0xffffffffu, sees ? s.x : 0x7fffffff);
  r.y = __reduce_max_sync(0xffffffffu, sees ? s.y : 0);
  r.z = __reduce_max_sync(0xffffffffu, live ? s.x : 0);
  r.w = __reduce_min_sync(0xffffffffu, live ? s.y : 0x7fffffff);
  return r;
}
__device__ __forceinline__ int4 span_range_join(int4 a, int4 b) {
  return make_int4(min(a.x, b.x), max(a.y, b.y), max(a.z, b.z), min(a.w, b.w));
}

}  // namespace rb

namespace rbh {

// Tensor map of heads [B, S, heads, D] with strides {batch, row, head} in elements, read in boxes of `rows` rows of 64 numbers of a head; what lies
// beyond D reads as zero.
inline int span_map(CUtensorMap* m, int dtype, const void* base, const long long* s, int B, int S, int heads, int D, int rows) {
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)heads, (uint64_t)B};
  uint64_t strides[4] = {2, (uint64_t)s[1] * 2, (uint64_t)s[2] * 2, (uint64_t)s[0] * 2};
  uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return encode_tensor_map(m, dtype, 4, const_cast<void*>(base), dims, strides, box, 1);
}

}  // namespace rbh
