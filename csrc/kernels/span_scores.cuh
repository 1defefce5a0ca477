// Scores of span attention: x = cap tanh(scale q.k / cap) - slope |distance| in units of log2 e, visible for keys lo <= j < hi.
// What the forward and the backward kernels share: the same arithmetic in the same order, so that the backward pass finds the weights of the forward one.
#pragma once
#include "sm100_common.cuh"

namespace rb {

constexpr float kLog2e = 1.4426950408889634f;

struct SpanScores {
  float scale2;        // scale log2 e
  float in, out2;      // scale / cap, cap log2 e (cap)
  float near;          // products up to this size are near enough to zero for the tanh's polynomial (below zero: none is)
  float far2;          // see span_reach; without a cap 0
  const float* norms;  // without a cap: [B, H + Hkv, 32] largest squared lengths of 32 parts of a head's queries, then of the key heads' keys; null: not known
  float k[4];          // its coefficients in the square of a product: tanh(in s) = s (k0 + k1 s^2 + k2 s^4 + k3 s^6)
  const float* slopes; // [H] or null
  const int2* spans;   // [B, Sq] {lo, hi} or null
  long long span_batch;// rows from one batch's spans to the next's (0: all batches share them)
  int causal;
};


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

// With a bias: how many places farther than a row's nearest key a key can be and still have a weight.  Where no score but for the bias is above m in size (the
// cap, or |scale| times the largest query's and key's lengths) the nearest key has -m - slope d or more, one that is r places farther m - slope (d + r) at
// most: from slope r = 2 m + 150 log 2 on its weight is below 2^-150 of the nearest's, which is zero in 32 bits.  Tiles that lie wholly there are left out.
constexpr int kSpanNoReach = 0x7fffffff;
__device__ __forceinline__ int span_reach(float far2, float slope) {          // far2: 2 m log2 e + 150
  const float r = far2 / (slope * kLog2e);
  return slope > 0.f && r < 2e9f ? static_cast<int>(r) + 2 : kSpanNoReach;
}
// Of a head; whole warps.  The bits of lengths, which are not negative, are in the lengths' order, with what is no number above all.
template <bool CAP>
__device__ __forceinline__ int span_head_reach(const SpanScores& c, int b, int h, int hkv, int H, int Hkv) {
  if (CAP) return span_reach(c.far2, c.slopes[h]);
  if (c.norms == nullptr) return kSpanNoReach;
  const float* of = c.norms + static_cast<long long>(b) * (H + Hkv) * 32 + (threadIdx.x & 31);
  const uint32_t q2 = __reduce_max_sync(0xffffffffu, __float_as_uint(of[h * 32])), k2 = __reduce_max_sync(0xffffffffu, __float_as_uint(of[(H + hkv) * 32]));
  return span_reach(2.002f * fabsf(c.scale2) * sqrtf(__uint_as_float(q2)) * sqrtf(__uint_as_float(k2)) + 150.f, c.slopes[h]);
}
// The part of a row's span that lies within `reach` of the key nearest to the row's place
__device__ __forceinline__ int2 span_near(int2 s, int place, int reach) {
  if (s.x >= s.y) return s;
  const long long w = static_cast<long long>(max(0, max(s.x - place, place - (s.y - 1)))) + reach;
  return make_int2(static_cast<int>(max(static_cast<long long>(s.x), place - w)), static_cast<int>(min(static_cast<long long>(s.y), place + w + 1)));
}

__device__ __forceinline__ uint64_t pair_at(const uint32_t* s, int i) { return f32x2(__uint_as_float(s[i]), __uint_as_float(s[i + 1])); }
__device__ __forceinline__ void set_pair(uint32_t* s, int i, uint64_t v) {
  const float2 f = f32x2_get(v);
  s[i] = __float_as_uint(f.x);
  s[i + 1] = __float_as_uint(f.y);
}
__device__ __forceinline__ uint64_t both(float a) { return f32x2(a, a); }

// What is added to the i-th of 32 neighbouring scores of a row (or of a key): base + step i, a bias that is linear along the tile and the number that
// the weights are relative to.  Sixteen additions of pairs from an exact beginning: what they round is below 2^-20 of the largest bias of the 32.
struct SpanRamp {
  float base, step;
};
// The same from pairs in shared memory (ADD: numbers to add, beside the ramp).
template <bool RAMP, bool ADD>
struct SpanAdd {
  uint64_t at, by;
  const float4* add;
  __device__ __forceinline__ SpanAdd(SpanRamp r, const float4* add_) : add(add_) {
    at = f32x2(r.base, RAMP ? r.base + r.step : r.base);
    by = both(2.f * r.step);
  }
  // of places i, i + 1: called for i = 0, 2, 4, ...
  __device__ __forceinline__ uint64_t next(int i) {
    uint64_t v = at;
    if (RAMP) at = add_f32x2(at, by);
    if (ADD) {
      const float4 f = add[i >> 2];
      const uint64_t w = i & 2 ? f32x2(f.z, f.w) : f32x2(f.x, f.y);
      v = RAMP ? add_f32x2(v, w) : w;
    }
    return v;
  }
};

// The polynomial: tanh(in s) out = s r(s).  Two values at a time on the FMA pipe, where the exponential and the reciprocal of the general form would take
// the special-function pipe, which the softmax already fills.
struct SpanTanh {
  uint64_t k0, k1, k2, k3;
  __device__ __forceinline__ SpanTanh(const SpanScores& c, float out) : k0(both(c.k[0] * out)), k1(both(c.k[1] * out)), k2(both(c.k[2] * out)), k3(both(c.k[3] * out)) {}
  __device__ __forceinline__ uint64_t r(uint64_t s) const {
    const uint64_t w = mul_f32x2(s, s);
    return fma_f32x2(fma_f32x2(fma_f32x2(k3, w, k2), w, k1), w, k0);
  }
};
// The general form, 1 - 2 / (1 + e^2u): absolute error of 2e-7 to 3e-7
__device__ __forceinline__ uint64_t span_tanh_any(uint32_t a, uint32_t b, const SpanScores& c) {
  const float e = 2.f * kLog2e * c.in;
  return f32x2(1.f - __fdividef(2.f, 1.f + fast_exp2(__uint_as_float(a) * e)), 1.f - __fdividef(2.f, 1.f + fast_exp2(__uint_as_float(b) * e)));
}

__device__ __forceinline__ float span_reach32(const uint32_t* s) {
  float mx[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 32; ++i) mx[i & 3] = fmaxf(mx[i & 3], fabsf(__uint_as_float(s[i])));
  return fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
}

// 32 products -> scores in log2 units plus what `add` gives, in place; SLIP: minus the cap's derivative, tanh^2 - 1, beside them.  `reach`: no product
// is larger (with a cap).  Whole warp: a vote decides between the two forms of the tanh.
template <bool CAP, bool SLIP, class Add>
__device__ __forceinline__ void span_score32(uint32_t* s, const SpanScores& c, Add add, uint32_t* slip, float reach) {
  if constexpr (!CAP) {
    const uint64_t k = both(c.scale2);
#pragma unroll
    for (int i = 0; i < 32; i += 2) set_pair(s, i, fma_f32x2(pair_at(s, i), k, add.next(i)));
  } else {
    if (__all_sync(0xffffffffu, reach <= c.near)) {
      const SpanTanh f(c, SLIP ? 1.f : c.out2);
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const uint64_t x = pair_at(s, i), r = f.r(x);
        if constexpr (SLIP) {
          const uint64_t t = mul_f32x2(x, r);
          set_pair(slip, i, fma_f32x2(t, t, both(-1.f)));
          set_pair(s, i, fma_f32x2(t, both(c.out2), add.next(i)));
        } else {
          set_pair(s, i, fma_f32x2(x, r, add.next(i)));
        }
      }
    } else {
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const uint64_t t = span_tanh_any(s[i], s[i + 1], c);
        if constexpr (SLIP) set_pair(slip, i, fma_f32x2(t, t, both(-1.f)));
        set_pair(s, i, fma_f32x2(t, both(c.out2), add.next(i)));
      }
    }
  }
}

// s_i -= slope2 |first + step i|, for tiles with keys on both sides of their rows' places
template <int STEP>
__device__ __forceinline__ void span_both_sides32(uint32_t* s, float slope2, float first) {
#pragma unroll
  for (int i = 0; i < 32; ++i) s[i] = __float_as_uint(fmaf(-slope2, fabsf(first + (float)(STEP * i)), __uint_as_float(s[i])));
}

// places of 32 that `seen` does not name get `other`
__device__ __forceinline__ void span_mask32(uint32_t* s, uint32_t seen, uint32_t other) {
#pragma unroll
  for (int i = 0; i < 32; ++i)
    if (!(seen >> i & 1)) s[i] = other;
}
// bit i set: place i of 32 lies in [lo, hi)
__device__ __forceinline__ uint32_t span_bits(int lo, int hi) {
  const int a = min(max(lo, 0), 32), b = min(max(hi, 0), 32);
  const uint32_t below_b = b >= 32 ? 0xffffffffu : (1u << b) - 1, below_a = a >= 32 ? 0xffffffffu : (1u << a) - 1;
  return below_b & ~below_a;
}

// Order of a launch's CTAs: heads in groups whose keys stay in the L2 cache together, in a group the tiles from the last to the first (FROM_END; causal: the
// longest first, so that the short ones fill the gaps at the end) or the other way, in a tile the group's heads.
struct SpanOrder {
  int tiles, units, group;
};
template <bool FROM_END>
__device__ __forceinline__ void span_place(const SpanOrder& o, int idx, int& tile, int& unit) {
  const int per = o.group * o.tiles, g = idx / per, in = idx - g * per, n = min(o.group, o.units - g * o.group);
  const int t = in / n;
  tile = FROM_END ? o.tiles - 1 - t : t;
  unit = g * o.group + in - t * n;
}

// Range of keys that rows of a tile reach, over the `live` lanes of a warp: {least lo, largest hi of what is `near`, largest lo, least hi of the spans}; a
// row without keys keeps the tile from being whole.
__device__ __forceinline__ int4 span_range_warp(int2 s, int2 near, bool live) {
  const bool sees = live && near.x < near.y;
  int4 r;
  r.x = __reduce_min_sync(0xffffffffu, sees ? near.x : 0x7fffffff);
  r.y = __reduce_max_sync(0xffffffffu, sees ? near.y : 0);
  r.z = __reduce_max_sync(0xffffffffu, live ? s.x : 0);
  r.w = __reduce_min_sync(0xffffffffu, live ? s.y : 0x7fffffff);
  return r;
}
__device__ __forceinline__ int4 span_range_join(int4 a, int4 b) {
  return make_int4(min(a.x, b.x), max(a.y, b.y), max(a.z, b.z), min(a.w, b.w));
}

}  // namespace rb

namespace rbh {

// What a call's scale and cap are to the kernels.  tanh(u) = u P(u^2) for |u| <= 0.625, P of degree 3 fitted so that the largest relative error is least:
// 3.1e-6.  At scores of 30 a weight is then off by 9.3e-5 of itself: a forty-second of bf16's rounding (half a step, 2^-8), a fifth of fp16's.  Of caps
// far above the scale the highest coefficients in the products are below fp32's range: they are left out, and the polynomial holds as far as they make no
// more difference than that.  (The general form, whose error is absolute, is no choice there: 3e-7 of a cap of 1e6 is 0.3.)  Of caps far below the scale
// they are above it, and the general form serves.
inline rb::SpanScores span_scores(float scale, float cap) {
  rb::SpanScores c{};
  c.scale2 = scale * rb::kLog2e;
  if (!(cap > 0.f)) return c;
  c.in = scale / cap;
  c.out2 = cap * rb::kLog2e;
  c.far2 = 2.f * c.out2 + 150.f;
  const float a = c.in < 0.f ? -c.in : c.in, w = c.in * c.in;
  const int terms = a > 0x1p-17f ? 4 : a > 0x1p-24f ? 3 : a > 0x1p-41f ? 2 : 1;
  c.near = (terms == 4 ? 0.625f : terms == 3 ? 0.2f : terms == 2 ? 0.07f : 0.003f) / a;
  if (!(c.near < 1e18f)) c.near = 1e18f;
  if (a > 0x1p17f) c.near = -1.f;
  c.k[0] = 0.999997256f * c.in;
  c.k[1] = terms > 1 ? -0.333099914f * c.in * w : 0.f;
  c.k[2] = terms > 2 ? 0.130206247f * c.in * w * w : 0.f;
  c.k[3] = terms > 3 ? -0.040117459f * c.in * w * w * w : 0.f;
  return c;
}

// Heads whose streamed rows (`bytes` each) take a quarter of the L2 cache, in groups of one size: with 63 heads and one more, whose longest tiles came last
// of all, the SMs were idle for a sixth of a launch.
inline int span_group(long long units, long long bytes) {
  long long fit = (32ll << 20) / (bytes > 0 ? bytes : 1);
  if (fit < 1) fit = 1;
  const long long groups = (units + fit - 1) / fit;
  return (int)(groups < 1 ? 1 : (units + groups - 1) / groups);
}

// Tensor map of heads [B, S, heads, D] with strides {batch, row, head} in elements, read in boxes of `rows` rows of 64 numbers of a head; what lies
// beyond D reads as zero.
inline int span_map(CUtensorMap* m, int dtype, const void* base, const long long* s, int B, int S, int heads, int D, int rows) {
  uint64_t dims[4] = {(uint64_t)D, (uint64_t)S, (uint64_t)heads, (uint64_t)B};
  uint64_t strides[4] = {2, (uint64_t)s[1] * 2, (uint64_t)s[2] * 2, (uint64_t)s[0] * 2};
  uint32_t box[4] = {64, (uint32_t)rows, 1, 1};
  return encode_tensor_map(m, dtype, 4, const_cast<void*>(base), dims, strides, box, 1);
}

}  // namespace rbh
