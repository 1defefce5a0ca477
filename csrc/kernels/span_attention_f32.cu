// Span attention in 32 bits, forward and backward (no TF32 rounding): softmax(cap tanh(scale q.k / cap) - slope |distance|) V over the keys lo <= j < hi of
// each row.  For models that train in 32 bits, whose heads are small: a row is a serial chain over its keys, on the FP32 pipes.  Tiles of 32 rows pass through
// shared memory; tiles that no row of the CTA reaches are left out.  The backward pass recomputes the weights from the log-sum-exp; its two
// halves, dQ by query rows and dK, dV by key rows (over all query heads that share the key head), run side by side in one grid, and nothing is added
// up in memory.  Bound by the FP32 pipes' issue, 9.3 TFLOP/s, or by the chain of a row.  Capped causal heads, us forward / forward and backward, in brackets
// the plain operators with all scores in memory: B 1, S 256, 4 heads of 32: 64 / 163 (105 / 428); B 4, S 1024, 8 of 64: 501 / 1826 (543 / 1310); B 2, S 2048,
// 8 of 128: 1814 / 6977 (1368 / 3399).  Calls go to those operators where they are ahead (f32_plain_is_ahead, ops/span.py); rows with spans, and more scores
// than they should keep, come here.  Larger models belong in 16 bits, where the tensor cores do it.
#include "attn_f32.cuh"
#include "span_scores.cuh"

namespace rb {

struct SpanF32Params {
  const float *q, *k, *v, *o, *dout;
  float *out, *lse, *dq, *dk, *dv;      // out, o, dq: [B, Sq, H, D]; dk, dv: [B, Sk, Hkv, D]; lse (natural): [B, H, Sq]
  long long qs[3], ks[3], vs[3], dos[3];     // {batch, row, head}
  int B, H, Hkv, Sq, Sk;
  float scale, cap;                     // cap 0: none
  SpanScores c;                         // slopes, spans, causal
};

// score of a product, and the factor that the cap puts on its gradient
__device__ __forceinline__ float span_f32_score(const SpanF32Params& p, float dot, float slope, int distance, float& slip) {
  float x = dot * p.scale;
  slip = 1.f;
  if (p.cap > 0.f) {
    const float t = tanhf(x / p.cap);
    slip = fmaf(-t, t, 1.f);
    x = p.cap * t;
  }
  return fmaf(-slope, (float)abs(distance), x);
}

// least lo and largest hi of the CTA's rows (empty ones aside)
__device__ __forceinline__ int2 span_f32_range(int2 s) {
  __shared__ int lo, hi;
  if (threadIdx.x == 0) { lo = 0x7fffffff; hi = 0; }
  __syncthreads();
  if (s.x < s.y) { atomicMin(&lo, s.x); atomicMax(&hi, s.y); }
  __syncthreads();
  return lo < hi ? make_int2(lo, hi) : make_int2(0, 0);
}

template <int D>
__global__ void __launch_bounds__(AF_THREADS) span_f32_fwd_kernel(const SpanF32Params p, int blocks) {
  using R = AttnF32Row<D>;
  __shared__ __align__(16) float sk[AF_TILE * D], sv[AF_TILE * D];
  const int sub = threadIdx.x % R::LANES, unit = blockIdx.x / blocks, h = unit % p.H, b = unit / p.H, hkv = h / (p.H / p.Hkv);
  const int row = (blocks - 1 - blockIdx.x % blocks) * R::ROWS + threadIdx.x / R::LANES, place = row + p.Sk - p.Sq;      // the longest first
  const float* k = p.k + b * p.ks[0] + hkv * p.ks[2];
  const float* v = p.v + b * p.vs[0] + hkv * p.vs[2];
  const float slope = p.c.slopes != nullptr ? p.c.slopes[h] : 0.f;
  float4 q[4], acc[4];
  af_zero(q);
  af_zero(acc);
  int2 span = make_int2(0, 0);
  if (row < p.Sq) {
    R::load(p.q + b * p.qs[0] + (long long)row * p.qs[1] + h * p.qs[2], sub, q);
    span = span_of(p.c, b, row, p.Sq, p.Sk);
  }
  const int2 all = span_f32_range(span);
  float m = -INFINITY, l = 0.f;
  for (int j0 = all.x; j0 < all.y; j0 += AF_TILE) {
    __syncthreads();
    af_tile<D>(sk, k, p.ks[1], j0, p.Sk);
    af_tile<D>(sv, v, p.vs[1], j0, p.Sk);
    __syncthreads();
    for (int j = 0; j < AF_TILE && j0 + j < all.y; j += 4) {
      float s[4], slip;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        float4 x[4];
        R::load(sk + (j + u) * D, sub, x);
        s[u] = R::dot(q, x);
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int key = j0 + j + u;
        s[u] = span_f32_score(p, R::all(s[u]), slope, place - key, slip);
        if (key < span.x || key >= span.y) s[u] = -INFINITY;
      }
      const float mn = fmaxf(m, fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3])));
      // no key of the group is seen by this row: all of them are -inf.  fmaxf passes over NaN, a sum does not.
      if (mn != -INFINITY || (s[0] + s[1]) + (s[2] + s[3]) != -INFINITY) {
        const float f = m == -INFINITY ? 0.f : expf(m - mn);
        l *= f;
#pragma unroll
        for (int c = 0; c < 4; ++c) { acc[c].x *= f; acc[c].y *= f; acc[c].z *= f; acc[c].w *= f; }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int key = j0 + j + u;
          if (key < span.x || key >= span.y) continue;
          const float w = expf(s[u] - mn);
          l += w;
          float4 x[4];
          R::load(sv + (j + u) * D, sub, x);
          af_axpy(w, x, acc);
        }
        m = mn;
      }
    }
  }
  if (row >= p.Sq) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
  for (int c = 0; c < 4; ++c) { acc[c].x *= inv; acc[c].y *= inv; acc[c].z *= inv; acc[c].w *= inv; }
  R::store(p.out + (((long long)b * p.Sq + row) * p.H + h) * D, sub, acc);
  if (sub == 0 && p.lse != nullptr) p.lse[((long long)b * p.H + h) * p.Sq + row] = l == 0.f ? -INFINITY : m + logf(l);
}

template <int D>
__global__ void __launch_bounds__(AF_THREADS) span_f32_bwd_kernel(const SpanF32Params p, int query_blocks, int query_units, int key_blocks) {
  using R = AttnF32Row<D>;
  __shared__ __align__(16) float sa[AF_TILE * D], sb[AF_TILE * D];
  __shared__ float s_lse[AF_TILE], s_delta[AF_TILE];
  __shared__ int2 s_span[AF_TILE];
  const int sub = threadIdx.x % R::LANES, off = p.Sk - p.Sq;
  const long long os = (long long)p.H * D;
  float4 x[4], y[4];
  if ((long long)blockIdx.x < (long long)query_blocks * query_units) {
    // ---- dQ of a block of queries ----
    const int unit = blockIdx.x / query_blocks, h = unit % p.H, b = unit / p.H, hkv = h / (p.H / p.Hkv);
    const int row = (query_blocks - 1 - blockIdx.x % query_blocks) * R::ROWS + threadIdx.x / R::LANES;
    const float* k = p.k + b * p.ks[0] + hkv * p.ks[2];
    const float* v = p.v + b * p.vs[0] + hkv * p.vs[2];
    const float slope = p.c.slopes != nullptr ? p.c.slopes[h] : 0.f;
    const bool live = row < p.Sq;
    float4 qr[4], g[4], acc[4];
    af_zero(qr);
    af_zero(g);
    af_zero(acc);
    float delta = 0.f, ls = 0.f;
    int2 span = make_int2(0, 0);
    if (live) {
      R::load(p.q + b * p.qs[0] + (long long)row * p.qs[1] + h * p.qs[2], sub, qr);
      R::load(p.dout + b * p.dos[0] + (long long)row * p.dos[1] + h * p.dos[2], sub, g);
      R::load(p.o + ((long long)b * p.Sq * p.H + h) * D + row * os, sub, x);
      delta = R::dot(g, x);
      ls = p.lse[((long long)b * p.H + h) * p.Sq + row];
      span = span_of(p.c, b, row, p.Sq, p.Sk);
    }
    delta = R::all(delta);
    const int2 all = span_f32_range(span);
    for (int j0 = all.x; j0 < all.y; j0 += AF_TILE) {
      __syncthreads();
      af_tile<D>(sa, k, p.ks[1], j0, p.Sk);
      af_tile<D>(sb, v, p.vs[1], j0, p.Sk);
      __syncthreads();
#pragma unroll 2
      for (int j = 0; j < AF_TILE; ++j) {
        const int key = j0 + j;
        if (key >= all.y) break;
        R::load(sa + j * D, sub, x);
        R::load(sb + j * D, sub, y);
        const float s = R::all(R::dot(qr, x)), dp = R::all(R::dot(g, y));
        float slip;
        const float z = span_f32_score(p, s, slope, row + off - key, slip);
        if (key >= span.x && key < span.y) af_axpy(expf(z - ls) * (dp - delta) * slip * p.scale, x, acc);
      }
    }
    if (live) R::store(p.dq + ((long long)b * p.Sq * p.H + h) * D + row * os, sub, acc);
    return;
  }
  // ---- dK and dV of a block of keys ----
  const int at = (int)(blockIdx.x - (long long)query_blocks * query_units), unit = at / key_blocks, hkv = unit % p.Hkv, b = unit / p.Hkv, group = p.H / p.Hkv;
  const int row0 = at % key_blocks * R::ROWS, row = row0 + threadIdx.x / R::LANES;      // early keys, which most rows see, first
  const bool live = row < p.Sk;
  float4 kr[4], vr[4], dk[4], dv[4];
  af_zero(kr);
  af_zero(vr);
  af_zero(dk);
  af_zero(dv);
  if (live) {
    R::load(p.k + b * p.ks[0] + (long long)row * p.ks[1] + hkv * p.ks[2], sub, kr);
    R::load(p.v + b * p.vs[0] + (long long)row * p.vs[1] + hkv * p.vs[2], sub, vr);
  }
  for (int i0 = 0; i0 < p.Sq; i0 += AF_TILE) {
    __syncthreads();                              // the last tile's rows have been read
    bool reaches = false;
    if (threadIdx.x < AF_TILE) {
      const int i = i0 + threadIdx.x;
      const int2 s = i < p.Sq ? span_of(p.c, b, i, p.Sq, p.Sk) : make_int2(0, 0);
      s_span[threadIdx.x] = s;
      reaches = s.x < s.y && s.x < row0 + R::ROWS && s.y > row0;
    }
    if (!__syncthreads_or(reaches)) continue;
    for (int h = hkv * group; h < (hkv + 1) * group; ++h) {
      const float slope = p.c.slopes != nullptr ? p.c.slopes[h] : 0.f;
      const float* dout = p.dout + b * p.dos[0] + h * p.dos[2];
      const float* o = p.o + ((long long)b * p.Sq * p.H + h) * D;
      __syncthreads();
      af_tile<D>(sa, p.q + b * p.qs[0] + h * p.qs[2], p.qs[1], i0, p.Sq);
      // dO, and sum dO O of its rows: D / 4 lanes a row
      for (int i = threadIdx.x; i < AF_TILE * D / 4; i += AF_THREADS) {
        const int r = i / (D / 4), c = i % (D / 4);
        float4 g = make_float4(0.f, 0.f, 0.f, 0.f);
        float part = 0.f;
        if (i0 + r < p.Sq) {
          g = *reinterpret_cast<const float4*>(dout + (long long)(i0 + r) * p.dos[1] + c * 4);
          const float4 u = *reinterpret_cast<const float4*>(o + (i0 + r) * os + c * 4);
          part = fmaf(g.x, u.x, fmaf(g.y, u.y, fmaf(g.z, u.z, g.w * u.w)));
        }
        *reinterpret_cast<float4*>(sb + r * D + c * 4) = g;
#pragma unroll
        for (int w = 1; w < D / 4; w <<= 1) part += __shfl_xor_sync(0xffffffffu, part, w);
        if (c == 0) {
          s_delta[r] = part;
          s_lse[r] = i0 + r < p.Sq ? p.lse[((long long)b * p.H + h) * p.Sq + i0 + r] : 0.f;
        }
      }
      __syncthreads();
#pragma unroll 2
      for (int i = 0; i < AF_TILE; ++i) {
        if (i0 + i >= p.Sq) break;
        R::load(sa + i * D, sub, x);
        R::load(sb + i * D, sub, y);
        const float s = R::all(R::dot(kr, x)), dp = R::all(R::dot(vr, y));
        float slip;
        const float z = span_f32_score(p, s, slope, i0 + i + off - row, slip);
        if (live && row >= s_span[i].x && row < s_span[i].y) {
          const float w = expf(z - s_lse[i]);
          af_axpy(w, y, dv);
          af_axpy(w * (dp - s_delta[i]) * slip * p.scale, x, dk);
        }
      }
    }
  }
  if (live) {
    const long long to = (((long long)b * p.Sk + row) * p.Hkv + hkv) * D;
    R::store(p.dk + to, sub, dk);
    R::store(p.dv + to, sub, dv);
  }
}

}  // namespace rb

extern "C" {

// fp32; head sizes 16, 32, 64, 128; q [B, Sq, H, D], k and v [B, Sk, Hkv, D]: rows of D numbers, 16-byte aligned, strides {batch, row, head}; spans, slopes and
// cap as in rb_span_fwd.  out [B, Sq, H, D] contiguous, lse [B, H, Sq] (natural) or null.  20: not covered.
int rb_span_f32_fwd(int D, const float* q, const float* k, const float* v, const long long* qs, const long long* ks, const long long* vs, const int* spans,
                    long long span_batch, const float* slopes, float* out, float* lse, int B, int H, int Hkv, int Sq, int Sk, int causal, float scale,
                    float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0 || Sq <= 0) return 0;
  if (Sk <= 0 || Hkv <= 0 || H % Hkv || (D != 16 && D != 32 && D != 64 && D != 128)) return 20;
  SpanF32Params p{};
  p.q = q; p.k = k; p.v = v; p.out = out; p.lse = lse;
  for (int i = 0; i < 3; ++i) { p.qs[i] = qs[i]; p.ks[i] = ks[i]; p.vs[i] = vs[i]; }
  p.B = B; p.H = H; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.scale = scale; p.cap = cap;
  p.c.slopes = slopes; p.c.spans = reinterpret_cast<const int2*>(spans); p.c.span_batch = span_batch; p.c.causal = causal;
  cudaStream_t st = (cudaStream_t)stream;
#define RB_AF(D_)                                                                                            \
  if (D == D_) {                                                                                             \
    const long long blocks = (Sq + AttnF32Row<D_>::ROWS - 1) / AttnF32Row<D_>::ROWS, grid = blocks * B * H;  \
    if (grid > 0x7fffffffll) return 20;                                                                      \
    span_f32_fwd_kernel<D_><<<(unsigned)grid, AF_THREADS, 0, st>>>(p, (int)blocks);                          \
    cudaError_t e = cudaGetLastError();                                                                      \
    return e == cudaSuccess ? 0 : 3000 + (int)e;                                                             \
  }
  RB_AF(16) RB_AF(32) RB_AF(64) RB_AF(128)
#undef RB_AF
  return 20;
}

// Gradients of rb_span_f32_fwd: o and lse from it; dq [B, Sq, H, D], dk and dv [B, Sk, Hkv, D] contiguous.
int rb_span_f32_bwd(int D, const float* q, const float* k, const float* v, const long long* qs, const long long* ks, const long long* vs, const int* spans,
                    long long span_batch, const float* slopes, const float* o, float* lse, const float* dout, const long long* dos, float* dq, float* dk,
                    float* dv, int B, int H, int Hkv, int Sq, int Sk, int causal, float scale, float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0 || Sq <= 0) return 0;
  if (Sk <= 0 || Hkv <= 0 || H % Hkv || (D != 16 && D != 32 && D != 64 && D != 128)) return 20;
  SpanF32Params p{};
  p.q = q; p.k = k; p.v = v; p.o = o; p.lse = lse; p.dout = dout; p.dq = dq; p.dk = dk; p.dv = dv;
  for (int i = 0; i < 3; ++i) { p.qs[i] = qs[i]; p.ks[i] = ks[i]; p.vs[i] = vs[i]; p.dos[i] = dos[i]; }
  p.B = B; p.H = H; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.scale = scale; p.cap = cap;
  p.c.slopes = slopes; p.c.spans = reinterpret_cast<const int2*>(spans); p.c.span_batch = span_batch; p.c.causal = causal;
  cudaStream_t st = (cudaStream_t)stream;
#define RB_AF(D_)                                                                                            \
  if (D == D_) {                                                                                             \
    constexpr int R = AttnF32Row<D_>::ROWS;                                                                  \
    const long long nq = (Sq + R - 1) / R, nk = (Sk + R - 1) / R, grid = nq * B * H + nk * B * Hkv;          \
    if (grid > 0x7fffffffll) return 20;                                                                      \
    span_f32_bwd_kernel<D_><<<(unsigned)grid, AF_THREADS, 0, st>>>(p, (int)nq, B * H, (int)nk);              \
    cudaError_t e = cudaGetLastError();                                                                      \
    return e == cudaSuccess ? 0 : 3000 + (int)e;                                                             \
  }
  RB_AF(16) RB_AF(32) RB_AF(64) RB_AF(128)
#undef RB_AF
  return 20;
}
}
