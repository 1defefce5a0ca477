// Span attention of one new token per sequence over a paged cache, sm_100a, 16-bit, heads of 8 to 128 numbers: softmax(cap tanh(scale q.k / cap) -
// slope distance) V over the keys start <= t < ctx of each sequence; token t of sequence b lies in page tables[b][t / page size].
//
// Bound by the bytes of the visible keys and values, which cross HBM once: the query heads that share a key head attend together.  That is at most 16
// rows for the tensor core, so the products are warp-level ones of 16 heads x 8 keys (or numbers), whose fragments stay in registers from scores to
// values.  A warp takes every fourth group of 16 keys of its CTA's part: it asks for the next groups (asynchronous copies of 16 bytes into a ring that only this
// warp reads, so no barriers) while it computes one, with a maximum, a sum and an accumulator of its own.  What is not there (behind the context, before the
// start, a page that the pool does not have) is not read; its place holds zeros and its weight is zero.
//
// Long contexts of few sequences are cut into parts, one CTA each.  Up to eight parts form a cluster and are joined through distributed shared memory in the
// same launch; more parts go through memory and a second kernel.
//
// Heads of 128: 48 sequences of up to 1250 tokens, 32 heads, biased: 114 us, 6.7 TB/s; 8 x 32768 visible of 60000, 32 heads over 8, capped: 153 us, 7.0
// TB/s; one of 1100: 7.2 us, launch and latency; 200 of up to 333 tokens, 12 heads over 4 of 64, pages of 17 tokens: 16 us, 3.2
// TB/s: four trips of a CTA, each of which waits for its pages' numbers before it can ask for keys.
#include "span_join.cuh"
#include "span_scores.cuh"
#include "warp_mma.cuh"

namespace rb {

struct SpanDecodeParams {
  const void* q;                 // row b, head h at q[b * q_sb + h * q_sh]
  long long q_sb, q_sh;
  const void *k, *v;             // [pages, page, Hkv, D], head_major: [pages, Hkv, page, D]
  const int *tables, *ctx, *starts;
  void* out;                     // [B, H, D]
  float *part_o, *part_lse2;     // [splits, B, H, D], [splits, B, H]: parts that are no cluster
  SpanScores c;
  int B, H, Hkv, D, page, pages, max_blocks, head_blocks, splits, head_major;
};

constexpr int kSdWarps = 4, kSdKeys = 16, kSdStages = 3;
constexpr int kSdCluster = 8;

template <int HD>
struct SpanDecodeCfg {
  static constexpr int CH = HD / 8;                                   // 16-byte pieces of a row
  static constexpr int TILE = kSdKeys * HD * 2, STAGE = 2 * TILE;     // K, V
  static constexpr int SMEM_BYTES = kSdWarps * kSdStages * STAGE;
  static_assert(SMEM_BYTES >= (kSdWarps + 1) * 16 * HD * 4, "the warps' results take the ring's place");
};

template <typename T>
__device__ __forceinline__ void span_mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (UmmaFormat<T>::value == 1) mma_bf16(c, a, b0, b1);
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void span_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t span_peer(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ float4 span_peer_load4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float span_peer_load(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
template <typename T>
__device__ __forceinline__ void span_store4(T* to, float4 v) {
  *reinterpret_cast<uint2*>(to) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
}

// Eight products -> scores in log2 units.  Whole warp: as in span_score32 a vote decides between the two forms of the tanh (the general one's error grows
// with the cap, not with the scores).
template <bool CAP>
__device__ __forceinline__ void span_scale8(uint32_t* x, const SpanScores& c) {
  if constexpr (!CAP) {
    const uint64_t k = both(c.scale2);
#pragma unroll
    for (int e = 0; e < 8; e += 2) set_pair(x, e, mul_f32x2(pair_at(x, e), k));
  } else {
    float reach = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) reach = fmaxf(reach, fabsf(__uint_as_float(x[e])));
    if (__all_sync(0xffffffffu, reach <= c.near)) {
      const SpanTanh f(c, c.out2);
#pragma unroll
      for (int e = 0; e < 8; e += 2) set_pair(x, e, mul_f32x2(pair_at(x, e), f.r(pair_at(x, e))));
    } else {
#pragma unroll
      for (int e = 0; e < 8; e += 2) set_pair(x, e, mul_f32x2(span_tanh_any(x[e], x[e + 1], c), both(c.out2)));
    }
  }
}

// CLUSTER: the parts of a row are the CTAs of a cluster
template <typename T, int HD, bool CAP, bool BIAS, bool CLUSTER>
__global__ void __launch_bounds__(kSdWarps * 32, 2) span_decode_kernel(const SpanDecodeParams p) {
  using C = SpanDecodeCfg<HD>;
  extern __shared__ __align__(128) uint8_t ring_all[];
  __shared__ float s_ml[kSdWarps][16][2], s_lse[16];
  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31, row_l = lane >> 2, quad = lane & 3;
  const int sp = blockIdx.x % p.splits;
  int idx = blockIdx.x / p.splits;
  const int rep = p.H / p.Hkv, hb = idx % p.head_blocks;
  idx /= p.head_blocks;
  const int g = idx % p.Hkv, b = idx / p.Hkv;
  const int h0 = g * rep + hb * 16, nh = min(16, rep - hb * 16);
  const long long room = static_cast<long long>(p.max_blocks) * p.page;
  const int ctx = p.ctx[b];
  int end = static_cast<int>(min(static_cast<long long>(max(ctx, 0)), room));
  int begin = p.starts != nullptr ? max(p.starts[b], 0) : 0;
  const int* table = p.tables + static_cast<long long>(b) * p.max_blocks;
  if constexpr (CAP && BIAS) {
    // what none of these heads gives a weight to is not read, provided that the nearest token is there
    const int reach = __reduce_max_sync(0xffffffffu, lane < nh ? span_reach(p.c.far2, p.c.slopes[h0 + lane]) : 0);
    if (end - begin > reach) {
      const int page = table[(end - 1) / p.page];
      if (page >= 0 && page < p.pages) begin = end - 1 - reach;
    }
  }
  {
    const int n = max(0, end - begin), per = (n + p.splits * 64 - 1) / (p.splits * 64) * 64;      // whole trips of the CTA
    const long long from = begin + static_cast<long long>(sp) * per;
    begin = static_cast<int>(min(from, static_cast<long long>(end)));
    end = static_cast<int>(min(static_cast<long long>(end), from + per));
  }
  const T *kc = reinterpret_cast<const T*>(p.k), *vc = reinterpret_cast<const T*>(p.v);
  const uint32_t ring = smem_u32(ring_all) + warp * kSdStages * C::STAGE;

  uint32_t seen_at[kSdStages];
  // group i of this warp into stage st; which of its 16 keys are there
  auto fetch = [&](int i, int st) -> uint32_t {
    const int t = begin + (i * kSdWarps + warp) * kSdKeys + lane;
    bool there = lane < kSdKeys && t < end;
    long long at = 0;
    if (there) {
      const int blk = t / p.page, page = table[blk], in = t - blk * p.page;
      there = page >= 0 && page < p.pages;
      if (there)
        at = (p.head_major ? (static_cast<long long>(page) * p.Hkv + g) * p.page + in : (static_cast<long long>(page) * p.page + in) * p.Hkv + g) * p.D;
    }
    const uint32_t bits = __ballot_sync(0xffffffffu, there);
    const uint32_t dst = ring + st * C::STAGE;
#pragma unroll
    for (int u = 0; u < kSdKeys * C::CH / 32; ++u) {
      const int c = lane + u * 32, key = c / C::CH, piece = c % C::CH;
      const long long from = __shfl_sync(0xffffffffu, at, key) + piece * 8;
      const bool live = (bits >> key & 1) && piece * 8 < p.D;
      const uint32_t to = dst + tile_at<C::CH>(key, piece);
      copy16(to, kc + (live ? from : 0), live);
      copy16(to + C::TILE, vc + (live ? from : 0), live);
    }
    return bits;
  };
  const int mine = end - begin - warp * kSdKeys;
  const int n = mine > 0 ? (mine + kSdWarps * kSdKeys - 1) / (kSdWarps * kSdKeys) : 0;
#pragma unroll
  for (int s = 0; s < kSdStages - 1; ++s) {
    seen_at[s] = s < n ? fetch(s, s) : 0;
    copy_commit();
  }
  // queries: rows row_l and row_l + 8 of the left operand
  uint32_t qa[HD / 16][4];
  {
    const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_sb + h0 * p.q_sh;
#pragma unroll
    for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = row_l + (e & 1) * 8, d = kk * 16 + quad * 2 + (e >> 1) * 8;
        qa[kk][e] = r < nh && d < p.D ? *reinterpret_cast<const uint32_t*>(q + r * p.q_sh + d) : 0u;
      }
  }
  float slope[2] = {0.f, 0.f};
  if constexpr (BIAS) {
#pragma unroll
    for (int r = 0; r < 2; ++r)
      if (row_l + r * 8 < nh) slope[r] = p.c.slopes[h0 + row_l + r * 8] * kLog2e;
  }
  float o[HD / 8][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < HD / 8; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) o[i][e] = 0.f;

  const int mat = lane >> 3, mr = lane & 7;
  for (int i0 = 0; i0 < n; i0 += kSdStages) {
#pragma unroll
    for (int st = 0; st < kSdStages; ++st) {          // unrolled: which keys of a stage are there stays in a register
      const int i = i0 + st;
      if (i >= n) break;
      copy_wait<kSdStages - 2>();
      __syncwarp();
      {
        constexpr int A = kSdStages - 1;
        const int next = (st + A) % kSdStages;
        seen_at[next] = i + A < n ? fetch(i + A, next) : 0;
        copy_commit();
      }
      const uint32_t kt = ring + st * C::STAGE, vt = kt + C::TILE, seen = seen_at[st];
      float s[2][4];
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e) s[j][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < HD / 16; ++kk) {
        uint32_t r[4];
        ldmatrix_x4(kt + tile_at<C::CH>((mat >> 1) * 8 + mr, kk * 2 + (mat & 1)), r);
        span_mma<T>(s[0], qa[kk], r[0], r[1]);
        span_mma<T>(s[1], qa[kk], r[2], r[3]);
      }
      uint32_t x[8];                                  // [8-key half][row, row + 8][key, key + 1]
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = __float_as_uint(s[e >> 2][e & 3]);
      span_scale8<CAP>(x, p.c);
      const int key0 = begin + (i * kSdWarps + warp) * kSdKeys + quad * 2;
      if constexpr (BIAS) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          x[e] = __float_as_uint(fmaf(-slope[(e >> 1) & 1], (float)(ctx - 1 - (key0 + (e >> 2) * 8 + (e & 1))), __uint_as_float(x[e])));
      }
      if (seen != 0xffffu) {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (!(seen >> (quad * 2 + (e >> 2) * 8 + (e & 1)) & 1)) x[e] = 0xff800000u;
      }
      float top[2], neg[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        top[r] = fmaxf(fmaxf(__uint_as_float(x[r * 2]), __uint_as_float(x[r * 2 + 1])), fmaxf(__uint_as_float(x[4 + r * 2]), __uint_as_float(x[5 + r * 2])));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 1));
        top[r] = fmaxf(top[r], __shfl_xor_sync(0xffffffffu, top[r], 2));
        top[r] = fmaxf(m[r], top[r]);
      }
      if (__any_sync(0xffffffffu, top[0] > m[0] || top[1] > m[1])) {
        float f[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          f[r] = m[r] == -INFINITY ? 0.f : fast_exp2(m[r] - top[r]);
          l[r] *= f[r];
          m[r] = top[r];
        }
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          o[c][0] *= f[0]; o[c][1] *= f[0];
          o[c][2] *= f[1]; o[c][3] *= f[1];
        }
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) neg[r] = m[r] == -INFINITY ? 0.f : -m[r];
      float w[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        w[e] = fast_exp2(__uint_as_float(x[e]) + neg[(e >> 1) & 1]);
        l[(e >> 1) & 1] += w[e];
      }
      const uint32_t pa[4] = {pack2<T>(w[0], w[1]), pack2<T>(w[2], w[3]), pack2<T>(w[4], w[5]), pack2<T>(w[6], w[7])};
#pragma unroll
      for (int c = 0; c < HD / 16; ++c) {
        uint32_t r[4];
        ldmatrix_x4_trans(vt + tile_at<C::CH>((mat & 1) * 8 + mr, c * 2 + (mat >> 1)), r);
        span_mma<T>(o[2 * c], pa, r[0], r[1]);
        span_mma<T>(o[2 * c + 1], pa, r[2], r[3]);
      }
      __syncwarp();                                   // the stage is asked for again in the next trip
    }
  }

  // the four warps' results meet in shared memory (in the ring's place)
  copy_wait<0>();
  __syncthreads();
  float* s_o = reinterpret_cast<float*>(ring_all);    // [warps][16][HD], then [16][HD]
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 1);
    l[r] += __shfl_xor_sync(0xffffffffu, l[r], 2);
    if (quad == 0) {
      s_ml[warp][row_l + r * 8][0] = m[r];
      s_ml[warp][row_l + r * 8][1] = l[r];
    }
#pragma unroll
    for (int c = 0; c < HD / 8; ++c)
      *reinterpret_cast<float2*>(s_o + (warp * 16 + row_l + r * 8) * HD + c * 8 + quad * 2) = make_float2(o[c][r * 2], o[c][r * 2 + 1]);
  }
  __syncthreads();
  float* s_out = s_o + kSdWarps * 16 * HD;
  const int pieces = nh * (HD / 4);
  T* out = reinterpret_cast<T*>(p.out) + (static_cast<long long>(b) * p.H + h0) * p.D;
  for (int i = threadIdx.x; i < pieces; i += kSdWarps * 32) {
    const int r = i / (HD / 4), d = i % (HD / 4) * 4;
    float top = -INFINITY, sum = 0.f;
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) top = fmaxf(top, s_ml[w][r][0]);
    float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kSdWarps; ++w) {
      if (s_ml[w][r][1] == 0.f) continue;             // no key
      const float e = fast_exp2(s_ml[w][r][0] - top);
      const float4 y = *reinterpret_cast<const float4*>(s_o + (w * 16 + r) * HD + d);
      sum = fmaf(e, s_ml[w][r][1], sum);
      f.x = fmaf(e, y.x, f.x); f.y = fmaf(e, y.y, f.y); f.z = fmaf(e, y.z, f.z); f.w = fmaf(e, y.w, f.w);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    f.x *= inv; f.y *= inv; f.z *= inv; f.w *= inv;
    const float lse2 = sum == 0.f ? -INFINITY : top + log2f(sum);
    if (CLUSTER) {
      *reinterpret_cast<float4*>(s_out + r * HD + d) = f;
      if (d == 0) s_lse[r] = lse2;
    } else if (d < p.D) {
      if (p.splits == 1) {
        span_store4(out + r * p.D + d, f);
      } else {
        const long long at = (static_cast<long long>(sp) * p.B + b) * p.H + h0 + r;
        *reinterpret_cast<float4*>(p.part_o + at * p.D + d) = f;
        if (d == 0) p.part_lse2[at] = lse2;
      }
    }
  }
  if constexpr (CLUSTER) {
    span_cluster_sync();
    for (int i = sp * kSdWarps * 32 + threadIdx.x; i < pieces; i += p.splits * kSdWarps * 32) {
      const int r = i / (HD / 4), d = i % (HD / 4) * 4;
      float e[kSdCluster], top = -INFINITY, sum = 0.f;
#pragma unroll
      for (int c = 0; c < kSdCluster; ++c) {
        e[c] = c < p.splits ? span_peer_load(span_peer(smem_u32(&s_lse[r]), c)) : -INFINITY;
        top = fmaxf(top, e[c]);
      }
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int c = 0; c < kSdCluster; ++c) {
        if (e[c] == -INFINITY) continue;              // no key in this part
        const float w = fast_exp2(e[c] - top);
        const float4 y = span_peer_load4(span_peer(smem_u32(s_out + r * HD + d), c));
        sum += w;
        f.x = fmaf(w, y.x, f.x); f.y = fmaf(w, y.y, f.y); f.z = fmaf(w, y.z, f.z); f.w = fmaf(w, y.w, f.w);
      }
      const float inv = sum == 0.f ? 0.f : 1.f / sum;
      if (d < p.D) span_store4(out + r * p.D + d, make_float4(f.x * inv, f.y * inv, f.z * inv, f.w * inv));
    }
    span_cluster_sync();                              // no CTA leaves while another one reads its memory
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
int launch_span_decode(const SpanDecodeParams& p, unsigned grid, cudaStream_t st) {
  const bool cluster = p.splits > 1 && p.splits <= kSdCluster;
  auto kern = cluster ? span_decode_kernel<T, HD, CAP, BIAS, true> : span_decode_kernel<T, HD, CAP, BIAS, false>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SpanDecodeCfg<HD>::SMEM_BYTES);
  if (e != cudaSuccess) return 2000 + (int)e;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(kSdWarps * 32);
  cfg.dynamicSmemBytes = SpanDecodeCfg<HD>::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster ? p.splits : 1;
  at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, kern, p);
  if (e != cudaSuccess) return 3000 + (int)e;
  if (p.splits > kSdCluster)
    return launch_span_join<T>(p.part_o, p.part_lse2, (T*)p.out, nullptr, p.B, p.H, 1, p.D, p.splits, st);
  return 0;
}

template <typename T>
int span_decode(const SpanDecodeParams& p, bool cap, unsigned grid, cudaStream_t st) {
  const bool bias = p.c.slopes != nullptr;
#define RB_SPAN(HD_)                                                                                                          \
  (cap ? bias ? launch_span_decode<T, HD_, true, true>(p, grid, st) : launch_span_decode<T, HD_, true, false>(p, grid, st)    \
       : bias ? launch_span_decode<T, HD_, false, true>(p, grid, st) : launch_span_decode<T, HD_, false, false>(p, grid, st))
  return p.D <= 64 ? RB_SPAN(64) : RB_SPAN(128);
#undef RB_SPAN
}

}  // namespace rb

extern "C" {

// Parts that contexts of up to max_ctx tokens are cut into, for B sequences of Hkv key heads that H query heads share: as many as fill every SM with two
// CTAs, in a cluster of 2, 4 or 8 of one trip (64 keys) each at least, or, where 8 would have more than 1536 keys each, through memory, of 512 at least.  us at
// several numbers, heads of 128, the rule's in brackets: 1 x 300 tokens, 32 heads over 8: 7.7 with 1 part, 7.0 with 2, [6.2 with 4], 5.6 with 8; 1 x 1100:
// 17.8 with 1, 8.8 with 4, [7.4 with 8], 10.4 with 12; 8 x 32768: 204 with 2, [153 with 4], 158 with 8; 48 x 1250, 32 key heads: [158 with 1], 176 with 2;
// over 2 heads of 64, 2 x 9000: [15.6 with 8], 17.3 with 18; 2 x 12000: [19.1 with 8], 18.3 with 24; 1 x 40000: 65.8 with 8, 34.8 with 24, [35.9 with 64].
int rb_span_decode_splits(int B, int H, int Hkv, int max_ctx) {
  if (B <= 0 || Hkv <= 0 || H <= 0) return 1;
  const long long rows = static_cast<long long>(B) * Hkv * ((H / Hkv + 15) / 16);
  const bool memory = max_ctx > rb::kSdCluster * 1536;
  const long long each = memory ? 512 : 64, most = (max_ctx + each - 1) / each, fill = 2ll * rbh::sm_count() / rows;
  long long s = fill < most ? fill : most;
  if (s < 1) s = 1;
  if (s > 64) s = 64;
  if (!memory || s < 2 * rb::kSdCluster) {
    if (s > rb::kSdCluster) s = rb::kSdCluster;
    while (s & (s - 1)) s &= s - 1;            // clusters of 2, 4, 8
  }
  return static_cast<int>(s);
}

// q [B, H, D] with strides q_sb, q_sh in elements, rows 4-byte aligned; caches contiguous, 16-byte aligned, of `pages` pages of `page` tokens; tables [B, max_blocks];
// ctx, starts (or null) [B]; D a multiple of 8, at most 128; out [B, H, D] contiguous, 8-byte aligned.  splits > 8: part_o [splits, B, H, D], 16-byte
// aligned, and part_lse2 [splits, B, H] are scratch.
int rb_span_decode(int dtype, int head_major, const void* q, long long q_sb, long long q_sh, const void* k, const void* v, const int* tables, const int* ctx,
                   const int* starts, const float* slopes, void* out, float* part_o, float* part_lse2, int B, int H, int Hkv, int D, int page, int pages,
                   int max_blocks, int splits, float scale, float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0) return 0;
  if (Hkv <= 0 || H % Hkv || D <= 0 || D > 128 || D % 8 || page <= 0 || pages < 0 || max_blocks < 0 || splits < 1) return 20;
  if (splits > kSdCluster ? !part_o || !part_lse2 : (splits & (splits - 1)) != 0) return 20;
  const auto off = [](const void* at, uintptr_t bytes) { return reinterpret_cast<uintptr_t>(at) % bytes != 0; };
  if (off(out, 8) || off(q, 4) || off(k, 16) || off(v, 16) || off(part_o, 16)) return 20;
  SpanDecodeParams p{};
  p.q = q; p.q_sb = q_sb; p.q_sh = q_sh; p.k = k; p.v = v; p.tables = tables; p.ctx = ctx; p.starts = starts;
  p.out = out; p.part_o = part_o; p.part_lse2 = part_lse2;
  p.c = rbh::span_scores(scale, cap);
  p.c.slopes = slopes;
  p.B = B; p.H = H; p.Hkv = Hkv; p.D = D; p.page = page; p.pages = pages; p.max_blocks = max_blocks; p.splits = splits; p.head_major = head_major;
  p.head_blocks = (H / Hkv + 15) / 16;
  const long long grid = static_cast<long long>(B) * Hkv * p.head_blocks * splits;
  if (grid > 0x7fffffffll) return 20;
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == rbh::DT_BF16) return span_decode<__nv_bfloat16>(p, cap > 0.f, (unsigned)grid, st);
  if (dtype == rbh::DT_F16) return span_decode<__half>(p, cap > 0.f, (unsigned)grid, st);
  return 20;
}
}
