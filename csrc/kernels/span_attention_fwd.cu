// Span attention forward for sm_100a (tcgen05 + TMEM + TMA): softmax(cap tanh(scale q.k / cap) - slope |distance|) V over the keys lo <= j < hi of
// each row, 16-bit, heads of 8 to 128 numbers.
//
// A CTA owns two tiles of 128 query rows of one head, each with a warpgroup of its own (a thread owns a row: maximum and sum never leave it) and its
// own S and O in tensor memory.  Tiles of 128 keys and of 128 values take turns in one ring of shared memory and serve both query tiles.  P
// (16-bit) lies over the first half of its S, from where P V reads it as left operand, and the next S of the tile follows that product in the
// issue order, so what a warpgroup waits for, S of its next tile, also says that P and O are at rest.  While one warpgroup waits for the tensor
// core the other one computes.  O is rescaled only when a row's maximum moved by more than 2^8.
//
// Keys that no row of a tile reaches are not read: each query tile goes over the tiles from its least lo to its largest hi.  Few rows over many
// keys would leave most SMs idle, so such calls cut the tiles of keys into `splits` parts, whose results (fp32, with their log-sum-exp) a second
// kernel joins.
#include "span_join.cuh"
#include "span_scores.cuh"

namespace rb {

struct SpanFwdParams {
  int B, H, Hkv, Sq, Sk, D;
  int q_tiles, splits;
  SpanScores c;
  void* o;           // [B, Sq, H, D]
  float* lse2;       // [B, H, Sq] log-sum-exp in log2 units, -inf: the row sees no key
  float* part_o;     // [splits, B, Sq, H, D] (splits > 1)
  float* part_lse2;  // [splits, B, H, Sq]
  int* status;
};

template <int HD>
struct SpanFwdCfg {
  static constexpr int SUB = HD / 64;                 // 64-column sub-tiles of a row
  static constexpr int SUB_BYTES = 128 * 128;         // [128 x 64] 16-bit
  static constexpr int TILE = SUB * SUB_BYTES;
  static constexpr int SLOTS = HD == 128 ? 5 : 9;     // K and V tiles in flight, in turn
  static constexpr int SMEM_BYTES = (2 + SLOTS) * TILE + 1024 + 256;
  static constexpr int S_COL = 0, O_COL = 256;        // of query tile x: + x * 128
};

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(320, 1)
    span_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const SpanFwdParams p) {
  using C = SpanFwdCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                                  // [2][TILE]
  uint8_t* sKV = sQ + 2 * C::TILE;                     // [SLOTS][TILE]: K0 V0 K1 V1 ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + C::SLOTS * C::TILE);
  uint64_t *q_full = bars, *full = bars + 1, *empty = full + C::SLOTS, *s_full = empty + C::SLOTS, *p_ready = s_full + 2, *o_done = p_ready + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(o_done + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  __shared__ int4 s_range[8];

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  int idx = blockIdx.x;
  const int q_tile = p.q_tiles - 1 - idx % p.q_tiles;  // causal: the longest first
  idx /= p.q_tiles;
  const int sp = idx % p.splits;
  idx /= p.splits;
  const int h = idx % p.H, b = idx / p.H;
  const int hkv = h / (p.H / p.Hkv);
  const int q0 = q_tile * 256, off = p.Sk - p.Sq;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tq);
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
    mbar_init(smem_u32(q_full), 1);
    for (int s = 0; s < C::SLOTS; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int x = 0; x < 2; ++x) {
      mbar_init(smem_u32(&s_full[x]), 1);
      mbar_init(smem_u32(&p_ready[x]), 128);
      mbar_init(smem_u32(&o_done[x]), 1);
    }
    *abort_flag = 0;
    fence_barrier_init();
  }
  int2 span = make_int2(0, 0);
  if (warp < 8) {
    const int row = q0 + threadIdx.x;
    const bool live = row < p.Sq;
    if (live) span = span_of(p.c, b, row, p.Sq, p.Sk);
    const int4 r = span_range_warp(span, live);
    if (lane == 0) s_range[warp] = r;
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_ptr), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;

  // tiles of keys [first, last) of each query tile, and of both
  int first[2], last[2], lo_all[2], hi_all[2];
#pragma unroll
  for (int x = 0; x < 2; ++x) {
    const int4 r = span_range_join(span_range_join(s_range[4 * x], s_range[4 * x + 1]), span_range_join(s_range[4 * x + 2], s_range[4 * x + 3]));
    first[x] = r.x < r.y ? r.x / 128 : 0;
    last[x] = r.x < r.y ? (r.y + 127) / 128 : 0;
    lo_all[x] = r.z;
    hi_all[x] = r.w;
  }
  int j0, j1;
  {
    const bool a = first[0] < last[0], c = first[1] < last[1];
    j0 = a && c ? min(first[0], first[1]) : a ? first[0] : first[1];
    j1 = max(last[0], last[1]);
    const int per = (j1 - j0 + p.splits - 1) / p.splits;
    const int from = j0 + sp * per, to = min(j1, from + per);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      first[x] = max(first[x], from);
      last[x] = max(first[x], min(last[x], to));
    }
    j0 = from;
    j1 = max(from, to);
  }
  const int n = j1 - j0;
  auto active = [&](int x, int j) { return first[x] <= j && j < last[x]; };

  if (warp == 8) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0 && n > 0) {
      const bool two = q0 + 128 < p.Sq;
      mbar_arrive_expect_tx(smem_u32(q_full), (two ? 2 : 1) * C::TILE);
#pragma unroll
      for (int s = 0; s < C::SUB; ++s) {
        tma_load_4d(smem_u32(sQ + s * C::SUB_BYTES), &tq, smem_u32(q_full), s * 64, q0, h, b);
        if (two) tma_load_4d(smem_u32(sQ + C::TILE + s * C::SUB_BYTES), &tq, smem_u32(q_full), s * 64, q0 + 128, h, b);
      }
      bool ok = true;
      int slot = 0;
      uint32_t ph = 0;
      for (int i = 0; i < 2 * n; ++i) {
        ok = mbar_wait(smem_u32(&empty[slot]), ph ^ 1, abort_flag, p.status, RB_ERR_TIMEOUT_EMPTY);
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[slot]);
        mbar_arrive_expect_tx(bar, C::TILE);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s)
          tma_load_4d(smem_u32(sKV + slot * C::TILE + s * C::SUB_BYTES), i & 1 ? &tv : &tk, bar, s * 64, (j0 + (i >> 1)) * 128, hkv, b);
        if (++slot == C::SLOTS) { slot = 0; ph ^= 1; }
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(10000);      // copies in flight land before the CTA's memory goes
    }
  } else if (warp == 9) {
    // ------------------------------ MMA issuer --------------------------------
    if (n > 0) {
      constexpr uint32_t idesc_s = make_idesc(UmmaFormat<T>::value, 0, 0, 128, 128);
      constexpr uint32_t idesc_o = make_idesc(UmmaFormat<T>::value, 0, 1, 128, HD);
      auto issue_s = [&](int x, int slot) {
        const uint64_t qd = make_smem_desc_sw128(smem_u32(sQ + x * C::TILE), 16, 1024);
        const uint64_t kd = make_smem_desc_sw128(smem_u32(sKV + slot * C::TILE), 16, 1024);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s)
          umma_f16_w4<2, 2>(tmem_base + C::S_COL + x * 128, qd + s * (C::SUB_BYTES >> 4), kd + s * (C::SUB_BYTES >> 4), idesc_s, s != 0);
        umma_commit_w(smem_u32(&s_full[x]));
      };
      bool ok = mbar_wait(smem_u32(q_full), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      if (ok) ok = mbar_wait(smem_u32(&full[0]), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      if (ok) {
        tc_fence_after();
#pragma unroll
        for (int x = 0; x < 2; ++x)
          if (active(x, j0)) issue_s(x, 0);
        umma_commit_w(smem_u32(&empty[0]));
      }
      int slot = 1;                    // of V(j); K(j + 1) stands in the next one
      uint32_t ph = 0, p_ph[2] = {0, 0};
      for (int j = j0; j < j1 && ok; ++j) {
        const int slot_k = slot + 1 == C::SLOTS ? 0 : slot + 1;
        const uint32_t ph_k = slot + 1 == C::SLOTS ? ph ^ 1 : ph;
        const bool more = j + 1 < j1;
        bool k_here = false;
        ok = mbar_wait(smem_u32(&full[slot]), ph, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
        if (!ok) break;
        const uint64_t vd = make_smem_desc_sw128(smem_u32(sKV + slot * C::TILE), C::SUB_BYTES, 1024);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          if (ok && active(x, j)) {
            ok = mbar_wait(smem_u32(&p_ready[x]), p_ph[x], abort_flag, p.status, RB_ERR_TIMEOUT_FLAG);
            if (ok) {
              p_ph[x] ^= 1;
              tc_fence_after();
#pragma unroll
              for (int s = 0; s < 2; ++s)
                umma_f16_ts_w4<8, 128>(tmem_base + C::O_COL + x * 128, tmem_base + C::S_COL + x * 128 + s * 32, vd + s * 512, idesc_o,
                                       (j > first[x] || s != 0) ? 1u : 0u);
              if (j + 1 == last[x]) umma_commit_w(smem_u32(&o_done[x]));
            }
          }
          if (ok && more && active(x, j + 1)) {
            if (!k_here) ok = mbar_wait(smem_u32(&full[slot_k]), ph_k, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
            if (ok) {
              k_here = true;
              tc_fence_after();
              issue_s(x, slot_k);
            }
          }
        }
        if (!ok) break;
        umma_commit_w(smem_u32(&empty[slot]));
        if (more) {
          if (!k_here) ok = mbar_wait(smem_u32(&full[slot_k]), ph_k, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);   // a tile that neither reaches
          if (!ok) break;
          umma_commit_w(smem_u32(&empty[slot_k]));
        }
        slot = slot_k + 1 == C::SLOTS ? 0 : slot_k + 1;
        ph = slot_k + 1 == C::SLOTS ? ph_k ^ 1 : ph_k;
      }
    }
  } else {
    // ------------------------------ softmax warpgroups ------------------------
    const int x = warp >> 2, t = threadIdx.x & 127;
    const int row0 = q0 + x * 128, row = row0 + t;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t s_addr = lane_addr + C::S_COL + x * 128, o_addr = lane_addr + C::O_COL + x * 128;
    const int begin = x ? first[1] : first[0], end = x ? last[1] : last[0];
    const int lo_max = x ? lo_all[1] : lo_all[0], hi_min = x ? hi_all[1] : hi_all[0];
    const float slope2 = BIAS ? p.c.slopes[h] * kLog2e : 0.f;
    float m = -INFINITY, l = 0.f;                 // maximum that P is relative to, and sum
    bool ok = true;
    uint32_t ph = 0;
    for (int j = begin; j < end; ++j, ph ^= 1) {
      ok = mbar_wait(smem_u32(&s_full[x]), ph, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int kv0 = j * 128;
      uint32_t s[4][32];
#pragma unroll
      for (int c = 0; c < 4; ++c) tmem_ld_32x32b_x32(s_addr + c * 32, s[c]);
      tmem_ld_wait();
      const bool masked = kv0 < lo_max || kv0 + 128 > hi_min;
      const int side = row0 + off >= kv0 + 127 ? 1 : row0 + 127 + off <= kv0 ? -1 : 0;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        span_scale<CAP, 32>(s[c], p.c);
        if constexpr (BIAS) span_bias<-1, 32>(s[c], slope2, (float)(row + off - kv0 - c * 32), side);
      }
      if (masked) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          const uint32_t seen = span_bits(span.x - kv0 - c * 32, span.y - kv0 - c * 32);
#pragma unroll
          for (int i = 0; i < 32; ++i)
            if (!(seen >> i & 1)) s[c][i] = 0xff800000u;
        }
      }
      float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int c = 0; c < 4; ++c)
#pragma unroll
        for (int i = 0; i < 32; i += 2)
          mx4[(i >> 1) & 3] = fmaxf(fmaxf(mx4[(i >> 1) & 3], __uint_as_float(s[c][i])), __uint_as_float(s[c][i + 1]));
      const float m_new = fmaxf(m, fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])));
      const bool need = m_new > m + 8.0f;         // also the first time that the row sees a key
      if (__any_sync(0xffffffffu, need)) {        // tensor memory is accessed by whole warps
        float alpha = 1.0f;
        if (need) {
          alpha = m == -INFINITY ? 0.0f : fast_exp2(m - m_new);
          m = m_new;
          l *= alpha;
        }
        if (j > begin) {
#pragma unroll 1
          for (int c = 0; c < HD / 16; ++c) {
            uint32_t r[16];
            tmem_ld_32x32b_x16(o_addr + c * 16, r);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 16; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * alpha);
            tmem_st_32x32b_x16(o_addr + c * 16, r);
          }
        }
      }
      const float neg = m == -INFINITY ? 0.f : -m;
      const uint64_t neg2 = f32x2(neg, neg);
      uint64_t l2[2] = {0, 0};
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        uint32_t packed[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float2 y = f32x2_get(add_f32x2(f32x2(__uint_as_float(s[c][2 * i]), __uint_as_float(s[c][2 * i + 1])), neg2));
          const float p0 = fast_exp2(y.x), p1 = fast_exp2(y.y);
          l2[i & 1] = add_f32x2(l2[i & 1], f32x2(p0, p1));
          packed[i] = pack2<T>(p0, p1);
        }
        tmem_st_32x32b_x16(s_addr + c * 16, packed);
      }
      const float2 la = f32x2_get(l2[0]), lb = f32x2_get(l2[1]);
      l += (la.x + la.y) + (lb.x + lb.y);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_ready[x]));
    }
    if (ok && begin < end) {
      ok = mbar_wait(smem_u32(&o_done[x]), 0, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_EMPTY);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok) {
      const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
      const long long at = ((static_cast<long long>(b) * p.Sq + row) * p.H + h) * p.D;
      const long long part = static_cast<long long>(sp) * p.B * p.H * p.Sq;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        if (c * 32 >= p.D) break;
        uint32_t r[32];
        if (begin < end) {
          tmem_ld_32x32b_x32(o_addr + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int i = 0; i < 32; ++i) r[i] = 0;
        }
        if (row >= p.Sq) continue;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          if (c * 32 + g * 8 >= p.D) break;
          float f[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) f[i] = l == 0.f ? 0.f : __uint_as_float(r[g * 8 + i]) * inv;
          if (p.splits == 1) {
            *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + at + c * 32 + g * 8) =
                make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
          } else {
            float4* to = reinterpret_cast<float4*>(p.part_o + part * p.D + at + c * 32 + g * 8);
            to[0] = make_float4(f[0], f[1], f[2], f[3]);
            to[1] = make_float4(f[4], f[5], f[6], f[7]);
          }
        }
      }
      if (row < p.Sq) {
        const long long r = (static_cast<long long>(b) * p.H + h) * p.Sq + row;
        const float v = l == 0.f ? -INFINITY : m + log2f(l);
        if (p.splits == 1) p.lse2[r] = v;
        else p.part_lse2[part + r] = v;
      }
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
int launch_span_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const SpanFwdParams& p, unsigned grid, cudaStream_t st) {
  auto kern = span_fwd_kernel<T, HD, CAP, BIAS>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SpanFwdCfg<HD>::SMEM_BYTES);
  if (e != cudaSuccess) return 2000 + (int)e;
  kern<<<grid, 320, SpanFwdCfg<HD>::SMEM_BYTES, st>>>(tq, tk, tv, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 3000 + (int)e;
}

template <typename T>
int span_fwd(int dtype, const void* q, const void* k, const void* v, const long long* qs, const long long* ks, const long long* vs, SpanFwdParams p,
             bool cap, cudaStream_t st) {
  CUtensorMap tq, tk, tv;
  int rc = rbh::span_map(&tq, dtype, q, qs, p.B, p.Sq, p.H, p.D, 128);
  if (!rc) rc = rbh::span_map(&tk, dtype, k, ks, p.B, p.Sk, p.Hkv, p.D, 128);
  if (!rc) rc = rbh::span_map(&tv, dtype, v, vs, p.B, p.Sk, p.Hkv, p.D, 128);
  if (rc) return 1000 + rc;
  const long long grid = static_cast<long long>(p.q_tiles) * p.splits * p.H * p.B;
  if (grid > 0x7fffffffll) return 20;
  const bool bias = p.c.slopes != nullptr;
#define RB_SPAN(HD_)                                                                                      \
  (cap ? bias ? launch_span_fwd<T, HD_, true, true>(tq, tk, tv, p, (unsigned)grid, st)                    \
              : launch_span_fwd<T, HD_, true, false>(tq, tk, tv, p, (unsigned)grid, st)                   \
       : bias ? launch_span_fwd<T, HD_, false, true>(tq, tk, tv, p, (unsigned)grid, st)                   \
              : launch_span_fwd<T, HD_, false, false>(tq, tk, tv, p, (unsigned)grid, st))
  rc = p.D <= 64 ? RB_SPAN(64) : RB_SPAN(128);
#undef RB_SPAN
  if (rc || p.splits == 1) return rc;
  return launch_span_join<T>(p.part_o, p.part_lse2, (T*)p.o, p.lse2, p.B, p.H, p.Sq, p.D, p.splits, st);
}

}  // namespace rb

extern "C" {

// Parts that the keys of a call are cut into: as many as fill the SMs once where the tiles of 256 rows alone leave half of them idle, each of four
// tiles of 128 keys at least.
int rb_span_fwd_splits(int B, int H, int Sq, int Sk) {
  const long long tiles = static_cast<long long>((Sq + 255) / 256) * B * H;
  if (tiles <= 0 || 2 * tiles > rbh::sm_count()) return 1;
  const long long most = (static_cast<long long>(Sk) + 511) / 512, fill = rbh::sm_count() / tiles;
  return static_cast<int>(most < 1 ? 1 : fill < most ? fill : most);
}

// q [B, Sq, H, D], k and v [B, Sk, Hkv, D]: 16-bit views, strides {batch, row, head} in elements (multiples of 8), 16-byte aligned; D a multiple of 8, at
// most 128.  o [B, Sq, H, D] contiguous, lse2 [B, H, Sq].  spans: rows {lo, hi} of int32, `span_batch` rows apart per batch, or null; slopes [H] or
// null; cap 0: none.  splits > 1: part_o [splits, B, Sq, H, D] and part_lse2 [splits, B, H, Sq] are scratch.
int rb_span_fwd(int dtype, const void* q, const void* k, const void* v, const long long* qs, const long long* ks, const long long* vs, const int* spans,
                long long span_batch, const float* slopes, void* o, float* lse2, float* part_o, float* part_lse2, int B, int H, int Hkv, int Sq, int Sk,
                int D, int splits, int causal, float scale, float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0 || Sq <= 0) return 0;
  if (Sk <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 128 || D % 8 || splits < 1 || (splits > 1 && (!part_o || !part_lse2))) return 20;
  SpanFwdParams p{};
  p.B = B; p.H = H; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.D = D;
  p.q_tiles = (Sq + 255) / 256;
  p.splits = splits;
  p.c.scale2 = scale * kLog2e;
  p.c.in = cap > 0.f ? scale / cap : 0.f;
  p.c.out2 = cap * kLog2e;
  p.c.slopes = slopes;
  p.c.spans = reinterpret_cast<const int2*>(spans);
  p.c.span_batch = span_batch;
  p.c.causal = causal;
  p.o = o; p.lse2 = lse2; p.part_o = part_o; p.part_lse2 = part_lse2;
  p.status = rbh::device_status_word();
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == rbh::DT_BF16) return span_fwd<__nv_bfloat16>(dtype, q, k, v, qs, ks, vs, p, cap > 0.f, st);
  if (dtype == rbh::DT_F16) return span_fwd<__half>(dtype, q, k, v, qs, ks, vs, p, cap > 0.f, st);
  return 20;
}
}
