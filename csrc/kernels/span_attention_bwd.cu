// Span attention backward for sm_100a (tcgen05 + TMEM + TMA), 16-bit, heads of 8 to 128 numbers.  With the scores x and weights p of the forward pass,
// t = tanh(scale q.k / cap), and delta = sum dO O of a row:
//
//   dP = dO V^T,  dS = p (dP - delta) (1 - t^2),  dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO
//
// Two kernels, so that every gradient is summed in one order (no atomics: the same inputs give the same gradients): dQ by tiles of query rows, then
// dK and dV by tiles of keys.  Both recompute S and dP; the two extra products cost what the atomics of a joint kernel would.  P and dS stay in tensor
// memory, where the next product takes them as its left operand.  Where few key heads leave SMs idle several CTAs share a tile of keys, and only then do
// sums pass through memory in fp32 (rb_span_bwd_parts).
//
// Bound by the softmax warps and the hand-over of tiles between them and the products: a 128 x 64 tile takes 1900 (biased) to 2500 cycles (capped) in
// either kernel, of which its four products fill 1280.  A CTA's beginning and end take 6000 to 8000 more.  Heads of 128, dQ and dK, dV: 4 x 1024 rows, 8
// heads, biased: 29 and 33 us; 8 x 2048 rows in 4 documents each, 16 heads, capped: 229 and 232 us, 222 TFLOP/s (8 operations a visible pair and number)
// together; 8192 rows, 16 heads over 4, capped and biased: 334 and 388 + 15 us for joining two parts.
//
// The first kernel also writes what the second one asks per query row: log-sum-exp, delta and the span, and per 32 rows the range of their spans,
// by which the second kernel leaves out tiles that do not reach its keys.  dS is rounded to 16 bits before the scale, which keeps small gradients
// of fp16 heads away from its subnormal numbers.
#include "span_scores.cuh"

#include <type_traits>

namespace rb {

struct SpanBwdParams {
  int B, H, Hkv, Sq, Sk, D;
  SpanOrder order;                  // of the launch: tiles of rows and heads, or tiles of keys and key heads
  SpanScores c;
  float grad_scale;                 // scale, negated with a cap (span_score32 gives its derivative negated)
  const float* lse2;                // [B, H, Sq]
  // per row, rows padded to a multiple of 64 (zeros there)
  float *row_lse2, *row_delta;      // [B, H, sq_pad], both negated
  int *row_lo, *row_hi;             // [B, sq_pad]
  int4* range;                      // [B, sq_pad / 32], with a bias [B, H, sq_pad / 32]: span_range_warp of 32 rows
  int sq_pad;
  void *dk, *dv;                    // [B, Sk, Hkv, D], dkvs: strides {batch, row, head}
  long long dkvs[3];
  int parts;                        // CTAs that share a tile of keys
  float* sums;                      // several parts: [parts, B, Hkv, tiles of 128 keys][dV, dK][HD / 32][128 keys][32, 16-byte pieces swizzled by the key]
  int* status;
};

template <typename T>
__device__ __forceinline__ void span_pack32(const uint32_t* f, uint32_t* w) {
#pragma unroll
  for (int i = 0; i < 16; ++i) w[i] = pack2<T>(__uint_as_float(f[2 * i]), __uint_as_float(f[2 * i + 1]));
}

// ---------------------------------------------------------------- dQ
// A CTA owns 128 query rows of a head and goes over tiles of 64 keys; two warpgroups take the tiles in turn, a thread owns a row.
//
// delta from the rounded O is off by 2^-9 of the row's gradient, which is more than dS itself where one key has nearly all the weight.  So the sweep takes
// it as a first guess d0 only, sums delta = sum p dP in fp32 beside, and corrects the result: dQ = scale (sum g (dP - d0) K + (d0 - delta) sum g K) with
// g = p (1 - t^2); sum g K is one product more, and the second kernel gets the exact delta.  (Gradients of bfloat16 heads with scores of deviation 4:
// 1.2 % off without it, 0.24 % with it; the roundings of dS and of the result leave 0.23 %.)
template <int HD>
struct SpanDqCfg {
  static constexpr int SUB = HD / 64, KV_SUB = 64 * 128, TILE = SUB * KV_SUB;          // 64 keys
  static constexpr int ROW_SUB = 128 * 128, ROWS = SUB * ROW_SUB;                       // 128 rows: as much as a stage's K and V
  static constexpr int STAGES = HD == 128 ? 4 : 8;
  static constexpr int SMEM_BYTES = 2 * ROWS + STAGES * 2 * TILE + 1024 + 256;
  static_assert(ROWS == 2 * TILE, "O lies in the last stage at first");
  static constexpr int DQ_COL = 0, GK_COL = 128, S_COL = 256, DP_COL = 384;     // S (then g and dS), dP of buffer w: + 64 w
};

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(320, 1)
    span_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo, const __grid_constant__ CUtensorMap to,
                   const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv, const __grid_constant__ CUtensorMap tdq,
                   const SpanBwdParams p) {
  using C = SpanDqCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* sQ = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sdO = sQ + C::ROWS;
  uint8_t* ring = sdO + C::ROWS;                                 // [STAGES] {K, V}
  uint8_t* sO = ring + (C::STAGES - 1) * 2 * C::TILE;
  uint64_t* bars = reinterpret_cast<uint64_t*>(ring + C::STAGES * 2 * C::TILE);
  uint64_t *full = bars, *empty = full + C::STAGES, *sdp_full = empty + C::STAGES, *ds_ready = sdp_full + 2, *dq_done = ds_ready + 2,
           *rows_full = dq_done + 1, *rows_read = rows_full + 1;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(rows_read + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  __shared__ int4 s_range[4];
  __shared__ float s_sum[2][2][128];                             // [first guess, sum][warpgroup]

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  int tile, unit;
  span_place<true>(p.order, blockIdx.x, tile, unit);
  const int q0 = tile * 128, h = unit % p.H, b = unit / p.H, hkv = h / (p.H / p.Hkv);
  const int off = p.Sk - p.Sq;
  const int t = threadIdx.x & 127, wg = warp >> 2, row = q0 + t;
  const bool live = row < p.Sq;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&sdp_full[w]), 1);
      mbar_init(smem_u32(&ds_ready[w]), 128);
    }
    mbar_init(smem_u32(dq_done), 1);
    mbar_init(smem_u32(rows_full), 1);
    mbar_init(smem_u32(rows_read), 256);
    *abort_flag = 0;
    fence_barrier_init();
    fence_proxy_async();
    // this thread's own barriers: the copies need no one else
    mbar_arrive_expect_tx(smem_u32(rows_full), 3 * C::ROWS);
#pragma unroll
    for (int s = 0; s < C::SUB; ++s) {
      tma_load_4d(smem_u32(sQ + s * C::ROW_SUB), &tq, smem_u32(rows_full), s * 64, q0, h, b);
      tma_load_4d(smem_u32(sdO + s * C::ROW_SUB), &tdo, smem_u32(rows_full), s * 64, q0, h, b);
      tma_load_4d(smem_u32(sO + s * C::ROW_SUB), &to, smem_u32(rows_full), s * 64, q0, h, b);
    }
  }
  int2 span = make_int2(0, 0);
  if (warp < 8) {
    if (live) span = span_of(p.c, b, row, p.Sq, p.Sk);
    const int4 r = span_range_warp(span, BIAS ? span_near(span, row + off, span_head_reach<CAP>(p.c, b, h, hkv, p.H, p.Hkv)) : span, live);
    if (warp < 4 && lane == 0) s_range[warp] = r;
  } else if (warp == 9) {
    tmem_alloc(smem_u32(tmem_ptr), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;
  const int4 all = span_range_join(span_range_join(s_range[0], s_range[1]), span_range_join(s_range[2], s_range[3]));
  const int j0 = all.x < all.y ? all.x / 64 : 0, n = all.x < all.y ? (all.y + 63) / 64 - j0 : 0;
  bool ok = true;

  if (warp == 8) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0) {
      int st = 0;
      uint32_t ph = 0;
      for (int i = 0; i < n; ++i) {
        ok = i == C::STAGES - 1 ? mbar_wait(smem_u32(rows_read), 0, abort_flag, p.status, RB_ERR_TIMEOUT_EMPTY)
                                : mbar_wait(smem_u32(&empty[st]), ph ^ 1, abort_flag, p.status, RB_ERR_TIMEOUT_EMPTY);
        if (!ok) break;
        const uint32_t bar = smem_u32(&full[st]), dst = smem_u32(ring + st * 2 * C::TILE);
        mbar_arrive_expect_tx(bar, 2 * C::TILE);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s) {
          tma_load_4d(dst + s * C::KV_SUB, &tk, bar, s * 64, (j0 + i) * 64, hkv, b);
          tma_load_4d(dst + C::TILE + s * C::KV_SUB, &tv, bar, s * 64, (j0 + i) * 64, hkv, b);
        }
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(10000);
    }
  } else if (warp == 9) {
    // ------------------------------ MMA issuer --------------------------------
    constexpr uint32_t idesc_s = make_idesc(UmmaFormat<T>::value, 0, 0, 128, 64);
    constexpr uint32_t idesc_q = make_idesc(UmmaFormat<T>::value, 0, 1, 128, HD);
    const uint64_t qd = make_smem_desc_sw128(smem_u32(sQ), 16, 1024), dod = make_smem_desc_sw128(smem_u32(sdO), 16, 1024);
    int st_in = 0, st_out = 0;
    uint32_t ph_in = 0;
    auto issue = [&](int i) {            // S and dP of tile i, the next stage
      ok = mbar_wait(smem_u32(&full[st_in]), ph_in, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      if (!ok) return;
      tc_fence_after();
      const uint32_t k = smem_u32(ring + st_in * 2 * C::TILE);
      const uint64_t kd = make_smem_desc_sw128(k, 16, 1024), vd = make_smem_desc_sw128(k + C::TILE, 16, 1024);
#pragma unroll
      for (int s = 0; s < C::SUB; ++s) {
        umma_f16_w4<2, 2>(tmem_base + C::S_COL + (i & 1) * 64, qd + s * (C::ROW_SUB >> 4), kd + s * (C::KV_SUB >> 4), idesc_s, s != 0);
        umma_f16_w4<2, 2>(tmem_base + C::DP_COL + (i & 1) * 64, dod + s * (C::ROW_SUB >> 4), vd + s * (C::KV_SUB >> 4), idesc_s, s != 0);
      }
      umma_commit_w(smem_u32(&sdp_full[i & 1]));
      if (++st_in == C::STAGES) { st_in = 0; ph_in ^= 1; }
    };
    if (n > 0) ok = mbar_wait(smem_u32(rows_full), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
    for (int i = 0; i < 2 && i < n && ok; ++i) issue(i);
    for (int i = 0; i < n && ok; ++i) {
      ok = mbar_wait(smem_u32(&ds_ready[i & 1]), (i >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_FLAG);
      if (!ok) break;
      tc_fence_after();
      const uint64_t kd = make_smem_desc_sw128(smem_u32(ring + st_out * 2 * C::TILE), C::KV_SUB, 1024);
      const uint32_t g = tmem_base + C::S_COL + (i & 1) * 64;
      umma_f16_ts_w4<8, 128>(tmem_base + C::GK_COL, g, kd, idesc_q, i != 0);
      umma_f16_ts_w4<8, 128>(tmem_base + C::DQ_COL, g + 32, kd, idesc_q, i != 0);
      umma_commit_w(smem_u32(&empty[st_out]));
      if (i + 1 == n) umma_commit_w(smem_u32(dq_done));
      if (++st_out == C::STAGES) st_out = 0;
      if (i + 2 < n) issue(i + 2);
    }
  } else {
    // ------------------------------ softmax warpgroups ------------------------
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const float slope2 = BIAS ? p.c.slopes[h] * kLog2e : 0.f;
    const uint32_t s_addr = lane_addr + C::S_COL + wg * 64, dp_addr = lane_addr + C::DP_COL + wg * 64;
    const float lse2 = live && span.x < span.y ? p.lse2[(static_cast<long long>(b) * p.H + h) * p.Sq + row] : 0.f;
    const long long at = (static_cast<long long>(b) * p.H + h) * p.sq_pad + row;
    if (wg == 0 && row < p.sq_pad) {
      p.row_lse2[at] = -lse2;
      if (h == 0) {
        p.row_lo[static_cast<long long>(b) * p.sq_pad + row] = span.x;
        p.row_hi[static_cast<long long>(b) * p.sq_pad + row] = span.y;
      }
      if (lane == 0 && (BIAS || h == 0)) {
        int4 r = s_range[warp];
        if (row + 32 > p.Sq) r.w = 0;             // rows behind the last one see nothing: their scores are masked
        p.range[(static_cast<long long>(BIAS ? unit : b) * p.sq_pad + row) / 32] = r;
      }
    }
    // first guess of delta: dO.O, half of the columns each.  By way of shared memory: a thread's own row of loads, 16 bytes of a line each, took 10000 cycles.
    ok = mbar_wait(smem_u32(rows_full), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
    ok = __all_sync(0xffffffffu, ok);
    float guess = 0.f;
#pragma unroll
    for (int c = 0; c < HD / 16; ++c) {
      const int d = wg * (HD / 2) + c * 8, in = t * 128 + (d >> 6) * C::ROW_SUB + ((((d >> 3) & 7) ^ (t & 7)) << 4);
      const uint4 v = *reinterpret_cast<const uint4*>(sdO + in), y = *reinterpret_cast<const uint4*>(sO + in);
      const uint32_t e4[4] = {v.x, v.y, v.z, v.w}, f4[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 e = unpack2<T>(e4[i]), f = unpack2<T>(f4[i]);
        guess = fmaf(e.x, f.x, fmaf(e.y, f.y, guess));
      }
    }
    fence_proxy_async_smem();                                // what was read before what a copy writes in its place: without it loads are still under way
    mbar_arrive(smem_u32(rows_read));
    s_sum[0][wg][t] = guess;
    asm volatile("bar.sync 1, 256;" ::: "memory");          // the softmax warps, also where a wait ran out
    guess = s_sum[0][0][t] + s_sum[0][1][t];
    uint64_t sum2 = 0;                                       // sum p dP of this warpgroup's tiles
    for (int i = wg; i < n && ok; i += 2) {
      ok = mbar_wait(smem_u32(&sdp_full[wg]), (i >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const int kv0 = (j0 + i) * 64;
      const bool masked = kv0 < all.z || kv0 + 64 > all.w;
      const int side = !BIAS ? 1 : p.c.causal || q0 + off >= kv0 + 63 ? 1 : q0 + 127 + off <= kv0 ? -1 : 0;
      const float slope = side > 0 ? slope2 : -slope2;
      const uint64_t minus = both(-guess);
      uint32_t g[2][16], ds[2][16];
      // g and dS of chunk c of 32 keys; PART: some of them are unseen
      auto chunk = [&](int c, auto part, uint32_t seen) {
        constexpr bool PART = decltype(part)::value;
        uint32_t s[32], dp[32], slip[32];
        tmem_ld_32x32b_x32(s_addr + c * 32, s);
        tmem_ld_32x32b_x32(dp_addr + c * 32, dp);
        tmem_ld_wait();
        if (PART) {                                          // what unseen keys hold decides nothing
          span_mask32(s, seen, 0);
          span_mask32(dp, seen, 0);
        }
        const float first = (float)(row + off - kv0 - c * 32), reach = CAP ? span_reach32(s) : 0.f;
        if (BIAS && side != 0) {
          span_score32<CAP, true>(s, p.c, SpanAdd<true, false>({fmaf(-slope, first, -lse2), slope}, nullptr), slip, reach);
        } else {
          span_score32<CAP, true>(s, p.c, SpanAdd<false, false>({-lse2, 0.f}, nullptr), slip, reach);
          if constexpr (BIAS) span_both_sides32<-1>(s, slope2, first);
        }
        if (PART) span_mask32(s, seen, 0xff800000u);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          uint64_t w = f32x2(fast_exp2(__uint_as_float(s[k])), fast_exp2(__uint_as_float(s[k + 1])));
          const uint64_t d = pair_at(dp, k);
          sum2 = fma_f32x2(w, d, sum2);
          if (CAP) w = mul_f32x2(w, pair_at(slip, k));
          const float2 a = f32x2_get(w), e = f32x2_get(mul_f32x2(w, add_f32x2(d, minus)));
          g[c][k / 2] = pack2<T>(a.x, a.y);
          ds[c][k / 2] = pack2<T>(e.x, e.y);
        }
      };
      if (!masked) {
        chunk(0, std::false_type{}, 0xffffffffu);
        chunk(1, std::false_type{}, 0xffffffffu);
      } else {
        // some chunks of a masked tile have nothing to see
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const uint32_t seen = span_bits(span.x - kv0 - c * 32, span.y - kv0 - c * 32);
          if (__all_sync(0xffffffffu, seen == 0)) {
#pragma unroll
            for (int k = 0; k < 16; ++k) g[c][k] = ds[c][k] = 0;
          } else {
            chunk(c, std::true_type{}, seen);
          }
        }
      }
      tmem_st_32x32b_x16(s_addr, g[0]);
      tmem_st_32x32b_x16(s_addr + 16, g[1]);
      tmem_st_32x32b_x16(s_addr + 32, ds[0]);
      tmem_st_32x32b_x16(s_addr + 48, ds[1]);
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&ds_ready[wg]));
    }
    const float2 part = f32x2_get(sum2);
    s_sum[1][wg][t] = part.x + part.y;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float delta = s_sum[1][0][t] + s_sum[1][1][t];
    if (wg == 1 && row < p.sq_pad) p.row_delta[at] = -delta;
    if (ok && n > 0) {
      ok = mbar_wait(smem_u32(dq_done), 0, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_EMPTY);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok) {
      // warpgroup w takes columns [w HD / 2, (w + 1) HD / 2): through shared memory, in the place of Q, and from there in whole rows
      const float slipped = guess - delta;
      uint8_t* stage = sQ + t * 128;
#pragma unroll 1
      for (int c = 0; c < HD / 64; ++c) {
        const int d0 = wg * (HD / 2) + c * 32;
        uint32_t r[32], k32[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(lane_addr + C::DQ_COL + d0, r);
          tmem_ld_32x32b_x32(lane_addr + C::GK_COL + d0, k32);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = k32[k] = 0;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = d0 + g * 8;
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int i = g * 8 + 2 * k;
            w[k] = pack2<T>(fmaf(slipped, __uint_as_float(k32[i]), __uint_as_float(r[i])) * p.grad_scale,
                            fmaf(slipped, __uint_as_float(k32[i + 1]), __uint_as_float(r[i + 1])) * p.grad_scale);
          }
          *reinterpret_cast<uint4*>(stage + (d >> 6) * C::ROW_SUB + ((((d >> 3) & 7) ^ (t & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync 1, 256;" ::: "memory");
    if (threadIdx.x == 0 && ok) {
#pragma unroll
      for (int s = 0; s < C::SUB; ++s)
        if (s * 64 < p.D) tma_store_4d(&tdq, smem_u32(sQ + s * C::ROW_SUB), s * 64, q0, h, b);
      tma_store_commit();
      tma_store_wait_read<0>();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// ---------------------------------------------------------------- dK, dV
// A CTA owns 128 keys of one key head and goes over the tiles of 64 query rows, of all query heads that share it, that reach them.  Products run on
// transposed tiles, S^T [key x row] = K Q^T and dP^T = V dO^T, so that a thread owns a key; P^T (its first 16 columns of 32) and dS^T (the other 16) lie
// over S^T and are the left operands of dV += P^T dO and dK += dS^T Q.
template <int HD>
struct SpanDkvCfg {
  static constexpr int SUB = HD / 64;
  static constexpr int KV_SUB = 128 * 128, KV_TILE = SUB * KV_SUB;      // [128 x 64] 16-bit sub-tiles
  static constexpr int Q_SUB = 64 * 128, Q_TILE = SUB * Q_SUB;
  static constexpr int STAGES = 4;                                       // Q, dO and 64 rows' {lse2, delta, lo, hi}
  static constexpr int SMEM_BYTES = 2 * KV_TILE + STAGES * (2 * Q_TILE + 1024) + 1024 + 256;
  static constexpr int ST_COL = 0, DP_COL = 128, DV_COL = 256, DK_COL = 384;     // S^T, dP^T of buffer w: + 64 w
};

__device__ __forceinline__ void bulk_store_1d(float* dst, uint32_t src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst), "r"(src), "r"(bytes) : "memory");
}

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(320, 1)
    span_dkv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const __grid_constant__ CUtensorMap tdo, const __grid_constant__ CUtensorMap tdk, const __grid_constant__ CUtensorMap tdv,
                    const SpanBwdParams p) {
  using C = SpanDkvCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sK = smem;
  uint8_t* sV = sK + C::KV_TILE;
  uint8_t* sQ = sV + C::KV_TILE;                    // [STAGES][Q, dO]
  uint8_t* sRow = sQ + C::STAGES * 2 * C::Q_TILE;   // [STAGES][lse2 64 | delta 64 | lo 64 | hi 64]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sRow + C::STAGES * 1024);
  uint64_t *kv_full = bars, *full = bars + 1, *empty = full + C::STAGES, *st_full = empty + C::STAGES, *ready = st_full + 2, *all_done = ready + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(all_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  // with a bias each head reaches its own tiles; what many heads share a key head, those from the last slot on have their union
  constexpr int SLOTS = BIAS ? 64 : 1;
  __shared__ int s_first[SLOTS], s_last[SLOTS];

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  int kv_tile, unit;
  const int parts = p.parts, rank = blockIdx.x % parts;
  span_place<false>(p.order, blockIdx.x / parts, kv_tile, unit);      // causal: the keys that most rows see first
  const int kv0 = kv_tile * 128, hkv = unit % p.Hkv, b = unit / p.Hkv, group = p.H / p.Hkv;
  const int off = p.Sk - p.Sq, q_tiles = p.sq_pad / 64;
  const int4* range = p.range + static_cast<long long>(BIAS ? b * p.H + hkv * group : b) * q_tiles * 2;
  const int per_range = BIAS ? q_tiles * 2 : 0;          // from a head's to the next one's

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tq);
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
    prefetch_tensormap(&tdo);
    mbar_init(smem_u32(kv_full), 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 1);
    }
    for (int w = 0; w < 2; ++w) {
      mbar_init(smem_u32(&st_full[w]), 1);
      mbar_init(smem_u32(&ready[w]), 256);
    }
    mbar_init(smem_u32(all_done), 1);
    *abort_flag = 0;
    for (int i = 0; i < SLOTS; ++i) {
      s_first[i] = 0x7fffffff;
      s_last[i] = -1;
    }
    fence_barrier_init();
  }
  if (warp == 9) {
    tmem_alloc(smem_u32(tmem_ptr), 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_ptr;
  // query tiles from the first to the last that reaches these keys (what lies between and does not is masked)
  const int lists = BIAS ? group : 1;
  for (int i = threadIdx.x; i < q_tiles * lists; i += 320) {
    const int g = i / q_tiles, tile = i - g * q_tiles;
    const int4 r = span_range_join(range[2 * i], range[2 * i + 1]);
    if (r.x < kv0 + 128 && r.y > kv0) {
      atomicMin(&s_first[min(g, SLOTS - 1)], tile);
      atomicMax(&s_last[min(g, SLOTS - 1)], tile);
    }
  }
  __syncthreads();
  // the sweep's tiles in turn: query tiles of the first head that has any, then of the next
  struct Place {
    int g, tile, last;
  };
  auto seek = [&](Place& c) {
    while (c.g < group && s_last[min(c.g, SLOTS - 1)] < 0) ++c.g;
    c.tile = c.g < group ? s_first[min(c.g, SLOTS - 1)] : 0;
    c.last = c.g < group ? s_last[min(c.g, SLOTS - 1)] : 0x7fffffff;
  };
  auto skip = [&](Place& c, int tiles) {
    c.tile += tiles;
    while (c.tile > c.last) {
      const int over = c.tile - c.last - 1;
      ++c.g;
      seek(c);
      c.tile += over;
    }
  };
  auto next = [&](Place& c) { skip(c, parts); };
  int n = 0;
  if (SLOTS > 1) {
    for (int g = 0; g < group; ++g) n += max(0, s_last[min(g, SLOTS - 1)] + 1 - s_first[min(g, SLOTS - 1)]);
  } else if (s_last[0] >= 0) {
    n = (s_last[0] + 1 - s_first[0]) * group;
  }
  Place start = {0, 0, 0};
  if (n > 0) {
    seek(start);
    skip(start, rank);
  }
  n = (n - rank + parts - 1) / parts;             // of this CTA: every parts-th one

  if (warp == 8) {
    // ------------------------------ TMA producer ------------------------------
    if (lane == 0 && n > 0) {
      mbar_arrive_expect_tx(smem_u32(kv_full), 2 * C::KV_TILE);
#pragma unroll
      for (int s = 0; s < C::SUB; ++s) {
        tma_load_4d(smem_u32(sK + s * C::KV_SUB), &tk, smem_u32(kv_full), s * 64, kv0, hkv, b);
        tma_load_4d(smem_u32(sV + s * C::KV_SUB), &tv, smem_u32(kv_full), s * 64, kv0, hkv, b);
      }
      bool ok = true;
      int st = 0;
      uint32_t ph = 0;
      Place at = start;
      for (int it = 0; it < n; ++it, next(at)) {
        ok = mbar_wait(smem_u32(&empty[st]), ph ^ 1, abort_flag, p.status, RB_ERR_TIMEOUT_EMPTY);
        if (!ok) break;
        const int h = hkv * group + at.g, tile = at.tile;
        const uint32_t bar = smem_u32(&full[st]), dst = smem_u32(sQ + st * 2 * C::Q_TILE), rows = smem_u32(sRow + st * 1024);
        mbar_arrive_expect_tx(bar, 2 * C::Q_TILE + 1024);
        const long long bh = (static_cast<long long>(b) * p.H + h) * p.sq_pad + tile * 64, bb = static_cast<long long>(b) * p.sq_pad + tile * 64;
        bulk_load_1d(rows, p.row_lse2 + bh, 256, bar);
        bulk_load_1d(rows + 256, p.row_delta + bh, 256, bar);
        bulk_load_1d(rows + 512, p.row_lo + bb, 256, bar);
        bulk_load_1d(rows + 768, p.row_hi + bb, 256, bar);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s) {
          tma_load_4d(dst + s * C::Q_SUB, &tq, bar, s * 64, tile * 64, h, b);
          tma_load_4d(dst + C::Q_TILE + s * C::Q_SUB, &tdo, bar, s * 64, tile * 64, h, b);
        }
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
      }
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(10000);
    }
  } else if (warp == 9) {
    // ------------------------------ MMA issuer --------------------------------
    if (n > 0) {
      constexpr int F = UmmaFormat<T>::value;
      constexpr uint32_t idesc_st = make_idesc(F, 0, 0, 128, 64), idesc_acc = make_idesc(F, 0, 1, 128, HD);
      bool ok = mbar_wait(smem_u32(kv_full), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      int st_in = 0, st_out = 0;
      uint32_t ph_in = 0;
      auto issue = [&](int it) {        // S^T and dP^T of tile `it`, the next stage
        ok = mbar_wait(smem_u32(&full[st_in]), ph_in, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
        if (!ok) return;
        tc_fence_after();
        const uint32_t q = smem_u32(sQ + st_in * 2 * C::Q_TILE);
        const uint64_t kd = make_smem_desc_sw128(smem_u32(sK), 16, 1024), vd = make_smem_desc_sw128(smem_u32(sV), 16, 1024);
        const uint64_t qd = make_smem_desc_sw128(q, 16, 1024), dod = make_smem_desc_sw128(q + C::Q_TILE, 16, 1024);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s) {
          umma_f16_w4<2, 2>(tmem_base + C::ST_COL + (it & 1) * 64, kd + s * (C::KV_SUB >> 4), qd + s * (C::Q_SUB >> 4), idesc_st, s != 0);
          umma_f16_w4<2, 2>(tmem_base + C::DP_COL + (it & 1) * 64, vd + s * (C::KV_SUB >> 4), dod + s * (C::Q_SUB >> 4), idesc_st, s != 0);
        }
        umma_commit_w(smem_u32(&st_full[it & 1]));
        if (++st_in == C::STAGES) { st_in = 0; ph_in ^= 1; }
      };
      if (ok) issue(0);
      for (int it = 0; it < n && ok; ++it) {
        if (it + 1 < n) issue(it + 1);
        if (ok) ok = mbar_wait(smem_u32(&ready[it & 1]), (it >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_FLAG);
        if (!ok) break;
        tc_fence_after();
        const uint32_t q = smem_u32(sQ + st_out * 2 * C::Q_TILE), pt = tmem_base + C::ST_COL + (it & 1) * 64;
        // 64 rows are four steps of 16: rows [32 h, 32 h + 32) lie in columns 32 h + {0 .. 15} (P^T) and 32 h + {16 .. 31} (dS^T)
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          umma_f16_ts_w(tmem_base + C::DV_COL, pt + (k >> 1) * 32 + (k & 1) * 8, make_smem_desc_sw128(q + C::Q_TILE + k * 2048, C::Q_SUB, 1024), idesc_acc,
                        (it | k) != 0);
          umma_f16_ts_w(tmem_base + C::DK_COL, pt + 16 + (k >> 1) * 32 + (k & 1) * 8, make_smem_desc_sw128(q + k * 2048, C::Q_SUB, 1024), idesc_acc,
                        (it | k) != 0);
        }
        umma_commit_w(smem_u32(&empty[st_out]));
        if (++st_out == C::STAGES) st_out = 0;
      }
      if (ok) umma_commit_w(smem_u32(all_done));
    }
  } else {
    // ------------------------------ softmax warps ------------------------------
    const int t = threadIdx.x & 127, half = warp >> 2;          // key within the tile == TMEM lane; which 32 rows
    const int kv = kv0 + t;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    bool ok = true;
    int st = 0;
    Place at = start;
    int4 here = make_int4(0, 0, 0, 0);            // of the tile: asked for one tile ahead
    float slope_here = 0.f;
    auto ask = [&]() {
      here = range[at.g * per_range + 2 * at.tile + half];
      if (BIAS) slope_here = __ldg(p.c.slopes + hkv * group + at.g);
    };
    if (n > 0) ask();
    for (int it = 0; it < n; ++it) {
      const int tile = at.tile;
      const int4 r = here;
      const float slope2 = slope_here * kLog2e;
      if (it + 1 < n) {
        next(at);
        ask();
      }
      ok = mbar_wait(smem_u32(&st_full[it & 1]), (it >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      // the products have read this stage, so its rows' numbers are there; the stage is free only after this tile's last products
      const uint8_t* rows = sRow + st * 1024 + half * 128;
      if (++st == C::STAGES) st = 0;
      const float4 *lse4 = reinterpret_cast<const float4*>(rows), *delta4 = reinterpret_cast<const float4*>(rows + 256);
      const int4 *lo4 = reinterpret_cast<const int4*>(rows + 512), *hi4 = reinterpret_cast<const int4*>(rows + 768);
      // the warp's 32 keys and these 32 rows: nothing seen, or all
      const int key0 = kv0 + (warp & 3) * 32;
      const bool none = key0 + 32 <= r.x || key0 >= r.y, part = !none && (key0 < r.z || key0 + 32 > r.w);
      const int first = tile * 64 + off;                        // place of the tile's first row among the keys
      const int side = !BIAS ? 1 : p.c.causal || first >= kv0 + 127 ? 1 : first + 63 <= kv0 ? -1 : 0;
      const uint32_t st_addr = lane_addr + C::ST_COL + (it & 1) * 64 + half * 32;
      uint32_t packed[16];
      if (none) {
#pragma unroll
        for (int k = 0; k < 16; ++k) packed[k] = 0;
        tmem_st_32x32b_x16(st_addr, packed);
        tmem_st_32x32b_x16(st_addr + 16, packed);
      } else {
        uint32_t s[32], dp[32], slip[32];
        tmem_ld_32x32b_x32(st_addr, s);
        tmem_ld_32x32b_x32(lane_addr + C::DP_COL + (it & 1) * 64 + half * 32, dp);
        tmem_ld_wait();
        uint32_t seen = 0xffffffffu;
        if (part) {
          seen = 0;
#pragma unroll
          for (int i4 = 0; i4 < 8; ++i4) {
            const int4 lo = lo4[i4], hi = hi4[i4];
            seen |= (kv >= lo.x && kv < hi.x ? 1u : 0u) << (i4 * 4) | (kv >= lo.y && kv < hi.y ? 2u : 0u) << (i4 * 4) |
                    (kv >= lo.z && kv < hi.z ? 4u : 0u) << (i4 * 4) | (kv >= lo.w && kv < hi.w ? 8u : 0u) << (i4 * 4);
          }
          span_mask32(s, seen, 0);         // what unseen keys hold decides nothing
        }
        const float away = (float)(first + half * 32 - kv), slope = side > 0 ? -slope2 : slope2, reach = CAP ? span_reach32(s) : 0.f;
        if (BIAS && side != 0) {
          span_score32<CAP, true>(s, p.c, SpanAdd<true, true>({slope * away, slope}, lse4), slip, reach);
        } else {
          span_score32<CAP, true>(s, p.c, SpanAdd<false, true>({0.f, 0.f}, lse4), slip, reach);
          if constexpr (BIAS) span_both_sides32<1>(s, slope2, away);
        }
#pragma unroll
        for (int k = 0; k < 32; ++k) s[k] = __float_as_uint(fast_exp2(__uint_as_float(s[k])));
        if (part) span_mask32(s, seen, 0);
        span_pack32<T>(s, packed);
        tmem_st_32x32b_x16(st_addr, packed);
#pragma unroll
        for (int k = 0; k < 32; k += 2) {
          const float4 d = delta4[k >> 2];
          uint64_t w = pair_at(s, k);
          if (CAP) w = mul_f32x2(w, pair_at(slip, k));
          set_pair(s, k, mul_f32x2(w, add_f32x2(pair_at(dp, k), k & 2 ? f32x2(d.z, d.w) : f32x2(d.x, d.y))));
        }
        if (part) span_mask32(s, seen, 0);
        span_pack32<T>(s, packed);
        tmem_st_32x32b_x16(st_addr + 16, packed);
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&ready[it & 1]));
    }
    if (ok && n > 0) {
      ok = mbar_wait(smem_u32(all_done), 0, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (parts > 1) {
      // warps 0-3 take dV, warps 4-7 dK: sums of this part, in chunks [128 keys x 32 columns] that take the place of all that was there
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t r[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(lane_addr + (half == 0 ? C::DV_COL : C::DK_COL) + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
        uint8_t* to = smem + (half * (HD / 32) + c) * 16384 + t * 128;
#pragma unroll
        for (int k = 0; k < 8; ++k) *reinterpret_cast<uint4*>(to + ((k ^ (t & 7)) << 4)) = make_uint4(r[4 * k], r[4 * k + 1], r[4 * k + 2], r[4 * k + 3]);
      }
    } else if (ok) {
      // warps 0-3 take dV, warps 4-7 dK: through shared memory, in the place of V and K, from there in whole rows
      uint8_t* stage = (half == 0 ? sV : sK) + t * 128;
      const float f = half == 0 ? 1.f : p.grad_scale;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        uint32_t r[32];
        if (n > 0) {
          tmem_ld_32x32b_x32(lane_addr + (half == 0 ? C::DV_COL : C::DK_COL) + c * 32, r);
          tmem_ld_wait();
        } else {                                     // no row sees these keys
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const int d = c * 32 + g * 8;
          uint32_t w[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) w[k] = pack2<T>(__uint_as_float(r[g * 8 + 2 * k]) * f, __uint_as_float(r[g * 8 + 2 * k + 1]) * f);
          *reinterpret_cast<uint4*>(stage + (d >> 6) * C::KV_SUB + ((((d >> 3) & 7) ^ (t & 7)) << 4)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
      }
    }
    fence_proxy_async_smem();
    asm volatile("bar.sync %0, 128;" ::"r"(1 + half) : "memory");          // these four warps, also where a wait ran out
    if (t == 0 && ok && parts > 1) {
      float* to = p.sums + (((static_cast<long long>(rank) * p.order.units + unit) * p.order.tiles + kv_tile) * 2 + half) * (HD * 128);
#pragma unroll
      for (int c = 0; c < HD / 32; ++c) bulk_store_1d(to + c * 4096, smem_u32(smem) + (half * (HD / 32) + c) * 16384, 16384);
      tma_store_commit();
      tma_store_wait_read<0>();
    } else if (t == 0 && ok) {
#pragma unroll
      for (int s = 0; s < C::SUB; ++s)
        if (s * 64 < p.D) tma_store_4d(half == 0 ? &tdv : &tdk, smem_u32((half == 0 ? sV : sK) + s * C::KV_SUB), s * 64, kv0, hkv, b);
      tma_store_commit();
      tma_store_wait_read<0>();
    }
  }

  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem_base, 512);
  }
}

// Adds up the parts of dK and dV, in their order: eight numbers a thread
template <typename T, int HD>
__global__ void __launch_bounds__(256) span_dkv_join_kernel(const SpanBwdParams p) {
  const long long tiles = static_cast<long long>(p.order.tiles) * p.order.units, i = blockIdx.x * 256ll + threadIdx.x;
  const int piece = i & 3, key = i >> 2 & 127, c = (i >> 9) % (HD / 16);
  const long long tile = i / (32 * HD);
  if (tile >= tiles) return;
  const int unit = static_cast<int>(tile / p.order.tiles), kv = static_cast<int>(tile % p.order.tiles) * 128 + key, d = (c & (HD / 32 - 1)) * 32 + piece * 8;
  if (kv >= p.Sk || d >= p.D) return;
  const float* at = p.sums + (tile * (HD / 16) + c) * 4096 + key * 32;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f), y = x;
  for (int r = 0; r < p.parts; ++r, at += tiles * (HD * 256)) {
    const float4 g = *reinterpret_cast<const float4*>(at + (((2 * piece) ^ (key & 7)) << 2)), e = *reinterpret_cast<const float4*>(at + (((2 * piece + 1) ^ (key & 7)) << 2));
    x.x += g.x; x.y += g.y; x.z += g.z; x.w += g.w;
    y.x += e.x; y.y += e.y; y.z += e.z; y.w += e.w;
  }
  const bool is_dk = c >= HD / 32;
  const float f = is_dk ? p.grad_scale : 1.f;
  T* to = reinterpret_cast<T*>(is_dk ? p.dk : p.dv) + unit / p.Hkv * p.dkvs[0] + kv * p.dkvs[1] + unit % p.Hkv * p.dkvs[2] + d;
  *reinterpret_cast<uint4*>(to) = make_uint4(pack2<T>(x.x * f, x.y * f), pack2<T>(x.z * f, x.w * f), pack2<T>(y.x * f, y.y * f), pack2<T>(y.z * f, y.w * f));
}

struct SpanBwdArrays {
  const void *q, *k, *v, *o, *dout, *dq, *dk, *dv;        // o [B, Sq, H, D] contiguous
  const long long *qs, *ks, *vs, *dos, *dqs, *dkvs;
};
// Tensor maps: rows of queries, gradients and results in boxes of 64 and 128 rows, keys and values too
struct SpanBwdMaps {
  CUtensorMap q64, q128, do64, do128, o128, dq128, k64, k128, v64, v128, dk128, dv128;
};

template <typename T, int HD, bool CAP, bool BIAS>
int launch_span_bwd(const SpanBwdMaps& m, SpanBwdParams p, cudaStream_t st) {
  auto dq = span_dq_kernel<T, HD, CAP, BIAS>;
  auto dkv = span_dkv_kernel<T, HD, CAP, BIAS>;
  cudaError_t e = cudaFuncSetAttribute(dq, cudaFuncAttributeMaxDynamicSharedMemorySize, SpanDqCfg<HD>::SMEM_BYTES);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(dkv, cudaFuncAttributeMaxDynamicSharedMemorySize, SpanDkvCfg<HD>::SMEM_BYTES);
  if (e != cudaSuccess) return 2000 + (int)e;
  const long long q_tiles = (p.Sq + 127) / 128, kv_tiles = (p.Sk + 127) / 128;
  if (q_tiles * p.H * p.B > 0x7fffffffll || kv_tiles * p.Hkv * p.B * (p.parts > HD / 8 ? p.parts : HD / 8) > 0x7fffffffll) return 20;
  p.order = {(int)q_tiles, p.H * p.B, rbh::span_group(static_cast<long long>(p.H) * p.B, 4ll * p.Sk * p.D * p.Hkv / p.H)};
  dq<<<(unsigned)(q_tiles * p.H * p.B), 320, SpanDqCfg<HD>::SMEM_BYTES, st>>>(m.q128, m.do128, m.o128, m.k64, m.v64, m.dq128, p);
  p.order = {(int)kv_tiles, p.Hkv * p.B, rbh::span_group(static_cast<long long>(p.Hkv) * p.B, 4ll * p.Sq * p.D * (p.H / p.Hkv))};
  dkv<<<(unsigned)(kv_tiles * p.Hkv * p.B * p.parts), 320, SpanDkvCfg<HD>::SMEM_BYTES, st>>>(m.q64, m.k128, m.v128, m.do64, m.dk128, m.dv128, p);
  if (p.parts > 1) span_dkv_join_kernel<T, HD><<<(unsigned)(kv_tiles * p.Hkv * p.B * (HD / 8)), 256, 0, st>>>(p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 3000 + (int)e;
}

template <typename T>
int span_bwd(int dtype, const SpanBwdArrays& a, const SpanBwdParams& p, bool cap, cudaStream_t st) {
  SpanBwdMaps m;
  const long long os[3] = {static_cast<long long>(p.Sq) * p.H * p.D, static_cast<long long>(p.H) * p.D, p.D};
  int rc = 0;
  auto rows = [&](CUtensorMap* map, const void* base, const long long* s, int box) {
    if (!rc) rc = rbh::span_map(map, dtype, base, s, p.B, p.Sq, p.H, p.D, box);
  };
  auto keys = [&](CUtensorMap* map, const void* base, const long long* s, int box) {
    if (!rc) rc = rbh::span_map(map, dtype, base, s, p.B, p.Sk, p.Hkv, p.D, box);
  };
  rows(&m.q64, a.q, a.qs, 64);
  rows(&m.q128, a.q, a.qs, 128);
  rows(&m.do64, a.dout, a.dos, 64);
  rows(&m.do128, a.dout, a.dos, 128);
  rows(&m.o128, a.o, os, 128);
  rows(&m.dq128, a.dq, a.dqs, 128);
  keys(&m.k64, a.k, a.ks, 64);
  keys(&m.k128, a.k, a.ks, 128);
  keys(&m.v64, a.v, a.vs, 64);
  keys(&m.v128, a.v, a.vs, 128);
  keys(&m.dk128, a.dk, a.dkvs, 128);
  keys(&m.dv128, a.dv, a.dkvs, 128);
  if (rc) return 1000 + rc;
  const bool bias = p.c.slopes != nullptr;
#define RB_SPAN(HD_)                                                                                               \
  (cap ? bias ? launch_span_bwd<T, HD_, true, true>(m, p, st) : launch_span_bwd<T, HD_, true, false>(m, p, st)     \
       : bias ? launch_span_bwd<T, HD_, false, true>(m, p, st) : launch_span_bwd<T, HD_, false, false>(m, p, st))
  return p.D <= 64 ? RB_SPAN(64) : RB_SPAN(128);
#undef RB_SPAN
}

}  // namespace rb

extern "C" {

// CTAs that share a tile of 128 keys of a key head in rb_span_bwd, each with every parts-th tile of rows, 8 of them at least: as many as make two CTAs per SM,
// twice that where heads `differ` in how far they reach (slopes and a cap or norms).  Whole backward pass with 1 and with these parts, heads of 128: 4096 tokens, 8
// heads over 1: 654 and 187 us (8 parts); 2048 tokens, 8 heads: 87.1 and 85.6 (2); 8192 tokens, 16 heads over 4, capped and biased: 940 and 750 (2), where
// the CTAs of the last key head would be at work alone.  Further parts cost 128 KB of sums a CTA: 4 x 2048 tokens, 16 heads over 4, whose 256 CTAs differ by
// their place only: 326 with 1 part, 360 with 2.
int rb_span_bwd_parts(int B, int H, int Hkv, int Sq, int Sk, int differ) {
  if (B <= 0 || Hkv <= 0 || H <= 0 || Sq <= 0 || Sk <= 0) return 1;
  const long long tiles = static_cast<long long>(B) * Hkv * ((Sk + 127ll) / 128), each = static_cast<long long>(H) / Hkv * ((Sq + 63ll) / 64);
  long long parts = (differ ? 4ll : 2ll) * rbh::sm_count() / tiles;
  if (parts > each / 8) parts = each / 8;
  return parts < 1 ? 1 : parts > 8 ? 8 : static_cast<int>(parts);
}

// Gradients of rb_span_fwd.  q, k, v, dout: 16-bit views as there; o contiguous, lse2 and norms (or null) from the forward call with the same arguments.  dq [B, Sq, H, D]; dk and
// dv [B, Sk, Hkv, D] of the same strides: views of 16-byte aligned rows.  scratch: 16-byte aligned, B pad (8 H + 8) bytes and another B pad / 2, with slopes
// B H pad / 2, with pad = Sq rounded up to a multiple of 64; nothing in it has to be set.  sums: with
// several parts fp32 [parts, B, Hkv, Sk rounded up to 128, 2, 64 or 128 (D)], 16-byte aligned.
int rb_span_bwd(int dtype, const void* q, const void* k, const void* v, const long long* qs, const long long* ks, const long long* vs, const int* spans,
                long long span_batch, const float* slopes, const float* norms, const void* o, const float* lse2, const void* dout, const long long* dos, void* scratch, float* sums,
                void* dq, void* dk, void* dv, const long long* dqs, const long long* dkvs, int B, int H, int Hkv, int Sq, int Sk, int D, int parts, int causal,
                float scale, float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0 || Sq <= 0) return 0;
  if (Sk <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 128 || D % 8 || Sq > 0x7fffffff - 128) return 20;
  if (parts < 1 || (parts > 1 && !sums)) return 20;
  if ((Sq + 63) / 64 * (static_cast<long long>(H) / Hkv) > 0x3fffffff) return 20;              // ranges of a key head's rows
  SpanBwdParams p{};
  p.B = B; p.H = H; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.D = D;
  p.c = rbh::span_scores(scale, cap);
  p.c.slopes = slopes;
  p.c.norms = norms;
  p.c.spans = reinterpret_cast<const int2*>(spans);
  p.c.span_batch = span_batch;
  p.c.causal = causal;
  p.grad_scale = cap > 0.f ? -scale : scale;
  p.lse2 = lse2;
  p.parts = parts; p.sums = sums; p.dk = dk; p.dv = dv;
  for (int i = 0; i < 3; ++i) p.dkvs[i] = dkvs[i];
  p.sq_pad = (Sq + 63) / 64 * 64;
  const long long rows = static_cast<long long>(B) * p.sq_pad;
  p.row_lse2 = reinterpret_cast<float*>(scratch);
  p.row_delta = p.row_lse2 + rows * H;
  p.row_lo = reinterpret_cast<int*>(p.row_delta + rows * H);
  p.row_hi = p.row_lo + rows;
  p.range = reinterpret_cast<int4*>(p.row_hi + rows);
  const SpanBwdArrays a = {q, k, v, o, dout, dq, dk, dv, qs, ks, vs, dos, dqs, dkvs};
  p.status = rbh::device_status_word();
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == rbh::DT_BF16) return span_bwd<__nv_bfloat16>(dtype, a, p, cap > 0.f, st);
  if (dtype == rbh::DT_F16) return span_bwd<__half>(dtype, a, p, cap > 0.f, st);
  return 20;
}
}
