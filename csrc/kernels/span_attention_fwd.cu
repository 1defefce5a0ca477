// Span attention forward for sm_100a (tcgen05 + TMEM + TMA): softmax(cap tanh(scale q.k / cap) - slope |distance|) V over the keys lo <= j < hi of
// each row, 16-bit, heads of 8 to 128 numbers.
//
// A CTA owns two tiles of 128 query rows of one head, each with a warpgroup of its own (a thread owns a row: maximum and sum never leave it) and its
// own S and O in tensor memory.  Tiles of 64 keys and of 64 values take turns in one ring of shared memory and serve both query tiles, from the last
// to the first: the nearest keys, whose scores the distance lowers least, come first.  S of a query tile has two buffers, so that a warpgroup finds its
// next tile's S there when it has done one: with one buffer (of 128 keys) it waited 1500 of 4300 cycles a tile for the products.  P (16-bit) lies over the
// first half of its S, from where P V reads it as left operand; the S that follows in that buffer comes after that product in the issue order.
//
// Keys that no row of a tile reaches are not read: each query tile goes over the tiles from its least lo to its largest hi.  Few rows over many
// keys would leave most SMs idle, so such calls cut the tiles of keys into `splits` parts, whose results (fp32, with their log-sum-exp) a second
// kernel joins.
//
// Bound by the softmax warps: of the 2300 cycles that a pair of 128 x 64 tiles takes, products fill 1280 (S 384 and P V 256 a tile) and the
// exponentials 1024.  A CTA's beginning and end take 8000 cycles more (one CTA fills an SM).  Heads of 128: 2 x 4096 rows, 32 heads over 8, biased:
// 308 us, 893 TFLOP/s (4 operations a visible pair and number), 257 us with far tiles left out; 512 rows over 8704 keys, 32 heads over 8, capped:
// 93 us, 761 TFLOP/s; 8 x 2048 rows in 4 documents each, 16 heads, capped: 165 us, 306 TFLOP/s of visible pairs.
#include "span_join.cuh"
#include "span_scores.cuh"

#include <type_traits>

namespace rb {

struct SpanFwdParams {
  int B, H, Hkv, Sq, Sk, D;
  int splits;
  SpanOrder order;   // of tiles of 256 rows and heads x parts
  SpanScores c;
  void* o;           // [B, Sq, H, D]
  float* lse2;       // [B, H, Sq] log-sum-exp in log2 units, -inf: the row sees no key (or null)
  float* part_o;     // [splits, B, Sq, H, D] (splits > 1)
  float* part_lse2;  // [splits, B, H, Sq]
  int* status;
};

template <int HD>
struct SpanFwdCfg {
  static constexpr int BN = 64;                       // keys of a tile
  static constexpr int SUB = HD / 64;                 // 64-column sub-tiles of a row
  static constexpr int Q_SUB = 128 * 128, Q_TILE = SUB * Q_SUB;       // 128 rows, 16-bit
  static constexpr int KV_SUB = BN * 128, KV_TILE = SUB * KV_SUB;
  static constexpr int STAGES = 5;                    // pairs of K and V tiles in flight
  static constexpr int SMEM_BYTES = 2 * Q_TILE + STAGES * 2 * KV_TILE + 1024 + 256;
  static constexpr int S_COL = 0, O_COL = 256;        // of query tile x: + x * 128; second buffer of S: + 64
  // Two softmax warpgroups and one of which three warps work.  They share out the registers that the launch gives the block.
  static constexpr int THREADS = 384, SOFTMAX_REGS = 224, OTHER_REGS = 56, LAUNCH_REGS = (2 * SOFTMAX_REGS + OTHER_REGS) / 3;
};

template <typename T, int HD, bool CAP, bool BIAS>
__global__ void __launch_bounds__(SpanFwdCfg<HD>::THREADS, 1)
    span_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                    const __grid_constant__ CUtensorMap to, const SpanFwdParams p) {
  using C = SpanFwdCfg<HD>;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  uint8_t* sQ = smem;                                  // [2][Q_TILE], at the end O
  uint8_t* sKV = sQ + 2 * C::Q_TILE;                   // [STAGES][2][KV_TILE]: {K0, K1}, {V0, K2}, {V1, K3}, ...
  uint64_t* bars = reinterpret_cast<uint64_t*>(sKV + C::STAGES * 2 * C::KV_TILE);
  // s_full, p_ready: [query tile][buffer]; o_done: [query tile], after the last product with V; o_last: [query tile], after the one before
  uint64_t *q_full = bars, *full = bars + 1, *empty = full + C::STAGES, *s_full = empty + C::STAGES, *p_ready = s_full + 4, *o_done = p_ready + 4, *o_last = o_done + 2;
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(o_last + 2);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_ptr + 1);
  __shared__ int4 s_range[8];

  const int warp = uniform_warp_idx(), lane = threadIdx.x & 31;
  int q_tile, unit;
  span_place<true>(p.order, blockIdx.x, q_tile, unit);
  const int sp = unit % p.splits, h = unit / p.splits % p.H, b = unit / p.splits / p.H;
  const int hkv = h / (p.H / p.Hkv);
  const int q0 = q_tile * 256, off = p.Sk - p.Sq;

  if (threadIdx.x == 0) {
    prefetch_tensormap(&tq);
    prefetch_tensormap(&tk);
    prefetch_tensormap(&tv);
    prefetch_tensormap(&to);
    mbar_init(smem_u32(q_full), 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(smem_u32(&full[s]), 1);
      mbar_init(smem_u32(&empty[s]), 2);        // both query tiles' products
    }
    for (int i = 0; i < 4; ++i) {
      mbar_init(smem_u32(&s_full[i]), 1);
      mbar_init(smem_u32(&p_ready[i]), 128);
    }
    for (int x = 0; x < 4; ++x) mbar_init(smem_u32(&o_done[x]), 1);      // o_last too
    *abort_flag = 0;
    fence_barrier_init();
  }
  int2 span = make_int2(0, 0);
  if (warp < 8) {
    const int row = q0 + threadIdx.x;
    const bool live = row < p.Sq;
    if (live) span = span_of(p.c, b, row, p.Sq, p.Sk);
    const int4 r = span_range_warp(span, BIAS ? span_near(span, row + off, span_head_reach<CAP>(p.c, b, h, hkv, p.H, p.Hkv)) : span, live);
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
    first[x] = r.x < r.y ? r.x / C::BN : 0;
    last[x] = r.x < r.y ? (r.y + C::BN - 1) / C::BN : 0;
    lo_all[x] = r.z;
    hi_all[x] = r.w;
  }
  int j0, j1;
  {
    const bool a = first[0] < last[0], c = first[1] < last[1];
    j0 = a && c ? min(first[0], first[1]) : a ? first[0] : first[1];
    j1 = max(last[0], last[1]);
    const int per = (j1 - j0 + p.splits - 1) / p.splits;
    const int from = j0 + sp * per, to_ = min(j1, from + per);
#pragma unroll
    for (int x = 0; x < 2; ++x) {
      first[x] = max(first[x], from);
      last[x] = max(first[x], min(last[x], to_));
    }
    j0 = from;
    j1 = max(from, to_);
  }
  const int n = j1 - j0;

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(C::OTHER_REGS));
    if (warp == 8 && lane == 0 && n > 0) {
      // ------------------------------ TMA producer ------------------------------
      const bool two = q0 + 128 < p.Sq;
      mbar_arrive_expect_tx(smem_u32(q_full), (two ? 2 : 1) * C::Q_TILE);
#pragma unroll
      for (int s = 0; s < C::SUB; ++s) {
        tma_load_4d(smem_u32(sQ + s * C::Q_SUB), &tq, smem_u32(q_full), s * 64, q0, h, b);
        if (two) tma_load_4d(smem_u32(sQ + C::Q_TILE + s * C::Q_SUB), &tq, smem_u32(q_full), s * 64, q0 + 128, h, b);
      }
      bool ok = true;
      int st = 0;
      uint32_t ph = 0;
      // two tiles (b: one of keys behind the last: none)
      auto bring = [&](const CUtensorMap* map_a, int a, int b_) {
        ok = mbar_wait(smem_u32(&empty[st]), ph ^ 1, abort_flag, p.status, RB_ERR_TIMEOUT_EMPTY);
        if (!ok) return;
        const uint32_t bar = smem_u32(&full[st]), dst = smem_u32(sKV + st * 2 * C::KV_TILE);
        mbar_arrive_expect_tx(bar, (b_ >= j0 ? 2 : 1) * C::KV_TILE);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s) {
          tma_load_4d(dst + s * C::KV_SUB, map_a, bar, s * 64, a * C::BN, hkv, b);
          if (b_ >= j0) tma_load_4d(dst + C::KV_TILE + s * C::KV_SUB, &tk, bar, s * 64, b_ * C::BN, hkv, b);
        }
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
      };
      bring(&tk, j1 - 1, j1 - 2);
      for (int j = j1 - 1; j >= j0 && ok; --j) bring(&tv, j, j - 2);
      if (!ok)
        for (int i = 0; i < 64; ++i) __nanosleep(10000);      // copies in flight land before the CTA's memory goes
    } else if ((warp == 9 || warp == 10) && n > 0) {
      // ------------------------------ MMA issuers -------------------------------
      // One warp per query tile: what a warp does between its products (waits and commits, some 100 cycles each) takes as long as they do.
      const int x = warp - 9;
      const int begin = x ? first[1] : first[0], end = x ? last[1] : last[0];
      constexpr uint32_t idesc_s = make_idesc(UmmaFormat<T>::value, 0, 0, 128, C::BN);
      constexpr uint32_t idesc_o = make_idesc(UmmaFormat<T>::value, 0, 1, 128, HD);
      const uint32_t s_tmem = tmem_base + C::S_COL + x * 128, o_tmem = tmem_base + C::O_COL + x * 128;
      const uint64_t qd = make_smem_desc_sw128(smem_u32(sQ + x * C::Q_TILE), 16, 1024);
      int st = 0;
      uint32_t ph = 0;
      auto issue_s = [&](int j, int at) {                     // K(j) in half `at` of the stage
        if (j < begin || j >= end) return;
        const int buf = (end - 1 - j) & 1;
        const uint64_t kd = make_smem_desc_sw128(smem_u32(sKV + (2 * st + at) * C::KV_TILE), 16, 1024);
#pragma unroll
        for (int s = 0; s < C::SUB; ++s)
          umma_f16_w4<2, 2>(s_tmem + buf * 64, qd + s * (C::Q_SUB >> 4), kd + s * (C::KV_SUB >> 4), idesc_s, s != 0);
        umma_commit_w(smem_u32(&s_full[2 * x + buf]));
      };
      auto leave = [&]() {
        umma_commit_w(smem_u32(&empty[st]));
        if (++st == C::STAGES) { st = 0; ph ^= 1; }
      };
      bool ok = mbar_wait(smem_u32(q_full), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      if (ok) ok = mbar_wait(smem_u32(&full[0]), 0, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
      if (ok) {
        tc_fence_after();
        issue_s(j1 - 1, 0);
        issue_s(j1 - 2, 1);
        leave();
      }
      for (int j = j1 - 1; j >= j0 && ok; --j) {
        ok = mbar_wait(smem_u32(&full[st]), ph, abort_flag, p.status, RB_ERR_TIMEOUT_FULL);
        if (!ok) break;
        if (j >= begin && j < end) {
          const int i = end - 1 - j, buf = i & 1;
          ok = mbar_wait(smem_u32(&p_ready[2 * x + buf]), (i >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_FLAG);
          if (!ok) break;
          tc_fence_after();
          umma_f16_ts_w4<8, 128>(o_tmem, s_tmem + buf * 64, make_smem_desc_sw128(smem_u32(sKV + 2 * st * C::KV_TILE), C::KV_SUB, 1024), idesc_o, i != 0);
          if (j <= begin + 1) umma_commit_w(smem_u32(j == begin ? &o_done[x] : &o_last[x]));
        } else {
          tc_fence_after();
        }
        issue_s(j - 2, 1);
        leave();
      }
    }
  } else {
    // ------------------------------ softmax warpgroups ------------------------
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(C::SOFTMAX_REGS));
    const int x = warp >> 2, t = threadIdx.x & 127;
    const int row0 = q0 + x * 128, row = row0 + t;
    const uint32_t lane_addr = tmem_base + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t o_addr = lane_addr + C::O_COL + x * 128;
    const int begin = x ? first[1] : first[0], end = x ? last[1] : last[0];
    const int lo_max = x ? lo_all[1] : lo_all[0], hi_min = x ? hi_all[1] : hi_all[0];
    const float slope2 = BIAS ? p.c.slopes[h] * kLog2e : 0.f;
    // Weights are relative to `ref`: a row's largest score in the first tile that it sees, where two passes look for it (the weight of a key that has nearly
    // all of it is then 1, and rounds to itself).  After that `ref` follows the maximum only when that may be far away, and a tile's weights are made in
    // one pass over its scores, without their maximum.  Where the largest product says that the reference may be no good, two passes do the tile again.
    // UP: how far above its reference a weight may be.  fp16 goes up to 2^16; bf16 has the range of fp32, but what a value of 2^90 times a weight of
    // 2^30 is still has to be a number.
    constexpr float UP = UmmaFormat<T>::value == 1 ? 30.f : 15.f;
    float ref = 0.f, l = 0.f;
    bool fresh = true, ok = true;                       // fresh: the row has seen no key yet
    bool flat = false, slow = false;                    // what the last tile needed: the general tanh, the two passes
    for (int i = 0; i < end - begin; ++i) {
      const int buf = i & 1;
      ok = mbar_wait(smem_u32(&s_full[2 * x + buf]), (i >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_FULL);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      tc_fence_after();
      const uint32_t s_addr = lane_addr + C::S_COL + x * 128 + buf * 64;
      const int kv0 = (end - 1 - i) * C::BN;
      const bool masked = kv0 < lo_max || kv0 + C::BN > hi_min;
      // where all distances that count have one sign the bias is a ramp
      const int side = !BIAS ? 1 : p.c.causal || row0 + off >= kv0 + C::BN - 1 ? 1 : row0 + 127 + off <= kv0 ? -1 : 0;
      const float slope = side > 0 ? slope2 : -slope2;
      const int away = row + off - kv0;                  // distance of the tile's first key
      // chunk c of 32 scores, plus `base`, what is unseen -inf; whether it has something to see; the largest product
      float reach = 0.f;
      auto scores = [&](int c, float base, uint32_t* s) -> bool {
        uint32_t seen = 0xffffffffu;
        bool part = false;
        if (masked) {
          seen = span_bits(span.x - kv0 - c * 32, span.y - kv0 - c * 32);
          if (__all_sync(0xffffffffu, seen == 0)) return false;
          part = !__all_sync(0xffffffffu, seen == 0xffffffffu);
        }
        tmem_ld_32x32b_x32(s_addr + c * 32, s);
        tmem_ld_wait();
        if (part) span_mask32(s, seen, 0);               // what unseen keys hold decides nothing
        reach = fmaxf(reach, span_reach32(s));
        if (BIAS && side != 0) {
          span_score32<CAP, false>(s, p.c, SpanAdd<true, false>({fmaf(-slope, (float)(away - c * 32), base), slope}, nullptr), nullptr, reach);
        } else {
          span_score32<CAP, false>(s, p.c, SpanAdd<false, false>({base, 0.f}, nullptr), nullptr, reach);
          if constexpr (BIAS) span_both_sides32<-1>(s, slope2, (float)(away - c * 32));
        }
        if (part) span_mask32(s, seen, 0xff800000u);
        return true;
      };
      // weights of a chunk of scores relative to ref
      auto weights = [&](const uint32_t* s, uint32_t* packed) -> float {
        uint64_t l2[2] = {0, 0};
#pragma unroll
        for (int k = 0; k < 16; ++k) {
          const float p0 = fast_exp2(__uint_as_float(s[2 * k])), p1 = fast_exp2(__uint_as_float(s[2 * k + 1]));
          l2[k & 1] = add_f32x2(l2[k & 1], f32x2(p0, p1));
          packed[k] = pack2<T>(p0, p1);
        }
        const float2 la = f32x2_get(l2[0]), lb = f32x2_get(l2[1]);
        return (la.x + la.y) + (lb.x + lb.y);
      };
      const bool sees = span.x < min(kv0 + C::BN, span.y) && span.y > max(kv0, span.x);
      bool done = false;
      if (!slow && !__any_sync(0xffffffffu, fresh && sees)) {
        uint32_t packed[2][16];
        float sum = 0.f;
        bool quick = !masked && side != 0 && !(CAP && flat);
        if (quick) {
          const SpanTanh f(p.c, p.c.out2);
          const uint64_t k = both(p.c.scale2);
          float far[4] = {0.f, 0.f, 0.f, 0.f};
          auto score = [&](uint32_t* s, int i, auto& add) {
            far[i & 2] = fmaxf(far[i & 2], fabsf(__uint_as_float(s[i])));
            far[(i & 2) + 1] = fmaxf(far[(i & 2) + 1], fabsf(__uint_as_float(s[i + 1])));
            if constexpr (CAP) {
              const uint64_t x2 = pair_at(s, i);
              set_pair(s, i, fma_f32x2(x2, f.r(x2), add.next(i)));
            } else {
              set_pair(s, i, fma_f32x2(pair_at(s, i), k, add.next(i)));
            }
          };
          // scores LAG pairs ahead of the weights: the FMA pipe and the special-function pipe work at the same time all along
          constexpr int LAG = 4;
          uint32_t s[64];
          tmem_ld_32x32b_x32(s_addr, s);
          tmem_ld_32x32b_x32(s_addr + 32, s + 32);
          tmem_ld_wait();
          SpanAdd<BIAS, false> add({BIAS ? fmaf(-slope, (float)away, -ref) : -ref, slope}, nullptr);
#pragma unroll
          for (int g = 0; g < LAG; ++g) score(s, 2 * g, add);
          uint64_t l2[2] = {0, 0};
#pragma unroll
          for (int g = 0; g < 32; ++g) {
            // the ramp begins anew half-way
            if (BIAS && g + LAG == 16) add = SpanAdd<BIAS, false>({fmaf(-slope, (float)(away - 32), -ref), slope}, nullptr);
            const float p0 = fast_exp2(__uint_as_float(s[2 * g])), p1 = fast_exp2(__uint_as_float(s[2 * g + 1]));
            if (g + LAG < 32) score(s, 2 * (g + LAG), add);
            l2[g & 1] = add_f32x2(l2[g & 1], f32x2(p0, p1));
            packed[g >> 4][g & 15] = pack2<T>(p0, p1);
          }
          const float2 la = f32x2_get(l2[0]), lb = f32x2_get(l2[1]);
          sum = (la.x + la.y) + (lb.x + lb.y);
          reach = fmaxf(fmaxf(far[0], far[1]), fmaxf(far[2], far[3]));
          if constexpr (CAP) {
            flat = __any_sync(0xffffffffu, !(reach <= p.c.near));
            quick = !flat;
          }
        }
        if (!quick) {
          // chunk by chunk: some have nothing to see, some all, some large products
          sum = reach = 0.f;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32];
            if (scores(c, -ref, s)) {
              sum += weights(s, packed[c]);
            } else {
#pragma unroll
              for (int k = 0; k < 16; ++k) packed[c][k] = 0;
            }
          }
          if (CAP && !masked) flat = __any_sync(0xffffffffu, !(reach <= p.c.near));
        }
        // no score of the row is above this: the cap and the largest product bound it
        float most = reach * fabsf(p.c.scale2);
        if (CAP) most = fminf(most, p.c.out2);
        if (BIAS && slope2 < 0.f) most = fmaf(-slope2, (float)max(abs(away), abs(away - C::BN + 1)), most);
        done = __all_sync(0xffffffffu, most - ref <= UP);
        if (done) {
          l += sum;
          tmem_st_32x32b_x16(s_addr, packed[0]);
          tmem_st_32x32b_x16(s_addr + 16, packed[1]);
        }
      }
      if (!done) {
        float mx = -INFINITY;
        reach = 0.f;
        if constexpr (BIAS) {
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32];
            if (!scores(c, 0.f, s)) continue;
#pragma unroll
            for (int k = 0; k < 32; ++k) mx = fmaxf(mx, __uint_as_float(s[k]));
          }
        } else {
          // scores rise with the products (fall, where the scale is below zero): the score of the largest is the largest
          const uint32_t flip = p.c.scale2 < 0.f ? 0x80000000u : 0u;
#pragma unroll 1
          for (int c = 0; c < 2; ++c) {
            uint32_t s[32];
            tmem_ld_32x32b_x32(s_addr + c * 32, s);
            tmem_ld_wait();
            const uint32_t seen = masked ? span_bits(span.x - kv0 - c * 32, span.y - kv0 - c * 32) : 0xffffffffu;
#pragma unroll
            for (int k = 0; k < 32; ++k)
              if (seen >> k & 1) mx = fmaxf(mx, __uint_as_float(s[k] ^ flip));
          }
          if (mx > -INFINITY) mx = CAP ? fabsf(p.c.out2) * tanhf(fabsf(p.c.in) * mx) : fabsf(p.c.scale2) * mx;
        }
        // a maximum that goes on rising is looked for at once in the next tile
        slow = !__all_sync(0xffffffffu, fresh || mx <= ref + UP);
        const bool need = mx > ref + UP || (fresh && mx > -INFINITY);
        if (__any_sync(0xffffffffu, need)) {               // tensor memory is accessed by whole warps
          const float alpha = !need ? 1.f : fresh ? 0.f : fast_exp2(ref - mx);
          if (need) ref = mx;
          l *= alpha;
          if (i > 0) {
            // O is at rest once the last tile's product has retired: the next tile's S comes after it
            ok = i + 1 < end - begin
                     ? mbar_wait(smem_u32(&s_full[2 * x + (buf ^ 1)]), ((i + 1) >> 1) & 1, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_EMPTY)
                     : mbar_wait(smem_u32(&o_last[x]), 0, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_EMPTY);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t r[16];
              tmem_ld_32x32b_x16(o_addr + c * 16, r);
              tmem_ld_wait();
#pragma unroll
              for (int k = 0; k < 16; ++k) r[k] = __float_as_uint(__uint_as_float(r[k]) * alpha);
              tmem_st_32x32b_x16(o_addr + c * 16, r);
            }
          }
        }
        fresh = fresh && mx == -INFINITY;
        // P of chunk c goes over what chunk 0 was read from
#pragma unroll 1
        for (int c = 0; c < 2; ++c) {
          uint32_t s[32], packed[16];
          if (scores(c, -ref, s)) {
            l += weights(s, packed);
          } else {
#pragma unroll
            for (int k = 0; k < 16; ++k) packed[k] = 0;
          }
          tmem_st_32x32b_x16(s_addr + c * 16, packed);
        }
      }
      tmem_st_wait();
      tc_fence_before();
      mbar_arrive(smem_u32(&p_ready[2 * x + buf]));
    }
    const int tiles = end - begin;
    const bool staged = p.splits == 1 && tiles > 0;
    if (ok && tiles > 0) {
      ok = mbar_wait(smem_u32(&o_done[x]), 0, abort_flag, p.status, RB_ERR_TIMEOUT_TMEM_EMPTY);
      ok = __all_sync(0xffffffffu, ok);
      tc_fence_after();
    }
    if (ok) {
      const float inv = l > 0.f ? 1.0f / l : l != l ? l : 0.f;
      const long long at = ((static_cast<long long>(b) * p.Sq + row) * p.H + h) * p.D;
      const long long part = static_cast<long long>(sp) * p.B * p.H * p.Sq;
      // O through shared memory, in the place of Q, and from there to memory in whole rows: a thread's row of its own stores, 16 bytes of a line each, took
      // 6000 to 10000 cycles.  Tiles without keys (whose Q may be on its way) and the parts' sums are stored row by row.
      uint8_t* stage = sQ + x * C::Q_TILE + t * 128;
#pragma unroll 1
      for (int c = 0; c < HD / 32; ++c) {
        if (c * 32 >= p.D) break;
        uint32_t r[32];
        if (tiles > 0) {
          tmem_ld_32x32b_x32(o_addr + c * 32, r);
          tmem_ld_wait();
        } else {
#pragma unroll
          for (int k = 0; k < 32; ++k) r[k] = 0;
        }
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          float f[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) f[k] = l == 0.f ? 0.f : __uint_as_float(r[g * 8 + k]) * inv;
          const uint4 v = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
          const int d = c * 32 + g * 8;
          if (staged) {
            *reinterpret_cast<uint4*>(stage + (d >> 6) * C::Q_SUB + ((((d >> 3) & 7) ^ (t & 7)) << 4)) = v;
          } else if (row < p.Sq && d < p.D) {
            if (p.splits == 1) {
              *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + at + d) = v;
            } else {
              float4* dst = reinterpret_cast<float4*>(p.part_o + part * p.D + at + d);
              dst[0] = make_float4(f[0], f[1], f[2], f[3]);
              dst[1] = make_float4(f[4], f[5], f[6], f[7]);
            }
          }
        }
      }
      if (row < p.Sq) {
        const long long r = (static_cast<long long>(b) * p.H + h) * p.Sq + row;
        const float v = l == 0.f ? -INFINITY : ref + log2f(l);
        if (p.splits > 1) p.part_lse2[part + r] = v;
        else if (p.lse2 != nullptr) p.lse2[r] = v;
      }
    }
    if (staged) {
      fence_proxy_async_smem();
      asm volatile("bar.sync %0, 128;" ::"r"(1 + x) : "memory");      // the warpgroup, also where a wait ran out
      if (t == 0 && ok) {
#pragma unroll
        for (int s = 0; s < C::SUB; ++s)
          if (s * 64 < p.D) tma_store_4d(&to, smem_u32(sQ + x * C::Q_TILE + s * C::Q_SUB), s * 64, row0, h, b);
        tma_store_commit();
        tma_store_wait_read<0>();
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

// Largest squared length of each of 32 parts of a head's rows: heads of queries, then of keys (SpanScores::norms).  8 or 16 lanes a row, 16 bytes each.
// Bound by reading both once: 84 MB (2 x 4096 rows, 32 heads and 8 of 128) in 17.7 us, 4.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(256) span_norms_kernel(const T* q, const T* k, long long qb, long long qr, long long qh, long long kb, long long kr, long long kh,
                                                         float* norms, int H, int Hkv, int Sq, int Sk, int D) {
  __shared__ uint32_t most[8];
  // neighbouring CTAs take neighbouring heads of the same rows
  const int units = gridDim.x / 32, part = blockIdx.x / units, unit = blockIdx.x - part * units, head = unit % (H + Hkv), b = unit / (H + Hkv);
  const bool of_q = head < H;
  const int S = of_q ? Sq : Sk, per = (S + 31) / 32, begin = min(S, part * per), end = min(S, begin + per);
  const long long step = of_q ? qr : kr;
  const int lanes = D <= 64 ? 8 : 16, rows = 256 / lanes, d = (threadIdx.x % lanes) * 8;
  const T* at = (of_q ? q + b * qb + head * qh : k + b * kb + (head - H) * kh) + d;
  uint32_t mx = 0;
  for (int r0 = begin; r0 < end; r0 += rows * 4) {
    uint4 v[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int r = r0 + u * rows + threadIdx.x / lanes;
      v[u] = r < end && d < D ? __ldg(reinterpret_cast<const uint4*>(at + r * step)) : make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const uint32_t w[4] = {v[u].x, v[u].y, v[u].z, v[u].w};
      float sum = 0.f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = unpack2<T>(w[i]);
        sum = fmaf(f.x, f.x, fmaf(f.y, f.y, sum));
      }
      for (int o = lanes / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      mx = max(mx, __float_as_uint(sum));
    }
  }
  mx = __reduce_max_sync(0xffffffffu, mx);
  if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = mx;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < 8; ++w) mx = max(mx, most[w]);
    norms[static_cast<long long>(unit) * 32 + part] = __uint_as_float(mx);
  }
}

template <typename T, int HD, bool CAP, bool BIAS>
int launch_span_fwd(const CUtensorMap& tq, const CUtensorMap& tk, const CUtensorMap& tv, const CUtensorMap& to, const SpanFwdParams& p, unsigned grid,
                    cudaStream_t st) {
  using C = SpanFwdCfg<HD>;
  auto kern = span_fwd_kernel<T, HD, CAP, BIAS>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM_BYTES);
  if (e != cudaSuccess) return 2000 + (int)e;
  cudaFuncAttributes fa;
  e = cudaFuncGetAttributes(&fa, kern);
  if (e != cudaSuccess) return 2000 + (int)e;
  if (fa.numRegs < C::LAUNCH_REGS) return 21;      // the warpgroups would wait for registers that the block does not have
  kern<<<grid, C::THREADS, C::SMEM_BYTES, st>>>(tq, tk, tv, to, p);
  e = cudaGetLastError();
  return e == cudaSuccess ? 0 : 3000 + (int)e;
}

template <typename T>
int span_fwd(int dtype, const void* q, const void* k, const void* v, const long long* qs, const long long* ks, const long long* vs, SpanFwdParams p,
             bool cap, cudaStream_t st) {
  CUtensorMap tq, tk, tv, to;
  const long long os[3] = {static_cast<long long>(p.Sq) * p.H * p.D, static_cast<long long>(p.H) * p.D, p.D};
  int rc = rbh::span_map(&tq, dtype, q, qs, p.B, p.Sq, p.H, p.D, 128);
  if (!rc) rc = rbh::span_map(&tk, dtype, k, ks, p.B, p.Sk, p.Hkv, p.D, 64);
  if (!rc) rc = rbh::span_map(&tv, dtype, v, vs, p.B, p.Sk, p.Hkv, p.D, 64);
  if (!rc) rc = rbh::span_map(&to, dtype, p.o, os, p.B, p.Sq, p.H, p.D, 128);
  if (rc) return 1000 + rc;
  const long long units = static_cast<long long>(p.splits) * p.H * p.B, grid = units * ((p.Sq + 255) / 256);
  if (grid > 0x7fffffffll) return 20;
  p.order = {(p.Sq + 255) / 256, (int)units, rbh::span_group(units, 4ll * p.Sk * p.D * p.Hkv / (p.splits * p.H) + 1)};
  const bool bias = p.c.slopes != nullptr;
  if (p.c.norms != nullptr) {
    const long long n = static_cast<long long>(p.B) * (p.H + p.Hkv) * 32;
    if (n > 0x7fffffffll) return 20;
    span_norms_kernel<T><<<(unsigned)n, 256, 0, st>>>((const T*)q, (const T*)k, qs[0], qs[1], qs[2], ks[0], ks[1], ks[2], const_cast<float*>(p.c.norms), p.H,
                                                      p.Hkv, p.Sq, p.Sk, p.D);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return 3000 + (int)e;
  }
#define RB_SPAN(HD_)                                                                                          \
  (cap ? bias ? launch_span_fwd<T, HD_, true, true>(tq, tk, tv, to, p, (unsigned)grid, st)                    \
              : launch_span_fwd<T, HD_, true, false>(tq, tk, tv, to, p, (unsigned)grid, st)                   \
       : bias ? launch_span_fwd<T, HD_, false, true>(tq, tk, tv, to, p, (unsigned)grid, st)                   \
              : launch_span_fwd<T, HD_, false, false>(tq, tk, tv, to, p, (unsigned)grid, st))
  rc = p.D <= 64 ? RB_SPAN(64) : RB_SPAN(128);
#undef RB_SPAN
  if (rc || p.splits == 1) return rc;
  return launch_span_join<T>(p.part_o, p.part_lse2, (T*)p.o, p.lse2, p.B, p.H, p.Sq, p.D, p.splits, st);
}

}  // namespace rb

extern "C" {

// Parts that the keys of a call are cut into: as many as fill the SMs once where the tiles of 256 rows alone leave half of them idle, each of 256 keys at
// least, 8 at most.  us at several numbers, heads of 128, the rule's in brackets: 512 rows over 8704 keys, 32 heads: 156 in 1 part, [93 in 2], 128 in 3; 1024
// over 4096, 18 heads: 78.8 in 1, [57.9 in 2]; 20 heads: [78.7 in 1], 94.8 in 2; 256 over 1024, 32 heads: 26.1 in 1, [22.2 in 4], 35.7 in 6; 64 over 4096, 8
// heads: 54.4 in 1, 22.2 in 4, [17.5 in 8], 19.5 in 16.
int rb_span_fwd_splits(int B, int H, int Sq, int Sk) {
  const long long tiles = static_cast<long long>((Sq + 255) / 256) * B * H;
  if (tiles <= 0 || 2 * tiles > rbh::sm_count()) return 1;
  const long long most = (static_cast<long long>(Sk) + 255) / 256, fill = rbh::sm_count() / tiles;
  const long long parts = fill < most ? fill : most;
  return static_cast<int>(parts < 1 ? 1 : parts > 8 ? 8 : parts);
}

// q [B, Sq, H, D], k and v [B, Sk, Hkv, D]: 16-bit views, strides {batch, row, head} in elements (multiples of 8), 16-byte aligned; D a multiple of 8, at
// most 128.  o [B, Sq, H, D] contiguous, lse2 [B, H, Sq].  spans: rows {lo, hi} of int32, `span_batch` rows apart per batch, or null; slopes [H] or
// null; cap 0: none.  splits > 1: part_o [splits, B, Sq, H, D] and part_lse2 [splits, B, H, Sq] are scratch.  norms: null, or
// with slopes and no cap fp32 [B, H + Hkv, 32] to note lengths in, by which tiles too far for a weight are left out.
int rb_span_fwd(int dtype, const void* q, const void* k, const void* v, const long long* qs, const long long* ks, const long long* vs, const int* spans,
                long long span_batch, const float* slopes, float* norms, void* o, float* lse2, float* part_o, float* part_lse2, int B, int H, int Hkv, int Sq, int Sk,
                int D, int splits, int causal, float scale, float cap, void* stream) {
  using namespace rb;
  if (B <= 0 || H <= 0 || Sq <= 0) return 0;
  if (Sk <= 0 || Hkv <= 0 || H % Hkv || D <= 0 || D > 128 || D % 8 || splits < 1 || (splits > 1 && (!part_o || !part_lse2))) return 20;
  SpanFwdParams p{};
  p.B = B; p.H = H; p.Hkv = Hkv; p.Sq = Sq; p.Sk = Sk; p.D = D;
  p.splits = splits;
  p.c = rbh::span_scores(scale, cap);
  p.c.slopes = slopes;
  p.c.norms = slopes && !(cap > 0.f) ? norms : nullptr;
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
