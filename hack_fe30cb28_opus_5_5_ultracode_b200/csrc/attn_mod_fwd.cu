// Attention forward with modified scores and masks on the 5th-generation tensor cores (head dims
// 64 and 128): see attn_mod.cuh for the score and the masks.
//
// One CTA takes two adjacent 128-query tiles of one head; both read the same K and V blocks of
// 128 keys, so each block crosses from L2 once for 256 queries. Nineteen warps:
//   warps 0-7, 8-15 softmax of tile 0 and of tile 1, two threads per query row (TMEM lane = row), 64
//                   of the 128 keys each: scores into registers, the row's maximum (the two threads
//                   exchange theirs through shared memory), P as 16-bit pairs into tensor memory,
//                   where the next product reads it as its A operand;
//   warps 16, 17    issue the MMAs of tile 0 and of tile 1: S_t = Q_t K^T into one score buffer that
//                   goes from tile to tile as soon as it has been read, and O_t += P_t V when P_t is
//                   there. So a tile's next scores are ready when its softmax warps are done with a
//                   block. (Each instruction of such a warp waits its turn among those of four softmax
//                   warps: one warp for both tiles took 1,800 cycles per tile and block, longer than
//                   the softmax.)
//   warp 18         TMA: Q tiles, then K and V blocks through a ring of tiles.
// TMEM columns: S [0, 128), P_0 [128, 192), P_1 [192, 256), O_0 [256, 256 + D), O_1 [384, 384 + D).
// The running maximum moves only when it grows by more than 2^8; then the row's O is rescaled.
// P is rounded to the input type for the product (half a step of 2^-8 or 2^-11 per probability,
// averaged over the row's keys); the row sum adds the unrounded values in fp32.
#include "attn_mod.cuh"
#include "profile.h"

namespace ql {

namespace {

template <int D, bool SPLIT>
struct FwdCfg {
  static constexpr int TILE = AM_T * D * 2;          // bytes of a 128-row tile
  static constexpr int Q_TILES = SPLIT ? 1 : 2;
  static constexpr int STAGES = D == 128 ? 7 - Q_TILES : 8;  // ring of K / V tiles
  static constexpr int OFF_KV = Q_TILES * TILE;
  static constexpr int OFF_M = OFF_KV + STAGES * TILE;  // [2 tiles][2 halves][128] fp32 exchange
  static constexpr int OFF_BAR = OFF_M + 4 * AM_T * 4;
  static constexpr int SMEM = OFF_BAR + 512;
};
constexpr int FWD_THREADS = 608;
constexpr int FWD_HC = 64;  // columns per softmax thread

// fp16 probabilities are kept as 2^7 P (at most 2^15, as P is at most 2^8 under a maximum that lags),
// so that the many small ones of a long row stay normal numbers; the row sum has the same factor.
template <typename T>
constexpr float FWD_P_SHIFT = std::is_same<T, __half>::value ? 7.f : 0.f;

// What the score's modes need per kernel.
struct ScoreConst {
  float sl2;    // scale * log2(e): plain scores
  float u;      // scale / cap
  float cap2;   // cap * log2(e)
  TanhShort ts;
};

// Scores of one row and one key block, in place: raw products stay in their units unless they are capped (the
// scale rides in the exponent's FMA), capped ones come in log2 units, masked ones are -inf. x: 64 values;
// dist0 = i - their first key; slope: the distance bias's, in the same units; side: 1 (-1) if every key of
// the block comes before (after) every query of the tile, else 0. A bias is one FMA of the score, the slope
// and an exact distance: sums of biases, from column to column, were off by up to seven roundings of the
// whole bias, which shows where far keys carry the weight (negative slopes).
template <int MODE, bool MASKED>
__device__ __forceinline__ void modify_scores(uint32_t* x, const ScoreConst& c, float slope,
                                              float dist0, float side, int rlo, int rhi) {
  if constexpr ((MODE & 1) != 0) {
    const int form = tanh_form<FWD_HC>(x, c.u);
    if (form == 0) {
#pragma unroll
      for (int i = 0; i < FWD_HC; i += 16) {
        uint64_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = pair_of(x + i + 2 * e);
        tanh_short2<8>(u, c.ts);
#pragma unroll
        for (int e = 0; e < 8; ++e) unpair(u[e], x + i + 2 * e);
      }
    } else if (form == 1) {
      const uint64_t uu = pk2(c.u, c.u), cc = pk2(c.cap2, c.cap2);
#pragma unroll
      for (int i = 0; i < FWD_HC; i += 16) {
        uint64_t u[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) u[e] = mul2(pair_of(x + i + 2 * e), uu);
        tanh_poly2<8>(u);
#pragma unroll
        for (int e = 0; e < 8; ++e) unpair(mul2(u[e], cc), x + i + 2 * e);
      }
    } else {
#pragma unroll
      for (int i = 0; i < FWD_HC; ++i)
        x[i] = __float_as_uint(tanhf(__uint_as_float(x[i]) * c.u) * c.cap2);
    }
  }
  if constexpr ((MODE & 2) != 0) {
    const uint64_t by = pk2(-slope, -slope);
    if (side != 0.f) {  // every key on one side of every query: |i - j| = side (dist0 - column)
      // four pairs of distances, moved on by eight columns at a time
      const float first = side * dist0;
      const uint64_t next = pk2(-8.f * side, -8.f * side);
      uint64_t away[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) away[e] = pk2(first - side * (float)(2 * e), first - side * (float)(2 * e + 1));
#pragma unroll
      for (int i = 0; i < FWD_HC; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          unpair(fma2(away[e], by, pair_of(x + i + 2 * e)), x + i + 2 * e);
          away[e] = add2(away[e], next);
        }
    } else {
#pragma unroll
      for (int i = 0; i < FWD_HC; ++i)
        x[i] = __float_as_uint(fmaf(fabsf(dist0 - (float)i), -slope, __uint_as_float(x[i])));
    }
  }
  if constexpr (MASKED) {
    const uint32_t m[2] = {col_mask(rlo, rhi), col_mask(rlo - 32, rhi - 32)};
#pragma unroll
    for (int i = 0; i < FWD_HC; ++i)
      if (!(m[i >> 5] >> (i & 31) & 1)) x[i] = 0xff800000u;  // -inf
  }
}

template <typename T, int D, int MODE, bool SPLIT>
__global__ void __launch_bounds__(FWD_THREADS, 1)
    attn_mod_fwd_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tk,
                        const __grid_constant__ CUtensorMap tv, const AttnModArgs a, int* err) {
  using C = FwdCfg<D, SPLIT>;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr int BOX = AM_T * 128;  // a 128-row x 64-column box
  pdl_enter();
  extern __shared__ __align__(1024) uint8_t smem[];  // no static shared memory: the base is aligned
  float* sM = reinterpret_cast<float*>(smem + C::OFF_M);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;                       // [2]
  uint64_t* s_full = bars + 2;                   // [2] the tile's scores written
  uint64_t* s_free = bars + 4;                   // [2] score buffer handed to the tile (8 warps)
  uint64_t* p_full = bars + 6;                   // [2] P written, O rescaled (8 warps)
  uint64_t* o_full = bars + 8;                   // [2] O += P V complete
  uint64_t* kv_raw = bars + 10;                  // a V tile whose dead rows are zeroed first
  uint64_t* drain = bars + 11;                   // [2]
  uint64_t* kv_full = bars + 13;                 // [STAGES]
  uint64_t* kv_empty = bars + 13 + C::STAGES;    // [STAGES] one arrival per tile
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 13 + 2 * C::STAGES);

  const int h = blockIdx.x % a.HQ, b = blockIdx.x / a.HQ;
  const int q0 = (gridDim.y - 1 - blockIdx.y) * C::Q_TILES * AM_T;  // the rows with the most keys first
  const AttnSeq seq = attn_seq(a, b);
  if (q0 >= seq.len) return;  // the whole CTA, before any barrier or TMEM is set up
  const int kvh = h / (a.HQ / a.HKV);
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  // the loading warp sets the barriers up and sends for Q while the others allocate and look at the mask
  if (warp == 18 && lane == 0) {
    for (int s = 0; s < 2; ++s) {
      mbar_init(&q_full[s], 1);
      mbar_init(&s_full[s], 1);
      mbar_init(&s_free[s], 8);
      mbar_init(&p_full[s], 8);
      mbar_init(&o_full[s], 1);
    }
    mbar_init(kv_raw, 1);
    mbar_init(&drain[0], 1);
    mbar_init(&drain[1], 1);
    for (int s = 0; s < C::STAGES; ++s) {
      mbar_init(&kv_full[s], 1);
      mbar_init(&kv_empty[s], 2);
    }
    fence_barrier_init();
    for (int t = 0; t < C::Q_TILES; ++t) {
      mbar_arrive_expect_tx(&q_full[t], C::TILE);
      tma_load_3d(smem + t * C::TILE, &tq, &q_full[t], 0, seq.start + q0 + t * AM_T, h * (D / 64));
    }
  }
  if (warp == 16) tmem_alloc(tmem_slot, 512);
  AttnBlocks tb0 = attn_tile_blocks(seq, q0), tb1 = SPLIT ? tb0 : attn_tile_blocks(seq, q0 + AM_T);
  tb0.first = uniform(tb0.first);
  tb0.end = uniform(tb0.end);
  tb1.first = uniform(tb1.first);
  tb1.end = uniform(tb1.end);
  // the blocks either tile visits: its own range, or the gap-free union where both have one
  const bool any0 = tb0.end > tb0.first, any1 = tb1.end > tb1.first + (SPLIT ? 1 : 0);
  const int jb = SPLIT || !any1 || (any0 && tb0.first < tb1.first) ? tb0.first : tb1.first;
  const int je = SPLIT || !any1 || (any0 && tb0.end > tb1.end) ? tb0.end : tb1.end;
  auto visits = [&](int t, int j) {
    if (SPLIT) return j >= tb0.first && j < tb0.end && ((j - tb0.first) & 1) == t;
    return t ? j >= tb1.first && j < tb1.end : j >= tb0.first && j < tb0.end;
  };
  if (warp == 18 && lane == 0 && je > jb) {  // the first K
    mbar_arrive_expect_tx(&kv_full[0], C::TILE);
    tma_load_3d(smem + C::OFF_KV, &tk, &kv_full[0], 0, seq.start + jb * AM_T, kvh * (D / 64));
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 18) {
    // ---- loads ----
    // A V tile with dead rows lands on kv_raw and is handed on when they have been zeroed, after the next
    // K has been sent for.
    int n = 0, unclean = -1;  // ring positions filled; the one whose rows are still to be zeroed
    uint32_t raw = 0;
    DeadRows dead;
    bool ok = true;
    auto clean = [&]() {
      if (unclean < 0) return true;
      if (!warp_wait(kv_raw, raw, err)) return false;
      raw ^= 1;
      attn_zero_rows<D / 64>(smem + C::OFF_KV + unclean * C::TILE, dead);
      fence_proxy_async_smem();
      warp_arrive(&kv_full[unclean]);
      unclean = -1;
      return true;
    };
    for (int j = jb; ok && j < je; ++j) {
      if (!visits(0, j) && !visits(1, j)) continue;
      const int row = j * AM_T;
#pragma unroll
      for (int is_v = 0; is_v < 2; ++is_v, ++n) {
        if (n == 0) continue;  // sent for above
        const int s = n % C::STAGES;
        if (is_v) {
          ok = clean();
          dead = attn_dead_rows(seq, row);
        }
        if (ok && n >= C::STAGES) ok = warp_wait(&kv_empty[s], (n / C::STAGES - 1) & 1, err);
        if (!ok) break;
        const bool dirty = is_v && dead.any;
        uint64_t* bar = dirty ? kv_raw : &kv_full[s];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, C::TILE);
          tma_load_3d(smem + C::OFF_KV + s * C::TILE, is_v ? &tv : &tk, bar, 0, seq.start + row, kvh * (D / 64));
        }
        if (dirty) unclean = s;
      }
    }
    if (ok) ok = clean();
    if (!ok && lane == 0) {  // a wait ran out: let the copies in flight land before the CTA goes
      mbar_wait(&q_full[0], 0, nullptr, 100000000ull);
      if (!SPLIT) mbar_wait(&q_full[1], 0, nullptr, 100000000ull);
      if (unclean >= 0) mbar_wait(kv_raw, raw, nullptr, 100000000ull);
      for (int k = max(0, n - C::STAGES); k < n; ++k)
        if (k % C::STAGES != unclean) mbar_wait(&kv_full[k % C::STAGES], (k / C::STAGES) & 1, nullptr, 100000000ull);
    }
  } else if (warp == 16 || warp == 17) {
    // ---- MMA of one tile ----
    const int t = warp - 16;
    if (je > jb) {
      constexpr uint32_t id_s = umma_idesc_f16(IS_BF16, 128, AM_T, false);
      constexpr uint32_t id_o = umma_idesc_f16(IS_BF16, 128, D, true);  // V is MN-major
      const uint32_t sq = desc_lo_k(smem_u32(smem + (SPLIT ? 0 : t * C::TILE)));
      const uint32_t sk = desc_lo_k(smem_u32(smem + C::OFF_KV));
      const uint32_t sv = desc_lo_mn(smem_u32(smem + C::OFF_KV), BOX);
      // The score buffer goes from item to item ((tile, block) pairs, block by block, tile 0 first): this
      // tile's next scores are formed when the softmax warps that read the item before pass the buffer
      // on to it (s_free). Blocks that only the other tile visits are handed back as they land, so that
      // both warps see every turn of the ring.
      const bool leads = t == 0 || !any0;  // has the first item
      int ring = 0;                        // position of the block's K in the ring (V follows)
      int n = 0, pend = -1;                // this tile's items so far; V of the product still to come
      auto gather = [&]() {                // O += P V of item n - 1
        const int s = pend % C::STAGES;
        if (!warp_wait(&kv_full[s], (pend / C::STAGES) & 1, err) || !warp_wait(&p_full[t], (n - 1) & 1, err))
          return false;
        tc_fence_after();
        umma_gather1(tmem + 256 + t * 128, tmem + 128 + t * 64, sv + s * (C::TILE >> 4), id_o, n > 1);
        warp_commit(&o_full[t]);
        warp_commit(&kv_empty[s]);
        pend = -1;
        return true;
      };
      bool ok = warp_wait(&q_full[SPLIT ? 0 : t], 0, err);
      for (int j = jb; ok && j < je; ++j) {
        const bool mine = visits(t, j);
        if (!mine && !visits(t ^ 1, j)) continue;  // not loaded
        if (!SPLIT && !mine && pend >= 0) ok = gather();  // it may have been the tile's last
        const int s = ring % C::STAGES, s1 = (ring + 1) % C::STAGES;
        if (ok) ok = warp_wait(&kv_full[s], (ring / C::STAGES) & 1, err);
        if (!ok) break;
        if (mine) {
          if (n > 0 || !leads) ok = warp_wait(&s_free[t], (n - (leads ? 1 : 0)) & 1, err);
          if (!ok) break;
          tc_fence_after();
          umma_score<D>(tmem, sq, sk + s * (C::TILE >> 4), id_s);
          warp_commit(&s_full[t]);
          warp_commit(&kv_empty[s]);
          if (pend >= 0) ok = gather();
          pend = ring + 1;
          ++n;
        } else {
          warp_arrive(&kv_empty[s]);
          ok = warp_wait(&kv_full[s1], ((ring + 1) / C::STAGES) & 1, err);
          if (ok) warp_arrive(&kv_empty[s1]);
        }
        ring += 2;
      }
      if (ok && pend >= 0) ok = gather();
      if (!ok) {  // a wait ran out: the products already issued finish before TMEM is freed
        warp_commit(&drain[t]);
        if (lane == 0) mbar_wait(&drain[t], 0, nullptr, 100000000ull);
        __syncwarp();
      }
    }
  } else {
    // ---- softmax ----
    const int t = warp >> 3, half = (warp >> 2) & 1, r = (warp & 3) * 32 + lane;
    const int qi = q0 + (SPLIT ? 0 : t * AM_T) + r;
    const AttnBlocks tb = t ? tb1 : tb0;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t ts = lane_base + half * FWD_HC, tp = lane_base + 128 + t * 64 + half * (FWD_HC / 2);
    const uint32_t to = lane_base + 256 + t * 128 + half * (D / 2);
    float* mine = sM + (2 * t + half) * AM_T + r;
    const float* other = sM + (2 * t + (half ^ 1)) * AM_T + r;
    // the two warps of a row meet in a named barrier once per block, also after a wait has run out: a
    // handshake over two mbarriers took 600 of a block's 3,300 cycles
    const int pair = 2 + t * 4 + (warp & 3);
    auto meet = [&]() { asm volatile("bar.sync %0, 64;" ::"r"(pair) : "memory"); };
    const int2 range = qi < seq.len ? attn_row_range(seq, qi) : make_int2(0, 0);
    ScoreConst c;
    c.sl2 = a.scale * 1.4426950408889634f;
    c.u = (MODE & 1) != 0 ? a.scale / a.softcap : 0.f;
    c.cap2 = a.softcap * 1.4426950408889634f;
    if constexpr ((MODE & 1) != 0) c.ts = tanh_short(c.u, c.cap2);
    const float slope = (MODE & 2) == 0 ? 0.f : (MODE & 1) != 0 ? a.slopes[h] * 1.4426950408889634f : a.slopes[h] / a.scale;
    const float mul = (MODE & 1) == 0 ? c.sl2 : 1.f;
    float m_run = -INFINITY, l_run = 0.f;
    bool ok = true;
    constexpr int STEP = SPLIT ? 2 : 1;
    for (int j = tb.first + (SPLIT ? t : 0); j < tb.end; j += STEP) {
      const int n = (j - tb.first) / STEP;
      ok = ok && warp_wait(&s_full[t], n & 1, err);
      if (!ok) {
        meet();
        continue;
      }
      tc_fence_after();
      uint32_t x[FWD_HC];
      tmem_ld32_nw(ts, x);
      tmem_ld32_nw(ts + 32, x + 32);
      tmem_wait_ld();
      tc_fence_before();
      // the buffer goes to tile 1 at this block, else to whichever tile visits the next one, or
      // (tile 0's last block before a gap) to tile 1
      const int heir = SPLIT ? (j + 1 < tb.end ? t ^ 1 : -1) : t == 0 && visits(1, j) ? 1 : visits(0, j + 1) ? 0 : visits(1, j + 1) || (t == 0 && any1) ? 1 : -1;
      if (heir >= 0) warp_arrive(&s_free[heir]);
      const bool masked = j < tb.ffirst || j >= tb.fend;
      const int j0 = j * AM_T + half * FWD_HC, qt = q0 / AM_T + (SPLIT ? 0 : t);
      const float side = j < qt ? 1.f : j > qt ? -1.f : 0.f;
      if (masked) modify_scores<MODE, true>(x, c, slope, (float)(qi - j0), side, range.x - j0, range.y - j0);
      else modify_scores<MODE, false>(x, c, slope, (float)(qi - j0), side, 0, 0);
      float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
      for (int i = 0; i < FWD_HC; i += 8)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          mx[e] = max3(mx[e], __uint_as_float(x[i + 2 * e]), __uint_as_float(x[i + 2 * e + 1]));
      // O_t += P_t V of the last block is complete: P_t may be written, O_t rescaled, and the other half has
      // read this thread's last maximum
      if (n > 0) ok = warp_wait(&o_full[t], (n - 1) & 1, err);
      const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
      *mine = top;
      meet();
      if (!ok) continue;
      tc_fence_after();
      const float ms = fmaxf(top, *other) * mul;
      float corr = 1.f;
      if (ms > m_run + 8.f) {
        corr = m_run == -INFINITY ? 0.f : ex2(m_run - ms);
        m_run = ms;
      }
      const float mneg = m_run == -INFINITY ? 0.f : FWD_P_SHIFT<T> - m_run;
      if (n > 0 && __any_sync(0xffffffffu, corr != 1.f)) {
#pragma unroll 1
        for (int u = 0; u < D / 32; ++u) {
          float ov[16];
          tmem_ld16(to + u * 16, ov);
#pragma unroll
          for (int e = 0; e < 16; ++e) ov[e] *= corr;
          tmem_st16(to + u * 16, ov);
        }
      }
      uint64_t sum[4] = {0, 0, 0, 0};  // pairs of +0.f
      const uint64_t mul_2 = pk2(mul, mul), neg_2 = pk2(mneg, mneg);
#pragma unroll
      for (int g = 0; g < FWD_HC; g += 32) {
        float w[16];  // 32 probabilities as 16-bit pairs
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          uint64_t y = fma2(pair_of(x + g + 2 * i), mul_2, neg_2);
          ex2_2<1>(&y);
          sum[i & 3] = add2(sum[i & 3], y);
          float pa, pb;
          up2(y, pa, pb);
          w[i] = __uint_as_float(pack_t2<T>(pa, pb));
        }
        tmem_st16(tp + g / 2, w);
      }
      tmem_wait_st();
      tc_fence_before();
      warp_arrive(&p_full[t]);
      float sa, sb;
      up2(add2(add2(sum[0], sum[1]), add2(sum[2], sum[3])), sa, sb);
      l_run = l_run * corr + (sa + sb);
    }
    const int count = max(0, tb.end - tb.first + STEP - 1 - (SPLIT ? t : 0)) / STEP;  // blocks it has had
    if (count > 0 && ok) {
      ok = warp_wait(&o_full[t], (count - 1) & 1, err);
      tc_fence_after();
    }
    // the row sum: both halves' sums, added in the same order in both threads
    *mine = l_run;
    meet();
    // O's columns [col0, col0 + COLS) of this thread's row: O_t / l, or with SPLIT both halves of the keys
    // brought to one maximum
    constexpr int COLS = D / 2 / STEP;
    const int col0 = (SPLIT ? 2 * t + half : half) * COLS;
    float l_row = half ? *other + l_run : l_run + *other, f0 = 1.f, f1 = 0.f;
    int count1 = 0;
    if constexpr (SPLIT) {
      asm volatile("bar.sync 1, 512;" ::: "memory");  // every sum has been read
      if (half == 0) {
        sM[2 * t * AM_T + r] = m_run;
        sM[(2 * t + 1) * AM_T + r] = l_row;
        if (!ok) sM[2 * t * AM_T + r] = NAN;
      }
      asm volatile("bar.sync 1, 512;" ::: "memory");
      tc_fence_after();
      const float m0 = sM[r], m1 = sM[2 * AM_T + r];
      m_run = fmaxf(m0, m1);
      f0 = m0 == -INFINITY ? 0.f : ex2(m0 - m_run);
      f1 = m1 == -INFINITY ? 0.f : ex2(m1 - m_run);
      l_row = f0 * sM[AM_T + r] + f1 * sM[3 * AM_T + r];
      ok = __all_sync(0xffffffffu, ok && m0 == m0 && m1 == m1);
      count1 = tb.end - tb.first > 1;
    }
    if (ok) {
      const float inv = l_row > 0.f ? 1.f / l_row : (l_row == 0.f ? 0.f : l_row);  // NaN stays
      // Q's tile has been read for the last time (or, with no block, has landed by now): the rows leave
      // through it
      if (tb.end == tb.first) warp_wait(&q_full[SPLIT ? 0 : t], 0, err);
      constexpr int W = 2 * COLS;  // bytes
      const uint32_t o_at = lane_base + 256 + (SPLIT ? 0 : t * 128) + col0;
      uint8_t* stage = smem + (SPLIT ? warp * 32 * W : t * C::TILE + (warp & 7) * 32 * W);
#pragma unroll
      for (int u = 0; u < COLS / 16; ++u) {
        float ov[16];
        if (tb.end > tb.first) {
          tmem_ld16(o_at + u * 16, ov);
          if constexpr (SPLIT) {
            float o1[16];
            if (count1) tmem_ld16(o_at + 128 + u * 16, o1);
#pragma unroll
            for (int e = 0; e < 16; ++e) ov[e] = count1 ? ov[e] * f0 + o1[e] * f1 : ov[e] * f0;
          }
        } else {
#pragma unroll
          for (int e = 0; e < 16; ++e) ov[e] = 0.f;
        }
#pragma unroll
        for (int v = 0; v < 2; ++v)
          *reinterpret_cast<uint4*>(stage_at<W>(stage, lane, 2 * u + v)) =
              make_uint4(pack_t2<T>(ov[8 * v] * inv, ov[8 * v + 1] * inv),
                         pack_t2<T>(ov[8 * v + 2] * inv, ov[8 * v + 3] * inv),
                         pack_t2<T>(ov[8 * v + 4] * inv, ov[8 * v + 5] * inv),
                         pack_t2<T>(ov[8 * v + 6] * inv, ov[8 * v + 7] * inv));
      }
      const int row = qi - lane;  // the warp's first
      T* out = reinterpret_cast<T*>(a.out_w) + ((int64_t)(seq.start + row) * a.HQ + h) * D + col0;
      stage_flush<W>(stage, reinterpret_cast<uint8_t*>(out), (int64_t)a.HQ * D * 2, seq.len - row);
      if (qi < seq.len && col0 == 0)
        a.lse[(int64_t)h * a.n + seq.start + qi] = (m_run - FWD_P_SHIFT<T> + log2f(l_row)) * 0.6931471805599453f;
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Documents: (first, end) of the run of equal ids each token is in, within its sequence; a token
// with a negative id gets the empty range (i, i). Two CTAs per sequence scan it in chunks of 4,096
// tokens, one forwards for the first tokens of the runs and one backwards for their ends.
constexpr int DOC_THREADS = 1024, DOC_PER = 4;

template <bool REV>
__device__ void doc_scan(const int32_t* ids, int len, int2* ranges, int* carry_smem) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int CH = DOC_THREADS * DOC_PER;
  const int nch = (len + CH - 1) / CH;
  int carry = REV ? len : 0;  // edge carried over from the chunks before
  for (int ch = 0; ch < nch; ++ch) {
    const int base = (REV ? nch - 1 - ch : ch) * CH + threadIdx.x * DOC_PER;
    int id[DOC_PER + 1];  // with the neighbour before (REV: after) the thread's tokens
#pragma unroll
    for (int e = 0; e <= DOC_PER; ++e) {
      const int i = base + e - (REV ? 0 : 1);
      id[e] = i >= 0 && i < len ? ids[i] : -1;
    }
    // an edge: forwards the first token of a run (its index), backwards the last (index + 1);
    // edge[e]: the nearest one at or before (REV: at or after) token e within the thread
    int edge[DOC_PER], best = REV ? 0x7fffffff : -1;
#pragma unroll
    for (int k = 0; k < DOC_PER; ++k) {
      const int e = REV ? DOC_PER - 1 - k : k, i = base + e;
      const bool is = REV ? (i == len - 1 || id[e] != id[e + 1]) : (i == 0 || id[e] != id[e + 1]);
      if (is && i < len) best = REV ? i + 1 : i;
      edge[e] = best;
    }
    // exclusive scan over the threads (max forwards; min over the later threads backwards)
    int v = best;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int w = REV ? __shfl_down_sync(0xffffffffu, v, o) : __shfl_up_sync(0xffffffffu, v, o);
      if (REV ? lane + o < 32 : lane >= o) v = REV ? min(v, w) : max(v, w);
    }
    if (lane == (REV ? 0 : 31)) carry_smem[warp] = v;
    int ex = REV ? __shfl_down_sync(0xffffffffu, v, 1) : __shfl_up_sync(0xffffffffu, v, 1);
    if (lane == (REV ? 31 : 0)) ex = REV ? 0x7fffffff : -1;
    __syncthreads();
    int all = REV ? 0x7fffffff : -1;
    for (int w = 0; w < DOC_THREADS / 32; ++w) {
      const int x = carry_smem[w];
      if (REV ? w > warp : w < warp) ex = REV ? min(ex, x) : max(ex, x);
      all = REV ? min(all, x) : max(all, x);
    }
    if (REV) ex = ex == 0x7fffffff ? carry : ex;
    else ex = ex == -1 ? carry : ex;
#pragma unroll
    for (int e = 0; e < DOC_PER; ++e) {
      const int i = base + e;
      if (i >= len) continue;
      const int found = edge[e] == (REV ? 0x7fffffff : -1) ? ex : edge[e];
      if (REV) ranges[i].y = id[e] < 0 ? i : found;
      else ranges[i].x = id[e + 1] < 0 ? i : found;
    }
    if (REV ? all != 0x7fffffff : all != -1) carry = all;
    __syncthreads();
  }
}

__global__ void __launch_bounds__(DOC_THREADS) doc_ranges_kernel(const int32_t* ids,
                                                                 const int32_t* cu, int2* ranges) {
  pdl_enter();
  __shared__ int sm[DOC_THREADS / 32];
  const int start = cu[blockIdx.x], len = cu[blockIdx.x + 1] - start;
  if (blockIdx.y == 0) doc_scan<false>(ids + start, len, ranges + start, sm);
  else doc_scan<true>(ids + start, len, ranges + start, sm);
}

template <typename T, int D, int MODE, bool SPLIT>
int launch_fwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mk,
               const CUtensorMap& mv, cudaStream_t s) {
  using C = FwdCfg<D, SPLIT>;
  static std::atomic<unsigned long long> done{0};
  auto kern = attn_mod_fwd_kernel<T, D, MODE, SPLIT>;
  const int st = attn_smem_limit(reinterpret_cast<const void*>(kern), C::SMEM, done);
  if (st != QL_STATUS_OK) return st;
  const dim3 grid((unsigned)(a.HQ * a.B), (unsigned)cdiv(a.max_len, C::Q_TILES * AM_T));
  launch_k(kern, grid, dim3(FWD_THREADS), C::SMEM, s, mq, mk, mv, a, status_word());
  return launched(1);
}

// Whether a CTA takes one query tile, and its two halves every second key block (SPLIT): the chain of
// the longest CTA is halved, against twice as many CTAs and twice the loads. Compared in key blocks
// per SM, as the longest CTA and as an SM's share of all, with 3 blocks' time for a CTA's set-up and
// end. Pairs against single tiles, us: 2,048 causal tokens of 12 heads 31 / 20; 8 x 64-2,048 of 4
// heads, capped 33 / 21; but 4 x 1,024 of 12 heads 23 / 28, 2,048 of 28 heads 40 / 52.
bool fwd_split(const AttnModArgs& a) {
  const double tiles = (double)cdiv(a.max_len, AM_T);
  const double reach = a.window > 0 ? (a.causal ? 1.0 : 2.0) * a.window / AM_T + 1 : 1e30;
  const double longest = tiles < reach ? tiles : reach;
  const double mean = a.causal && longest == tiles ? (tiles + 1) / 2 : longest;
  const double pairs = (double)cdiv(a.n, 2 * AM_T) * a.HQ / sm_count();
  const double whole = fmax(longest + 3, pairs * (mean + 3)), split = fmax(longest / 2 + 3, pairs * (mean + 6));
  return split < 0.85 * whole;
}

template <typename T, int D, int MODE>
int pick_fwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv,
             cudaStream_t s) {
  return fwd_split(a) ? launch_fwd<T, D, MODE, true>(a, mq, mk, mv, s) : launch_fwd<T, D, MODE, false>(a, mq, mk, mv, s);
}

template <typename T, int D>
int dispatch_fwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mk,
                 const CUtensorMap& mv, cudaStream_t s) {
  switch (attn_mode(a)) {
    case 0: return pick_fwd<T, D, 0>(a, mq, mk, mv, s);
    case 1: return pick_fwd<T, D, 1>(a, mq, mk, mv, s);
    case 2: return pick_fwd<T, D, 2>(a, mq, mk, mv, s);
    default: return pick_fwd<T, D, 3>(a, mq, mk, mv, s);
  }
}

}  // namespace

int attn_doc_ranges(const int32_t* doc_ids, const int32_t* cu_seqlens, int B, int n, int2* ranges,
                    cudaStream_t s) {
  launch_k(doc_ranges_kernel, dim3((unsigned)B, 2), dim3(DOC_THREADS), 0, s, doc_ids, cu_seqlens, ranges);
  return launched(1);
}

// The checks both directions share.
int attn_mod_check(const ql_attn_mod_args& m, AttnModArgs& a) {
  if (m.D != 64 && m.D != 128) return QL_STATUS_UNSUPPORTED;
  if (m.dtype != QL_F16 && m.dtype != QL_BF16) return QL_STATUS_BAD_ARG;
  if (m.n < 0 || m.B < 0 || m.max_len < 0 || m.max_len > m.n || m.n > (1 << 29) || m.HKV <= 0 ||
      m.HQ <= 0 || m.HQ % m.HKV != 0 || m.window < 0)
    return QL_STATUS_BAD_ARG;
  if ((int64_t)m.HQ * m.B > 0x7fffffff || cdiv(m.max_len, AM_T) > 65535) return QL_STATUS_UNSUPPORTED;
  if (!(m.scale > 0.f && m.scale < INFINITY) || !(m.softcap >= 0.f && m.softcap < INFINITY))
    return QL_STATUS_BAD_ARG;
  if (m.slopes != nullptr && m.scale < 1e-30f) return QL_STATUS_BAD_ARG;  // slope / scale has to stay finite
  // tanh_short's coefficients hold (scale / softcap)^7: finite up to 10^4, a cap that bends every score
  if (m.softcap > 0.f && m.softcap < 1e-4f * m.scale) return QL_STATUS_BAD_ARG;
  // scale and softcap times log2(e) have to be finite, scale / softcap a normal number
  if (m.scale > 2.3e38f || m.softcap > 2.3e38f || (m.softcap > 0.f && m.scale / m.softcap < 1.1754944e-38f))
    return QL_STATUS_BAD_ARG;
  if (m.n > 0 && m.B > 0 && (m.q == nullptr || m.k == nullptr || m.v == nullptr || m.out == nullptr ||
                             m.lse == nullptr || m.cu_seqlens == nullptr))
    return QL_STATUS_BAD_ARG;
  if (m.doc_ids != nullptr && (m.ranges == nullptr || (reinterpret_cast<uintptr_t>(m.ranges) & 7)))
    return QL_STATUS_BAD_ARG;
  // TMA: 16-byte aligned bases and row strides
  if (((reinterpret_cast<uintptr_t>(m.q) | reinterpret_cast<uintptr_t>(m.k) |
        reinterpret_cast<uintptr_t>(m.v) | reinterpret_cast<uintptr_t>(m.out)) & 15) ||
      ((m.ldq | m.ldk | m.ldv) & 7) || m.ldq < (int64_t)m.HQ * m.D ||
      m.ldk < (int64_t)m.HKV * m.D || m.ldv < (int64_t)m.HKV * m.D)
    return QL_STATUS_BAD_ARG;
  a = AttnModArgs{};
  a.q = m.q;
  a.k = m.k;
  a.v = m.v;
  a.out = m.out;
  a.out_w = m.out;
  a.lse = m.lse;
  a.cu_seqlens = m.cu_seqlens;
  a.slopes = m.slopes;
  a.prefix_len = m.prefix_len;
  a.docs = m.doc_ids != nullptr ? reinterpret_cast<const int2*>(m.ranges) : nullptr;
  a.scale = m.scale;
  a.softcap = m.softcap;
  a.n = m.n;
  a.B = m.B;
  a.max_len = m.max_len;
  a.HQ = m.HQ;
  a.HKV = m.HKV;
  a.causal = m.causal;
  a.window = m.window < (1 << 30) ? m.window : (1 << 30);
  return QL_STATUS_OK;
}

int attn_mod_fwd(const ql_attn_mod_args& m, cudaStream_t s) {
  AttnModArgs a;
  int st = attn_mod_check(m, a);
  if (st != QL_STATUS_OK) return st;
  if (m.n == 0 || m.B == 0 || m.max_len == 0) return QL_STATUS_OK;
  // out may take q's place: a CTA writes the rows and the head whose q it alone has read
  const int64_t rows = m.n, row = (int64_t)m.HQ * m.D;
  const bool in_place = m.out == m.q && m.ldq == row;
  if (outputs_overlap({{m.out, rows * row * 2}, {m.lse, rows * m.HQ * 4}, {m.doc_ids != nullptr ? m.ranges : nullptr, rows * 8}},
                      {{in_place ? nullptr : m.q, ((rows - 1) * m.ldq + row) * 2},
                       {m.k, ((rows - 1) * m.ldk + (int64_t)m.HKV * m.D) * 2},
                       {m.v, ((rows - 1) * m.ldv + (int64_t)m.HKV * m.D) * 2},
                       {m.cu_seqlens, ((int64_t)m.B + 1) * 4},
                       {m.slopes, (int64_t)m.HQ * 4},
                       {m.prefix_len, (int64_t)m.B * 4},
                       {m.doc_ids, rows * 4}}))
    return QL_STATUS_BAD_ARG;
  ProfScope prof(PK_ATTN_FWD, 0, 0, s);
  if (m.doc_ids != nullptr) {
    st = attn_doc_ranges(m.doc_ids, m.cu_seqlens, m.B, m.n, reinterpret_cast<int2*>(m.ranges), s);
    if (st != QL_STATUS_OK) return st;
  }
  const bool bf = m.dtype == QL_BF16;
  CUtensorMap mq, mk, mv;
  if (attn_head_map(&mq, m.q, m.n, m.HQ, m.D, m.ldq, bf) != QL_STATUS_OK ||
      attn_head_map(&mk, m.k, m.n, m.HKV, m.D, m.ldk, bf) != QL_STATUS_OK ||
      attn_head_map(&mv, m.v, m.n, m.HKV, m.D, m.ldv, bf) != QL_STATUS_OK)
    return QL_STATUS_CUDA;
  if (m.D == 128) return bf ? dispatch_fwd<__nv_bfloat16, 128>(a, mq, mk, mv, s)
                            : dispatch_fwd<__half, 128>(a, mq, mk, mv, s);
  return bf ? dispatch_fwd<__nv_bfloat16, 64>(a, mq, mk, mv, s) : dispatch_fwd<__half, 64>(a, mq, mk, mv, s);
}

}  // namespace ql
