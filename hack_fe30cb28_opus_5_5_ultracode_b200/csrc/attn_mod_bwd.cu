// Attention backward with modified scores and masks on the 5th-generation tensor cores (head dims
// 64 and 128): see attn_mod.cuh for the score and the masks. With y the score in log2 units,
//   P = 2^(y - lse2),  dP = dO V^T,  dS = P (dP - Dvec) (1 - tanh^2),
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,   Dvec = rowsum(dO * O).
//
// Two kernels, each recomputing P: one sums dQ over the keys of a query tile, the other dK and dV
// over the queries of a key block. That is 7 products where one kernel for all three needs 5, but
// dQ is then summed in tensor memory instead of by fp32 reductions in L2 (64 KB of them per
// 128 x 128 tile), the result is bit-identical from run to run, and the gradients leave in 16 bits
// with no fp32 buffer to zero and convert. P and dS are rounded to the input type for the products;
// every sum is fp32.
//
// Both kernels: eight softmax warps, two threads per TMEM lane (each 64 of the 128 columns; there is
// no row reduction, the forward's lse is known), one MMA warp, one TMA warp. The 16-bit P and dS go
// back into the tensor-memory columns their scores came from - each thread inside its own 64
// columns - and are read there as the A operand of the next product.
#include "attn_mod.cuh"
#include "profile.h"

namespace ql {

namespace {

constexpr int BWD_THREADS = 320;
constexpr int BOX = AM_T * 128;  // a 128-row x 64-column box
constexpr int HC = 64;           // columns per softmax thread

struct BwdConst {
  float sl2, u, cap2, slope2;
};

// 64 raw scores of one TMEM lane into probabilities times what the cap's derivative leaves of them
// (f, in place of x), and into plain probabilities as 16-bit pairs (p16, KEEP_P). neg_lse: pairs of
// -lse2 by column (PER_COL, from shared memory) or one value. Masked columns [0, lo) and [hi, 64)
// give 0. dist0: row index minus the first column's, for the distance bias.
template <typename T, int MODE, bool MASKED, bool PER_COL, bool KEEP_P>
__device__ __forceinline__ void bwd_probs(uint32_t* x, uint32_t* p16, const BwdConst& c,
                                          const float* neg_lse, float neg_lse_row, float dist0,
                                          int lo, int hi) {
  bool poly = true;
  if constexpr ((MODE & 1) != 0) {
    float mx = 0.f;
#pragma unroll
    for (int i = 0; i < HC; i += 2)
      mx = max3(mx, fabsf(__uint_as_float(x[i])), fabsf(__uint_as_float(x[i + 1])));
    poly = __all_sync(0xffffffffu, mx * c.u <= TANH_POLY_MAX);
  }
  const uint64_t row2 = pk2(neg_lse_row, neg_lse_row);
#pragma unroll
  for (int i = 0; i < HC; i += 4) {
    uint64_t nl[2] = {row2, row2};
    if constexpr (PER_COL) {
      const float4 l = *reinterpret_cast<const float4*>(neg_lse + i);
      nl[0] = pk2(l.x, l.y);
      nl[1] = pk2(l.z, l.w);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = i + 2 * e;
      const uint64_t raw = pk2(__uint_as_float(x[k]), __uint_as_float(x[k + 1]));
      uint64_t y, bend = 0;
      if constexpr ((MODE & 1) != 0) {
        uint64_t th;
        if (poly) {
          th = tanh_poly2(mul2(raw, pk2(c.u, c.u)));
        } else {
          th = pk2(tanhf(__uint_as_float(x[k]) * c.u), tanhf(__uint_as_float(x[k + 1]) * c.u));
        }
        bend = fma2(mul2(th, pk2(-1.f, -1.f)), th, pk2(1.f, 1.f));
        y = fma2(th, pk2(c.cap2, c.cap2), nl[e]);
      } else {
        y = fma2(raw, pk2(c.sl2, c.sl2), nl[e]);
      }
      float ya, yb;
      up2(y, ya, yb);
      if constexpr ((MODE & 2) != 0) {
        ya -= fabsf(c.slope2 * (dist0 - (float)k));
        yb -= fabsf(c.slope2 * (dist0 - (float)(k + 1)));
      }
      float pa = ex2(ya), pb = ex2(yb);
      if constexpr (MASKED) {
        if (k < lo || k >= hi) pa = 0.f;
        if (k + 1 < lo || k + 1 >= hi) pb = 0.f;
      }
      if constexpr (KEEP_P) p16[k / 2] = pack_t2<T>(pa, pb);
      if constexpr ((MODE & 1) != 0) {
        float fa, fb;
        up2(mul2(pk2(pa, pb), bend), fa, fb);
        // a masked score may be anything, infinities and NaN too: its factor is 0
        x[k] = __float_as_uint(MASKED && pa == 0.f ? 0.f : fa);
        x[k + 1] = __float_as_uint(MASKED && pb == 0.f ? 0.f : fb);
      } else {
        x[k] = __float_as_uint(pa);
        x[k + 1] = __float_as_uint(pb);
      }
    }
  }
}

// dS = f (dP dscale - Dvec') as 16-bit pairs; neg_d: -Dvec' by column or one value.
template <typename T, bool MASKED, bool PER_COL>
__device__ __forceinline__ void bwd_ds(const uint32_t* f, const uint32_t* dp, float* ds16, float dscale,
                                       const float* neg_d, float neg_d_row, int lo, int hi) {
  const uint64_t row2 = pk2(neg_d_row, neg_d_row), ds2 = pk2(dscale, dscale);
#pragma unroll
  for (int i = 0; i < HC; i += 4) {
    uint64_t nd[2] = {row2, row2};
    if constexpr (PER_COL) {
      const float4 l = *reinterpret_cast<const float4*>(neg_d + i);
      nd[0] = pk2(l.x, l.y);
      nd[1] = pk2(l.z, l.w);
    }
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int k = i + 2 * e;
      uint64_t v = fma2(pk2(__uint_as_float(dp[k]), __uint_as_float(dp[k + 1])), ds2, nd[e]);
      v = mul2(v, pk2(__uint_as_float(f[k]), __uint_as_float(f[k + 1])));
      float a, b;
      up2(v, a, b);
      if constexpr (MASKED) {  // 0 times whatever a masked place holds
        if (k < lo || k >= hi) a = 0.f;
        if (k + 1 < lo || k + 1 >= hi) b = 0.f;
      }
      ds16[k / 2] = __uint_as_float(pack_t2<T>(a, b));
    }
  }
}

// TMEM column of k-step kk (16 elements) of a 16-bit A operand kept in two halves of 32 columns at
// the start of each thread half's 64.
__device__ __forceinline__ uint32_t a_col(int kk) { return (kk >> 2) * 64 + (kk & 3) * 8; }

template <int MODE>
__device__ __forceinline__ BwdConst bwd_const(const AttnModArgs& a, int h) {
  BwdConst c;
  c.sl2 = a.scale * 1.4426950408889634f;
  c.u = (MODE & 1) != 0 ? a.scale / a.softcap : 0.f;
  c.cap2 = a.softcap * 1.4426950408889634f;
  c.slope2 = (MODE & 2) != 0 ? a.slopes[h] * 1.4426950408889634f : 0.f;
  return c;
}

// 16 consecutive columns of one row: 16-bit (scaled) into dst
template <typename T>
__device__ __forceinline__ void store_row16(T* dst, const float* v, float s) {
#pragma unroll
  for (int u = 0; u < 4; ++u)
    reinterpret_cast<uint4*>(dst)[u] =
        make_uint4(pack_t2<T>(v[8 * u] * s, v[8 * u + 1] * s), pack_t2<T>(v[8 * u + 2] * s, v[8 * u + 3] * s),
                   pack_t2<T>(v[8 * u + 4] * s, v[8 * u + 5] * s), pack_t2<T>(v[8 * u + 6] * s, v[8 * u + 7] * s));
}

// ---------------------------------------------------------------------------------------------
// dQ (and Dvec): one CTA per (128-query tile, query head, sequence)
// ---------------------------------------------------------------------------------------------
// Per key block j: S = Q K^T into one of two score buffers, dP = dO V^T, then dQ += dS K. The next
// block's S runs while the softmax warps work on this one; after dS_j the tensor core does
// dP_{j+1}, dQ_j and S_{j+2}. TMEM: S [0, 256), dP [256, 384), dQ [384, 384 + D).
template <int D>
struct DqCfg {
  static constexpr int TILE = AM_T * D * 2;
  static constexpr int KST = 3, VST = 2;
  static constexpr int OFF_DO = TILE, OFF_K = 2 * TILE, OFF_V = OFF_K + KST * TILE;
  static constexpr int OFF_D = OFF_V + VST * TILE;      // [2][128] partial Dvec
  static constexpr int OFF_BAR = OFF_D + 2 * AM_T * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
};

template <typename T, int D, int MODE>
__global__ void __launch_bounds__(BWD_THREADS, 1)
    attn_mod_dq_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                       const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                       const AttnModArgs a, int* err) {
  using C = DqCfg<D>;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  pdl_enter();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sD = reinterpret_cast<float*>(smem + C::OFF_D);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* q_full = bars;       // Q
  uint64_t* do_full = bars + 1;  // dO
  uint64_t* s_full = bars + 2;   // [2]
  uint64_t* dp_full = bars + 4;  // dP written
  uint64_t* ds_full = bars + 5;  // dS written, dP read (256 threads)
  uint64_t* dq_full = bars + 6;
  uint64_t* raw = bars + 7;
  uint64_t* drain = bars + 8;
  uint64_t* k_full = bars + 9;    // [3]
  uint64_t* k_empty = bars + 12;  // [3]
  uint64_t* v_full = bars + 15;   // [2]
  uint64_t* v_empty = bars + 17;  // [2]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 19);

  const int h = blockIdx.x % a.HQ, b = blockIdx.x / a.HQ;
  const int q0 = (gridDim.y - 1 - blockIdx.y) * AM_T;
  const AttnSeq seq = attn_seq(a, b);
  if (q0 >= seq.len) return;  // the whole CTA, before any barrier or TMEM is set up
  const int kvh = h / (a.HQ / a.HKV);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnBlocks tb = attn_tile_blocks(seq, q0);
  const int nblk = tb.end - tb.first;

  if (threadIdx.x == 0) {
    mbar_init(q_full, 1);
    mbar_init(do_full, 1);
    mbar_init(&s_full[0], 1);
    mbar_init(&s_full[1], 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 256);
    mbar_init(dq_full, 1);
    mbar_init(raw, 1);
    mbar_init(drain, 1);
    for (int s = 0; s < C::KST; ++s) {
      mbar_init(&k_full[s], 1);
      mbar_init(&k_empty[s], 1);
    }
    for (int s = 0; s < C::VST; ++s) {
      mbar_init(&v_full[s], 1);
      mbar_init(&v_empty[s], 1);
    }
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 9) {
    // ---- loads ----
    bool ok = true;
    int kn = 0, vn = 0;
    uint32_t raw_phase = 0;
    if (lane == 0 && nblk > 0) {
      mbar_arrive_expect_tx(q_full, C::TILE);
      tma_load_3d(smem, &tq, q_full, 0, seq.start + q0, h * (D / 64));
    }
    for (int n = 0; ok && n < nblk; ++n) {
      const int row = (tb.first + n) * AM_T;
      {  // K: dead rows zeroed (dQ = dS K would add 0 times whatever they hold)
        const int s = n % C::KST;
        uint32_t bad[4];
        const bool dirty = attn_dead_rows(seq, row, bad);
        if (n >= C::KST) ok = warp_wait(&k_empty[s], (n / C::KST - 1) & 1, err);
        if (!ok) break;
        uint8_t* dst = smem + C::OFF_K + s * C::TILE;
        uint64_t* bar = dirty ? raw : &k_full[s];
        if (lane == 0) {
          mbar_arrive_expect_tx(bar, C::TILE);
          tma_load_3d(dst, &tk, bar, 0, seq.start + row, kvh * (D / 64));
        }
        if (n == 0 && lane == 0) {
          mbar_arrive_expect_tx(do_full, C::TILE);
          tma_load_3d(smem + C::OFF_DO, &tdo, do_full, 0, seq.start + q0, h * (D / 64));
        }
        if (dirty) {
          ok = warp_wait(raw, raw_phase, err);
          if (!ok) break;
          raw_phase ^= 1;
          attn_zero_rows<D / 64>(dst, bad);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&k_full[s]);
        }
        kn = n + 1;
      }
      {
        const int s = n % C::VST;
        if (n >= C::VST) ok = warp_wait(&v_empty[s], (n / C::VST - 1) & 1, err);
        if (!ok) break;
        if (lane == 0) {
          mbar_arrive_expect_tx(&v_full[s], C::TILE);
          tma_load_3d(smem + C::OFF_V + s * C::TILE, &tv, &v_full[s], 0, seq.start + row, kvh * (D / 64));
        }
        vn = n + 1;
      }
    }
    if (!ok && lane == 0) {  // a wait ran out: let the copies in flight land before the CTA goes
      mbar_wait(q_full, 0, nullptr, 100000000ull);
      mbar_wait(do_full, 0, nullptr, 100000000ull);
      for (int n = max(0, kn - C::KST); n < kn; ++n)
        mbar_wait(&k_full[n % C::KST], (n / C::KST) & 1, nullptr, 100000000ull);
      for (int n = max(0, vn - C::VST); n < vn; ++n)
        mbar_wait(&v_full[n % C::VST], (n / C::VST) & 1, nullptr, 100000000ull);
    }
  } else if (warp == 8) {
    // ---- MMA ----
    if (lane == 0 && nblk > 0) {
      constexpr uint32_t id_s = umma_idesc_f16(IS_BF16, 128, AM_T, false);
      constexpr uint32_t id_q = umma_idesc_f16(IS_BF16, 128, D, true);
      const uint32_t sq = smem_u32(smem), sdo = smem_u32(smem + C::OFF_DO);
      const uint32_t sk = smem_u32(smem + C::OFF_K), sv = smem_u32(smem + C::OFF_V);
      auto product = [&](uint32_t d, uint32_t A, uint32_t B) {  // [128 x 128] over D
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * BOX + (kk & 3) * 32;
          umma_f16(d, umma_desc_k_sw128(A + off), umma_desc_k_sw128(B + off), id_s, kk > 0);
        }
      };
      auto score = [&](int n) {  // S_n
        const bool got = mbar_wait(&k_full[n % C::KST], (n / C::KST) & 1, err);
        if (got) {
          tc_fence_after();
          product(tmem + (n & 1) * 128, sq, sk + (n % C::KST) * C::TILE);
          umma_commit(&s_full[n & 1]);
        }
        return got;
      };
      auto dprob = [&](int n) {  // dP_n
        const bool got = mbar_wait(&v_full[n % C::VST], (n / C::VST) & 1, err);
        if (got) {
          tc_fence_after();
          product(tmem + 256, sdo, sv + (n % C::VST) * C::TILE);
          umma_commit(dp_full);
          umma_commit(&v_empty[n % C::VST]);
        }
        return got;
      };
      bool ok = mbar_wait(q_full, 0, err) && score(0) && mbar_wait(do_full, 0, err) && dprob(0);
      if (ok && nblk > 1) ok = score(1);
      for (int n = 0; ok && n < nblk; ++n) {
        ok = mbar_wait(ds_full, n & 1, err);
        if (!ok) break;
        tc_fence_after();
        if (n + 1 < nblk) ok = dprob(n + 1);
        if (!ok) break;
        const uint32_t bk = sk + (n % C::KST) * C::TILE, as = tmem + (n & 1) * 128;
#pragma unroll
        for (int kk = 0; kk < AM_T / 16; ++kk)
          umma_f16_ts(tmem + 384, as + a_col(kk), umma_desc_mn_sw128(bk + kk * 2048, BOX, 1024), id_q,
                      n > 0 || kk > 0);
        umma_commit(&k_empty[n % C::KST]);
        if (n + 1 == nblk) umma_commit(dq_full);
        if (n + 2 < nblk) ok = score(n + 2);
      }
      if (!ok) {
        umma_commit(drain);
        mbar_wait(drain, 0, nullptr, 100000000ull);
      }
    }
  } else {
    // ---- softmax ----
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, qi = q0 + r;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool live = qi < seq.len;
    const int2 range = live ? attn_row_range(seq, qi) : make_int2(0, 0);
    const bool sees = range.y > range.x;
    const BwdConst c = bwd_const<MODE>(a, h);
    const int64_t row = (int64_t)(seq.start + qi) * a.HQ + h;
    // Dvec: each of the row's two threads takes half of the head
    float part = 0.f;
    if (sees) {
      const uint4* o = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.out) + row * D + half * (D / 2));
      const uint4* g = reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.dout) + row * D + half * (D / 2));
#pragma unroll
      for (int u = 0; u < D / 16; ++u) {
        const uint4 ov = o[u], gv = g[u];
        const T* ot = reinterpret_cast<const T*>(&ov);
        const T* gt = reinterpret_cast<const T*>(&gv);
#pragma unroll
        for (int e = 0; e < 8; ++e) part = fmaf(to_f<T>(ot[e]), to_f<T>(gt[e]), part);
      }
    }
    sD[half * AM_T + r] = part;
    asm volatile("bar.sync 1, 256;" ::: "memory");
    const float dvec = sD[r] + sD[AM_T + r];
    float neg_lse = -INFINITY;  // 2^-inf = 0 for a row that sees nothing
    if (live) {
      if (half == 0) a.dvec[(int64_t)h * a.n + seq.start + qi] = dvec;
      if (sees) neg_lse = a.lse[(int64_t)h * a.n + seq.start + qi] * -1.4426950408889634f;
    }
    bool ok = true;
    for (int n = 0; n < nblk; ++n) {
      const int j = tb.first + n, j0 = j * AM_T + half * HC;
      const bool masked = j < tb.ffirst || j >= tb.fend;
      const int lo = range.x - j0, hi = range.y - j0;
      ok = warp_wait(&s_full[n & 1], (n >> 1) & 1, err);
      if (!ok) break;
      tc_fence_after();
      const uint32_t ts = lane_base + (n & 1) * 128 + half * HC;
      uint32_t x[HC], dp[HC];
      tmem_ld32_nw(ts, x);
      tmem_ld32_nw(ts + 32, x + 32);
      tmem_wait_ld();
      if (masked) bwd_probs<T, MODE, true, false, false>(x, nullptr, c, nullptr, neg_lse, (float)(qi - j0), lo, hi);
      else bwd_probs<T, MODE, false, false, false>(x, nullptr, c, nullptr, neg_lse, (float)(qi - j0), 0, 0);
      ok = warp_wait(dp_full, n & 1, err);
      if (!ok) break;
      tc_fence_after();
      tmem_ld32_nw(lane_base + 256 + half * HC, dp);
      tmem_ld32_nw(lane_base + 256 + half * HC + 32, dp + 32);
      tmem_wait_ld();
      float w[32];
      if (masked) bwd_ds<T, true, false>(x, dp, w, 1.f, nullptr, -dvec, lo, hi);
      else bwd_ds<T, false, false>(x, dp, w, 1.f, nullptr, -dvec, 0, 0);
      tmem_st32(ts, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(ds_full);
    }
    if (ok && nblk > 0) {
      ok = warp_wait(dq_full, 0, err);
      tc_fence_after();
    }
    if (ok) {
      T* dst = reinterpret_cast<T*>(a.dq) + row * D + half * (D / 2);
#pragma unroll 1
      for (int u = 0; u < D / 64; ++u) {
        float v[32];
        if (nblk > 0) {
          tmem_ld32(lane_base + 384 + half * (D / 2) + u * 32, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        if (live) store_row16<T>(dst + u * 32, v, a.scale);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// ---------------------------------------------------------------------------------------------
// dK and dV: one CTA per (128-key block, KV head, split of its query heads, sequence)
// ---------------------------------------------------------------------------------------------
// K and V stay in shared memory; for every query head of the split, the query tiles that see the
// block stream through a ring (Q, dO, -lse2, -Dvec). Per tile: S^T = K Q^T, dP^T = V dO^T,
// dV += P^T dO, dK += dS^T Q. While the softmax warps form P the tensor core does the last tile's dK
// and this one's dP^T, while they form dS it does dV and the next tile's S^T.
// TMEM: S^T [0, 128), dP^T [128, 256), dV [256, 256 + D), dK [384, 384 + D).
// fp16: P is kept as 2^8 P (at most 2^8 where P is 1), so that the small probabilities of long rows
// stay normal numbers; dS and dV take the factor back in fp32.
template <int D>
struct DkvCfg {
  static constexpr int TILE = AM_T * D * 2;
  static constexpr int ST = 2;
  static constexpr int OFF_V = TILE, OFF_Q = 2 * TILE, OFF_DO = OFF_Q + ST * TILE;
  static constexpr int OFF_L = OFF_DO + ST * TILE;  // [ST][2][128] fp32
  static constexpr int OFF_BAR = OFF_L + ST * 2 * AM_T * 4;
  static constexpr int SMEM = OFF_BAR + 256 + 1024;
};

template <typename T, int D, int MODE>
__global__ void __launch_bounds__(BWD_THREADS, 1)
    attn_mod_dkv_kernel(const __grid_constant__ CUtensorMap tq, const __grid_constant__ CUtensorMap tdo,
                        const __grid_constant__ CUtensorMap tk, const __grid_constant__ CUtensorMap tv,
                        const AttnModArgs a, int* err) {
  using C = DkvCfg<D>;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr float P_SHIFT = IS_BF16 ? 0.f : 8.f, P_BACK = IS_BF16 ? 1.f : 1.f / 256.f;
  pdl_enter();
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  float* sL = reinterpret_cast<float*>(smem + C::OFF_L);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* kv_full = bars;
  uint64_t* s_full = bars + 1;
  uint64_t* p_full = bars + 2;   // P written (256 threads)
  uint64_t* dp_full = bars + 3;
  uint64_t* ds_full = bars + 4;  // dS written (256 threads)
  uint64_t* out_full = bars + 5;
  uint64_t* raw = bars + 6;
  uint64_t* drain = bars + 7;
  uint64_t* q_full = bars + 8;    // [2] Q landed, -lse2 and -Dvec stored (1 + 32 lanes)
  uint64_t* do_full = bars + 10;  // [2]
  uint64_t* q_empty = bars + 12;  // [2] every product reading the stage completed
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 14);

  const int per_seq = a.HKV * a.splits;
  const int b = blockIdx.x / per_seq, kvh = (blockIdx.x % per_seq) / a.splits;
  const int split = blockIdx.x % a.splits;
  const int heads = a.HQ / a.HKV / a.splits, h0 = kvh * (a.HQ / a.HKV) + split * heads;
  const int k0 = blockIdx.y * AM_T;
  const AttnSeq seq = attn_seq(a, b);
  if (k0 >= seq.len) return;  // the whole CTA, before any barrier or TMEM is set up
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const AttnBlocks tb = attn_key_blocks(seq, k0);
  const int ntile = tb.end - tb.first, steps = ntile * heads;

  if (threadIdx.x == 0) {
    mbar_init(kv_full, 1);
    mbar_init(s_full, 1);
    mbar_init(p_full, 256);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, 256);
    mbar_init(out_full, 1);
    mbar_init(raw, 1);
    mbar_init(drain, 1);
    for (int s = 0; s < C::ST; ++s) {
      mbar_init(&q_full[s], 33);
      mbar_init(&do_full[s], 1);
      mbar_init(&q_empty[s], 1);
    }
    fence_barrier_init();
    prefetch_tmap(&tq);
    prefetch_tmap(&tdo);
    prefetch_tmap(&tk);
    prefetch_tmap(&tv);
  }
  if (warp == 8) tmem_alloc(tmem_slot, 512);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  if (warp == 9) {
    // ---- loads ----
    bool ok = true;
    int issued = 0;
    uint32_t raw_phase = 0;
    if (lane == 0 && steps > 0) {
      mbar_arrive_expect_tx(kv_full, 2 * C::TILE);
      tma_load_3d(smem, &tk, kv_full, 0, seq.start + k0, kvh * (D / 64));
      tma_load_3d(smem + C::OFF_V, &tv, kv_full, 0, seq.start + k0, kvh * (D / 64));
    }
    for (int n = 0; ok && n < steps; ++n) {
      const int s = n % C::ST, h = h0 + n / ntile, row = (tb.first + n % ntile) * AM_T;
      uint32_t bad[4];
      const bool dirty = attn_dead_rows(seq, row, bad);
      if (n >= C::ST) ok = warp_wait(&q_empty[s], (n / C::ST - 1) & 1, err);
      if (!ok) break;
      uint8_t* sq = smem + C::OFF_Q + s * C::TILE;
      uint8_t* sdo = smem + C::OFF_DO + s * C::TILE;
      if (lane == 0) {
        if (dirty) {
          mbar_arrive_expect_tx(raw, 2 * C::TILE);
        } else {
          mbar_arrive_expect_tx(&q_full[s], C::TILE);
          mbar_arrive_expect_tx(&do_full[s], C::TILE);
        }
        tma_load_3d(sq, &tq, dirty ? raw : &q_full[s], 0, seq.start + row, h * (D / 64));
        tma_load_3d(sdo, &tdo, dirty ? raw : &do_full[s], 0, seq.start + row, h * (D / 64));
      }
      const int64_t at = (int64_t)h * a.n + seq.start + row;
      float* l = sL + s * 2 * AM_T;
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int t = u * 32 + lane;
        const float lse = row + t < seq.len ? a.lse[at + t] : -INFINITY;
        // a query that sees nothing (lse -inf) or lies past the end: probability 0
        l[t] = lse == -INFINITY ? -INFINITY : fmaf(lse, -1.4426950408889634f, P_SHIFT);
        l[AM_T + t] = row + t < seq.len ? a.dvec[at + t] * -P_BACK : 0.f;
      }
      if (dirty) {
        ok = warp_wait(raw, raw_phase, err);
        if (!ok) break;
        raw_phase ^= 1;
        attn_zero_rows<D / 64>(sq, bad);
        attn_zero_rows<D / 64>(sdo, bad);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) {
          mbar_arrive(&q_full[s]);
          mbar_arrive(&do_full[s]);
        }
      }
      mbar_arrive(&q_full[s]);
      issued = n + 1;
    }
    if (!ok && lane == 0) {  // a wait ran out: let the copies in flight land before the CTA goes
      mbar_wait(kv_full, 0, nullptr, 100000000ull);
      for (int n = max(0, issued - C::ST); n < issued; ++n) {
        mbar_wait(&q_full[n % C::ST], (n / C::ST) & 1, nullptr, 100000000ull);
        mbar_wait(&do_full[n % C::ST], (n / C::ST) & 1, nullptr, 100000000ull);
      }
    }
  } else if (warp == 8) {
    // ---- MMA ----
    if (lane == 0 && steps > 0) {
      constexpr uint32_t id_s = umma_idesc_f16(IS_BF16, 128, AM_T, false);
      constexpr uint32_t id_o = umma_idesc_f16(IS_BF16, 128, D, true);
      const uint32_t sk = smem_u32(smem), sv = smem_u32(smem + C::OFF_V);
      const uint32_t sq = smem_u32(smem + C::OFF_Q), sdo = smem_u32(smem + C::OFF_DO);
      auto product = [&](uint32_t d, uint32_t A, uint32_t B) {
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          const uint32_t off = (kk >> 2) * BOX + (kk & 3) * 32;
          umma_f16(d, umma_desc_k_sw128(A + off), umma_desc_k_sw128(B + off), id_s, kk > 0);
        }
      };
      auto gather = [&](uint32_t d, uint32_t A, uint32_t B, bool more) {  // d += A^T-in-TMEM . B
#pragma unroll
        for (int kk = 0; kk < AM_T / 16; ++kk)
          umma_f16_ts(d, A + a_col(kk), umma_desc_mn_sw128(B + kk * 2048, BOX, 1024), id_o, more || kk > 0);
      };
      bool ok = mbar_wait(kv_full, 0, err) && mbar_wait(&q_full[0], 0, err);
      if (ok) {
        tc_fence_after();
        product(tmem, sk, sq);
        umma_commit(s_full);
        ok = mbar_wait(&do_full[0], 0, err);
      }
      if (ok) {
        tc_fence_after();
        product(tmem + 128, sv, sdo);
        umma_commit(dp_full);
      }
      for (int n = 0; ok && n < steps; ++n) {
        const int s = n % C::ST, s1 = (n + 1) % C::ST;
        const uint32_t ph1 = ((n + 1) / C::ST) & 1;
        ok = mbar_wait(p_full, n & 1, err);
        if (!ok) break;
        tc_fence_after();
        gather(tmem + 256, tmem, sdo + s * C::TILE, n > 0);  // dV += P^T dO
        if (n + 1 < steps) {
          ok = mbar_wait(&q_full[s1], ph1, err);
          if (!ok) break;
          tc_fence_after();
          product(tmem, sk, sq + s1 * C::TILE);
          umma_commit(s_full);
        }
        ok = mbar_wait(ds_full, n & 1, err);
        if (!ok) break;
        tc_fence_after();
        gather(tmem + 384, tmem + 128, sq + s * C::TILE, n > 0);  // dK += dS^T Q
        umma_commit(&q_empty[s]);
        if (n + 1 < steps) {
          ok = mbar_wait(&do_full[s1], ph1, err);
          if (!ok) break;
          tc_fence_after();
          product(tmem + 128, sv, sdo + s1 * C::TILE);
          umma_commit(dp_full);
        } else {
          umma_commit(out_full);
        }
      }
      if (!ok) {
        umma_commit(drain);
        mbar_wait(drain, 0, nullptr, 100000000ull);
      }
    }
  } else {
    // ---- softmax ----
    const int half = warp >> 2, r = (warp & 3) * 32 + lane, key = k0 + r;
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool live = key < seq.len;
    const int2 range = live ? attn_key_range(seq, key) : make_int2(0, 0);
    BwdConst c = bwd_const<MODE>(a, h0);
    bool ok = true;
    for (int n = 0; n < steps; ++n) {
      const int s = n % C::ST, j = tb.first + n % ntile, i0 = j * AM_T + half * HC;
      if ((MODE & 2) != 0 && n > 0 && n % ntile == 0) c = bwd_const<MODE>(a, h0 + n / ntile);
      const bool masked = j < tb.ffirst || j >= tb.fend;
      const int lo = range.x - i0, hi = range.y - i0;
      ok = warp_wait(s_full, n & 1, err);
      if (ok) ok = warp_wait(&q_full[s], (n / C::ST) & 1, err);  // -lse2 and -Dvec are visible
      if (!ok) break;
      tc_fence_after();
      const float* nl = sL + s * 2 * AM_T + half * HC;
      const uint32_t ts = lane_base + half * HC;
      uint32_t x[HC], dp[HC];
      tmem_ld32_nw(ts, x);
      tmem_ld32_nw(ts + 32, x + 32);
      tmem_wait_ld();
      uint32_t p16[HC / 2];
      if (masked) bwd_probs<T, MODE, true, true, true>(x, p16, c, nl, 0.f, (float)(key - i0), lo, hi);
      else bwd_probs<T, MODE, false, true, true>(x, p16, c, nl, 0.f, (float)(key - i0), 0, 0);
      tmem_st32(ts, reinterpret_cast<const float*>(p16));
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(p_full);
      ok = warp_wait(dp_full, n & 1, err);
      if (!ok) break;
      tc_fence_after();
      tmem_ld32_nw(ts + 128, dp);
      tmem_ld32_nw(ts + 160, dp + 32);
      tmem_wait_ld();
      float w[32];
      if (masked) bwd_ds<T, true, true>(x, dp, w, P_BACK, nl + AM_T, 0.f, lo, hi);
      else bwd_ds<T, false, true>(x, dp, w, P_BACK, nl + AM_T, 0.f, 0, 0);
      tmem_st32(ts + 128, w);
      tmem_wait_st();
      tc_fence_before();
      mbar_arrive(ds_full);
    }
    if (ok && steps > 0) {
      ok = warp_wait(out_full, 0, err);
      tc_fence_after();
    }
    if (ok) {
      const int64_t at = ((int64_t)(seq.start + key) * a.HKV + kvh) * D + half * (D / 2);
      const int64_t plane = (int64_t)a.n * a.HKV * D;
#pragma unroll 1
      for (int u = 0; u < D / 32; ++u) {  // dV's columns, then dK's
        const bool is_k = u >= D / 64;
        const int col = (is_k ? u - D / 64 : u) * 32;
        const float sc = is_k ? a.scale : P_BACK;
        float v[32];
        if (steps > 0) {
          tmem_ld32(lane_base + (is_k ? 384 : 256) + half * (D / 2) + col, v);
        } else {
#pragma unroll
          for (int e = 0; e < 32; ++e) v[e] = 0.f;
        }
        if (!live) continue;
        if (a.splits == 1) {
          store_row16<T>(reinterpret_cast<T*>(is_k ? a.dk : a.dv) + at + col, v, sc);
        } else {
          float4* dst = reinterpret_cast<float4*>(a.parts + (2 * split + (is_k ? 0 : 1)) * plane + at + col);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            dst[e] = make_float4(v[4 * e] * sc, v[4 * e + 1] * sc, v[4 * e + 2] * sc, v[4 * e + 3] * sc);
        }
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dk / dv of every row of a sequence: the splits' partials added in split order, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) attn_mod_sum_kernel(const AttnModArgs a, int D) {
  pdl_enter();
  const int64_t plane = (int64_t)a.n * a.HKV * D;
  const int64_t have = (int64_t)(a.cu_seqlens[a.B] - a.cu_seqlens[0]) * a.HKV * D;
  const int64_t first = (int64_t)a.cu_seqlens[0] * a.HKV * D;
  const int64_t i = (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * 4;
  if (i >= have) return;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int p = 0; p < a.splits; ++p) {
      const float4 v = *reinterpret_cast<const float4*>(a.parts + (2 * p + which) * plane + first + i);
      s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
    }
    T* dst = reinterpret_cast<T*>(which == 0 ? a.dk : a.dv) + first + i;
    *reinterpret_cast<uint2*>(dst) = make_uint2(pack_t2<T>(s.x, s.y), pack_t2<T>(s.z, s.w));
  }
}

// How many CTAs share a KV head's query heads: as few as keep the longest CTA (a key block that
// every query tile sees) under half of an SM's share of all tiles, because each split costs a
// write and a read of fp32 dk and dv; a divisor of the group. (8,192 tokens, 12 / 2 heads: 3 of the
// 6 heads per CTA.)
int dkv_splits(const AttnModArgs& a) {
  const int group = a.HQ / a.HKV;
  const double tiles = (double)cdiv(a.max_len, AM_T);
  const double reach = a.window > 0 ? (a.causal ? 1.0 : 2.0) * a.window / AM_T + 1 : 1e30;
  const double longest = tiles < reach ? tiles : reach;               // query tiles per head and block
  const double mean = a.causal && longest == tiles ? tiles / 2 : longest;
  const double share = (double)cdiv(a.n, AM_T) * a.HQ * mean / sm_count();
  for (int s = 1; s < group; ++s)
    if (group % s == 0 && (group / s) * longest <= 0.5 * share) return s;
  return group;
}

template <typename T, int D, int MODE>
int launch_bwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mdo,
               const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  static unsigned long long done_q = 0, done_kv = 0;
  auto kq = attn_mod_dq_kernel<T, D, MODE>;
  auto kkv = attn_mod_dkv_kernel<T, D, MODE>;
  int st = attn_smem_limit(reinterpret_cast<const void*>(kq), DqCfg<D>::SMEM, &done_q);
  if (st == QL_STATUS_OK) st = attn_smem_limit(reinterpret_cast<const void*>(kkv), DkvCfg<D>::SMEM, &done_kv);
  if (st != QL_STATUS_OK) return st;
  const unsigned tiles = (unsigned)cdiv(a.max_len, AM_T);
  int* err = status_word();
  launch_k(kq, dim3((unsigned)(a.HQ * a.B), tiles), dim3(BWD_THREADS), DqCfg<D>::SMEM, s, mq, mdo, mk,
           mv, a, err);
  launch_k(kkv, dim3((unsigned)(a.HKV * a.splits * a.B), tiles), dim3(BWD_THREADS), DkvCfg<D>::SMEM, s,
           mq, mdo, mk, mv, a, err);
  if (a.splits > 1)
    launch_k(attn_mod_sum_kernel<T>, dim3((unsigned)cdiv((int64_t)a.n * a.HKV * (D / 4), 256)), dim3(256),
             0, s, a, D);
  return launched(a.splits > 1 ? 3 : 2);
}

template <typename T, int D>
int dispatch_bwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mdo,
                 const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  switch (attn_mode(a)) {
    case 0: return launch_bwd<T, D, 0>(a, mq, mdo, mk, mv, s);
    case 1: return launch_bwd<T, D, 1>(a, mq, mdo, mk, mv, s);
    case 2: return launch_bwd<T, D, 2>(a, mq, mdo, mk, mv, s);
    default: return launch_bwd<T, D, 3>(a, mq, mdo, mk, mv, s);
  }
}

int64_t dvec_floats(const AttnModArgs& a) { return ((int64_t)a.HQ * a.n + 3) / 4 * 4; }

}  // namespace

int64_t attn_mod_bwd_workspace(const ql_attn_mod_args& m) {
  AttnModArgs a;
  if (attn_mod_check(m, a) != QL_STATUS_OK) return 0;
  const int splits = dkv_splits(a);
  return dvec_floats(a) + (splits > 1 ? 2 * (int64_t)splits * a.n * a.HKV * m.D : 0);
}

int attn_mod_bwd(const ql_attn_mod_args& m, cudaStream_t s) {
  AttnModArgs a;
  int st = attn_mod_check(m, a);
  if (st != QL_STATUS_OK) return st;
  if (m.n == 0 || m.B == 0 || m.max_len == 0) return QL_STATUS_OK;
  if (m.dout == nullptr || m.dq == nullptr || m.dk == nullptr || m.dv == nullptr ||
      ((reinterpret_cast<uintptr_t>(m.dout) | reinterpret_cast<uintptr_t>(m.dq) |
        reinterpret_cast<uintptr_t>(m.dk) | reinterpret_cast<uintptr_t>(m.dv) |
        reinterpret_cast<uintptr_t>(m.workspace)) & 15))
    return QL_STATUS_BAD_ARG;
  a.splits = dkv_splits(a);
  if (m.workspace == nullptr || m.workspace_floats < attn_mod_bwd_workspace(m)) return QL_STATUS_BAD_ARG;
  a.dout = m.dout;
  a.dq = m.dq;
  a.dk = m.dk;
  a.dv = m.dv;
  a.dvec = m.workspace;
  a.parts = m.workspace + dvec_floats(a);
  ProfScope prof(PK_ATTN_BWD, 0, 0, s);
  if (m.doc_ids != nullptr) {
    st = attn_doc_ranges(m.doc_ids, m.cu_seqlens, m.B, m.n, reinterpret_cast<int2*>(m.ranges), s);
    if (st != QL_STATUS_OK) return st;
  }
  const bool bf = m.dtype == QL_BF16;
  CUtensorMap mq, mdo, mk, mv;
  if (attn_head_map(&mq, m.q, m.n, m.HQ, m.D, m.ldq, bf) != QL_STATUS_OK ||
      attn_head_map(&mdo, m.dout, m.n, m.HQ, m.D, (int64_t)m.HQ * m.D, bf) != QL_STATUS_OK ||
      attn_head_map(&mk, m.k, m.n, m.HKV, m.D, m.ldk, bf) != QL_STATUS_OK ||
      attn_head_map(&mv, m.v, m.n, m.HKV, m.D, m.ldv, bf) != QL_STATUS_OK)
    return QL_STATUS_CUDA;
  if (m.D == 128) return bf ? dispatch_bwd<__nv_bfloat16, 128>(a, mq, mdo, mk, mv, s)
                            : dispatch_bwd<__half, 128>(a, mq, mdo, mk, mv, s);
  return bf ? dispatch_bwd<__nv_bfloat16, 64>(a, mq, mdo, mk, mv, s)
            : dispatch_bwd<__half, 64>(a, mq, mdo, mk, mv, s);
}

}  // namespace ql
