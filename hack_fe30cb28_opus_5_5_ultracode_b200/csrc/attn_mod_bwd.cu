// Attention backward with modified scores and masks on the 5th-generation tensor cores (head dims
// 64 and 128): see attn_mod.cuh for the score and the masks. With y the score in log2 units,
//   P = 2^(y - lse2),  dP = dO V^T,  dS = P (dP - Dvec) (1 - tanh^2),
//   dQ = scale dS K,   dK = scale dS^T Q,   dV = P^T dO,   Dvec = rowsum(dO * O) = rowsum(P * dP).
//
// Two launches of one kernel, each recomputing P: the first sums dQ over the keys of a query tile,
// the second dK and dV over the queries of a key block. One kernel for all three would need 5
// products where these need 8, but dQ would have to be summed by fp32 reductions in L2 (64 KB of them
// per 128 x 128 tile); here every sum stays in tensor memory, the result is bit-identical from run to
// run, and the gradients leave in 16 bits with no fp32 buffer to zero and convert.
//
// Both roles keep two 128-row tiles X, Y of their own rows in shared memory and stream two tiles U, W:
//             X    Y    U    W    S         dP          acc1        acc2
//   dQ        Q    dO   K    V    Q K^T     dO V^T      P K         dS K
//   dK, dV    K    V    Q    dO   K Q^T     V dO^T      P^T dO      dS^T Q
// S is read into registers at once, so the next step's S is formed while this one's P is; P and dS go,
// as 16-bit values, into the tensor-memory columns that dP leaves when it has been read (each thread
// 16 + 16 of its own 32 columns) and are the A operand of acc1 and acc2. The tensor core's acc1, acc2
// and next dP then run beside the next step's P. (With P in S's columns the next S had to wait for
// acc1, and 8,192 causal tokens of 12 + 2 heads took 5% longer.) Sixteen softmax warps, four threads
// per TMEM lane with 32 of the 128 columns each (no row reduction: the forward's lse is known).
//
// That shape takes 624 us for both launches (forward: 160): eight products at 1,320 TFLOP/s, near what
// the tensor cores sustain under the board's power limit. Twice the softmax's exponentials ride along.
//
// Why the dQ role needs P K: Dvec from the forward's 16-bit output is off by the output's rounding,
// and that error enters a whole row of dS with one sign - dQ was up to 1.9 times as far from the
// 64-bit gradient as its own rounding, dK likewise. So the dQ role starts from that Dvec, sums the row
// r = sum P (dP - Dvec) in fp32 (zero for an exact Dvec), and puts it right at the end:
// dQ = scale (dS K - r P K); the second launch reads Dvec + r. P and dS are rounded to the input
// type for the products, in two parts where few terms are summed (PARTS_ROWS); every sum is fp32. An fp16
// dS above 65,504 is infinite, also where scale dS would not be.
#include "attn_mod.cuh"
#include "profile.h"

namespace ql {

namespace {

constexpr int BWD_SOFTMAX = 512;              // softmax threads: four per TMEM lane
constexpr int BWD_THREADS = BWD_SOFTMAX + 64;
constexpr int BOX = AM_T * 128;               // a 128-row x 64-column box
constexpr int HC = 32;                        // columns per softmax thread

// In a tile none of whose rows sees more than so many others, P and dS take part in the products as two
// 16-bit numbers each (`parts`), their roundings and the roundings of what those leave: where few terms make
// up a gradient the errors of single roundings do not average out, and one short batch in 12 had a dQ or
// dK more than 1.5 times as far from the 64-bit one as its own rounding (in two parts none of 109). The
// rule looks at the tile's own mask, so a sequence has the same gradients whatever it is packed with. The
// second parts lie in S's columns, and the next S waits for their products. Both launches, single
// against two parts, us: 64 x 60 tokens of 12 + 2 heads 101 / 113, 4 x 300 in documents of 90 28 / 33,
// 8,192 with a window of 100 118 / 150, 24 k of 28 + 4 heads in documents of 90 610 / 785. Rows that do without
// pay for the choice: 8,192 causal tokens 607 / 624 (the softmax warps have no register left).
constexpr int PARTS_ROWS = 256;

// Two values as 16-bit numbers: their roundings, or (REST) the roundings of what those leave
template <typename T, bool REST>
__device__ __forceinline__ float part_t2(float a, float b) {
  uint32_t h = pack_t2<T>(a, b);
  if constexpr (REST) {
    const T* v = reinterpret_cast<const T*>(&h);
    h = pack_t2<T>(a - to_f<T>(v[0]), b - to_f<T>(v[1]));
  }
  return __uint_as_float(h);
}

// The second parts of 32 values to 16 columns of tensor memory (tmem_wait_st() before they are read)
template <typename T>
__device__ __forceinline__ void store_second(const uint32_t* x, uint32_t taddr) {
  float l[HC / 2];
#pragma unroll
  for (int e = 0; e < HC / 2; ++e) l[e] = part_t2<T, true>(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
  tmem_st16(taddr, l);
}

struct BwdConst {
  float sl2, u, cap2;
  float slope;  // the distance bias's, in units of raw products, or (capped) of log2
  TanhShort ts;
};

// 16 raw scores of one TMEM lane into the factors of dS (f, in place of x): probabilities times the
// cap's derivative, which comes as tanh^2 - 1: f of a capped score has the other sign until the
// gradients' last scaling. p16: the probabilities themselves as 16-bit pairs, where they are not f (a capped
// score of the dK / dV role). form: tanh_form of the warp's
// scores. neg_lse: -lse2 by column (PER_COL, from shared memory) or
// one value. Columns whose bit in seen is 0 give 0. dist0: row index minus the first column's, for
// the distance bias. p: plain probabilities where the caller needs them beside f (a capped score of
// the dQ role). With parts, p16's second part goes to the tensor-memory columns at rest.
template <typename T, int MODE, bool MASKED, bool PER_COL>
__device__ __forceinline__ void bwd_probs(uint32_t* x, float* p16, float* p, const BwdConst& c, int form,
                                          const float* neg_lse, float neg_lse_row, float dist0, uint32_t seen, uint32_t rest,
                                          bool parts) {
  uint64_t y[8], bend[8];
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    y[e] = y[e + 1] = pk2(neg_lse_row, neg_lse_row);
    if constexpr (PER_COL) {
      const float4 l = *reinterpret_cast<const float4*>(neg_lse + 2 * e);
      y[e] = pk2(l.x, l.y);
      y[e + 1] = pk2(l.z, l.w);
    }
  }
  if constexpr ((MODE & 1) != 0) {
    uint64_t th[8];
    if (form == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) th[e] = pair_of(x + 2 * e);
      tanh_short2<8>(th, c.ts);
    } else if (form == 1) {
#pragma unroll
      for (int e = 0; e < 8; ++e) th[e] = mul2(pair_of(x + 2 * e), pk2(c.u, c.u));
      tanh_poly2<8>(th);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        th[e] = pk2(tanhf(__uint_as_float(x[2 * e]) * c.u), tanhf(__uint_as_float(x[2 * e + 1]) * c.u));
    }
    // the distance bias in the order of the forward's roundings, so that its lse fits
    if constexpr ((MODE & 2) != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float ta, tb;
        up2(mul2(th[e], pk2(c.cap2, c.cap2)), ta, tb);
        y[e] = add2(pk2(fmaf(fabsf(dist0 - (float)(2 * e)), -c.slope, ta), fmaf(fabsf(dist0 - (float)(2 * e + 1)), -c.slope, tb)), y[e]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = fma2(th[e], pk2(c.cap2, c.cap2), y[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) bend[e] = fma2(th[e], th[e], pk2(-1.f, -1.f));  // tanh^2 - 1: sign below
  } else {
    if constexpr ((MODE & 2) != 0) {
#pragma unroll
      for (int k = 0; k < 16; ++k) x[k] = __float_as_uint(fmaf(fabsf(dist0 - (float)k), -c.slope, __uint_as_float(x[k])));
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = fma2(pair_of(x + 2 * e), pk2(c.sl2, c.sl2), y[e]);
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int k = 2 * e;
    ex2_2<1>(y + e);
    float pa, pb, fa, fb;
    up2(y[e], pa, pb);
    if constexpr (MASKED) {
      if (!(seen >> k & 1)) pa = 0.f;
      if (!(seen >> (k + 1) & 1)) pb = 0.f;
    }
    fa = pa;
    fb = pb;
    if constexpr ((MODE & 1) != 0) {
      up2(mul2(pk2(pa, pb), bend[e]), fa, fb);
      // a masked score may be anything, infinities and NaN too: its factor is 0
      if (MASKED && pa == 0.f) fa = 0.f;
      if (MASKED && pb == 0.f) fb = 0.f;
      if constexpr (PER_COL) {
        y[e] = pk2(pa, pb);
        p16[e] = part_t2<T, false>(pa, pb);
      } else {
        p[k] = pa;
        p[k + 1] = pb;
      }
    }
    x[k] = __float_as_uint(fa);
    x[k + 1] = __float_as_uint(fb);
  }
  if constexpr ((MODE & 1) != 0 && PER_COL) {
    if (parts) {
      float l[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float pa, pb;
        up2(y[e], pa, pb);
        l[e] = part_t2<T, true>(pa, pb);
      }
      tmem_st8(rest, l);
    }
  }
}

// dS = f (dP dscale - Dvec'), in place of f and as 16-bit pairs; neg_d: -Dvec' by column or one value. The dQ
// role also gets sum p (dP - Dvec) of its columns.
template <typename T, int MODE, bool MASKED, bool PER_COL, int N>
__device__ __forceinline__ float bwd_ds(uint32_t* f, const float* p, const uint32_t* dp, float* ds16,
                                        float dscale, const float* neg_d, float neg_d_row, uint32_t seen) {
  const uint64_t row2 = pk2(neg_d_row, neg_d_row), ds2 = pk2(dscale, dscale);
  uint64_t sum[2] = {0, 0};  // pairs of +0.f
#pragma unroll
  for (int i = 0; i < N; i += 16) {
    uint64_t g[8];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint64_t nd[2] = {row2, row2};
      if constexpr (PER_COL) {
        const float4 l = *reinterpret_cast<const float4*>(neg_d + i + 2 * e);
        nd[0] = pk2(l.x, l.y);
        nd[1] = pk2(l.z, l.w);
      }
      g[e] = fma2(pair_of(dp + i + 2 * e), ds2, nd[0]);
      g[e + 1] = fma2(pair_of(dp + i + 2 * e + 2), ds2, nd[1]);
    }
    if constexpr (MASKED) {  // 0 times whatever a masked place holds
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int k = i + 2 * e;
        float a, b;
        up2(g[e], a, b);
        g[e] = pk2(seen >> k & 1 ? a : 0.f, seen >> (k + 1) & 1 ? b : 0.f);
      }
    }
    if constexpr (!PER_COL && (MODE & 1) != 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e & 1] = fma2(g[e], pk2(p[i + 2 * e], p[i + 2 * e + 1]), sum[e & 1]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) g[e] = mul2(g[e], pair_of(f + i + 2 * e));
    if constexpr (!PER_COL && (MODE & 1) == 0) {
#pragma unroll
      for (int e = 0; e < 8; ++e) sum[e & 1] = add2(sum[e & 1], g[e]);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float a, b;
      up2(g[e], a, b);
      unpair(g[e], f + i + 2 * e);
      ds16[i / 2 + e] = part_t2<T, false>(a, b);
    }
  }
  float a, b;
  up2(add2(sum[0], sum[1]), a, b);
  return a + b;
}

template <int MODE>
__device__ __forceinline__ BwdConst bwd_const(const AttnModArgs& a, int h) {
  BwdConst c;
  c.sl2 = a.scale * 1.4426950408889634f;
  c.u = (MODE & 1) != 0 ? a.scale / a.softcap : 0.f;
  c.cap2 = a.softcap * 1.4426950408889634f;
  if constexpr ((MODE & 1) != 0) c.ts = tanh_short(c.u, 1.f);
  c.slope = (MODE & 2) == 0 ? 0.f : (MODE & 1) != 0 ? a.slopes[h] * 1.4426950408889634f : a.slopes[h] / a.scale;
  return c;
}

// 16 values as 16-bit chunks 2 u and 2 u + 1 of the row
template <typename T, int W>
__device__ __forceinline__ void stage16(uint8_t* stage, int row, int u, const float* v) {
#pragma unroll
  for (int c = 0; c < 2; ++c)
    *reinterpret_cast<uint4*>(stage_at<W>(stage, row, 2 * u + c)) =
        make_uint4(pack_t2<T>(v[8 * c], v[8 * c + 1]), pack_t2<T>(v[8 * c + 2], v[8 * c + 3]),
                   pack_t2<T>(v[8 * c + 4], v[8 * c + 5]), pack_t2<T>(v[8 * c + 6], v[8 * c + 7]));
}

template <int D>
struct BwdCfg {
  static constexpr int TILE = AM_T * D * 2;
  // U is held from its step's S to its acc2, W (dO of the dK / dV role, V of the other) not as long:
  // with pairs of stages a tile's copy left one step's time before its S was due, and S waited for it
  static constexpr int UST = 3, WST = 2;
  static constexpr int OFF_Y = TILE, OFF_U = 2 * TILE, OFF_W = OFF_U + UST * TILE;
  static constexpr int OFF_L = OFF_W + WST * TILE;          // [2][2][128] fp32: -lse2, -Dvec by column;
                                                            // dQ role: [4][128] a row's partial sums
  static constexpr int OFF_D = OFF_L + 4 * AM_T * 4;        // dQ role: [128] Dvec of the 16-bit output
  static constexpr int OFF_BAR = OFF_D + AM_T * 4;
  static constexpr int SMEM = OFF_BAR + 512;
};

// One CTA per (128-row tile, head, sequence): query tiles of every query head for dQ; for dK and dV key
// blocks of every KV head, times a.splits CTAs that share its query heads.
// fp16, dK / dV: P is kept as 2^8 P (at most 2^8 where P is 1), so that the small probabilities of
// long rows stay normal numbers; dS and dV take the factor back in fp32.
// TMEM: S, then the second parts of P and dS [0, 128), dP, then P and dS [128, 256), acc1 [256, 256 + D),
// acc2 [384, 384 + D).
template <typename T, int D, int MODE, bool DKV>
__global__ void __launch_bounds__(BWD_THREADS, 1)
    attn_mod_bwd_kernel(const __grid_constant__ CUtensorMap tx, const __grid_constant__ CUtensorMap ty,
                        const __grid_constant__ CUtensorMap tu, const __grid_constant__ CUtensorMap tw,
                        const AttnModArgs a, int* err) {
  using C = BwdCfg<D>;
  constexpr bool IS_BF16 = std::is_same<T, __nv_bfloat16>::value;
  constexpr float SIGN = (MODE & 1) != 0 ? -1.f : 1.f;  // of f, see bwd_probs
  constexpr float P_SHIFT = !DKV || IS_BF16 ? 0.f : 8.f, P_BACK = !DKV || IS_BF16 ? 1.f : 1.f / 256.f;
  pdl_enter();
  extern __shared__ __align__(1024) uint8_t smem[];  // no static shared memory: the base is aligned
  float* sL = reinterpret_cast<float*>(smem + C::OFF_L);
  float* sR = sL;
  float* sD = reinterpret_cast<float*>(smem + C::OFF_D);
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + C::OFF_BAR);
  uint64_t* xy_full = bars;
  uint64_t* s_full = bars + 1;
  uint64_t* dp_full = bars + 2;
  uint64_t* ds_full = bars + 3;  // dS written (all softmax warps)
  uint64_t* out_full = bars + 4;
  uint64_t* drain = bars + 6;
  uint64_t* p_full = bars + 7;   // P written, dP read (all softmax warps)
  uint64_t* s_free = bars + 8;   // S read (all softmax warps)
  uint64_t* l_full = bars + 9;   // [2] -lse2 and -Dvec of a step stored
  uint64_t* l_empty = bars + 11; // [2] and read (all softmax warps)
  uint64_t* u_full = bars + 13;  // [UST]
  uint64_t* u_empty = u_full + C::UST;
  uint64_t* w_full = u_empty + C::UST;  // [WST]
  uint64_t* w_empty = w_full + C::WST;
  uint64_t* raw = w_empty + C::WST;     // [UST + WST] copies whose dead rows are zeroed first
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(raw + C::UST + C::WST);

  const int group = a.HQ / a.HKV;
  const int per_seq = DKV ? a.HKV * a.splits : a.HQ;
  const int b = blockIdx.x / per_seq, part_of_seq = blockIdx.x % per_seq;
  const int kvh = DKV ? part_of_seq / a.splits : part_of_seq / group;
  const int split = DKV ? part_of_seq % a.splits : 0;
  const int g0 = DKV ? group * split / a.splits : 0;    // query heads this CTA runs through
  const int heads = DKV ? group * (split + 1) / a.splits - g0 : 1;
  const int h0 = DKV ? kvh * group + g0 : part_of_seq;
  // the tiles with the most work first (causal: the last queries, the first keys)
  const int r0 = (DKV ? blockIdx.y : gridDim.y - 1 - blockIdx.y) * AM_T;
  const AttnSeq seq = attn_seq(a, b);
  if (r0 >= seq.len) return;  // the whole CTA, before any barrier or TMEM is set up
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  // dQ role: the tile's rows of O and dO for Dvec, eight rows a warp in whole lines (a thread per quarter
  // row, as the softmax has them, took 12,000 cycles to read its way through 128 lines at a time)
  constexpr int LPR = D / 8, RPI = 32 / LPR;  // lanes per row, rows per load
  uint4 ov[8 / RPI], gv[8 / RPI];
  if (!DKV && warp < 16) {
#pragma unroll
    for (int i = 0; i < 8 / RPI; ++i) {
      const int row = r0 + warp * 8 + i * RPI + lane / LPR;
      const int64_t at = ((int64_t)(seq.start + row) * a.HQ + h0) * D + (lane % LPR) * 8;
      ov[i] = gv[i] = make_uint4(0u, 0u, 0u, 0u);
      if (row < seq.len) {
        ov[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.out) + at);
        gv[i] = *reinterpret_cast<const uint4*>(reinterpret_cast<const T*>(a.dout) + at);
      }
    }
  }
  // the loading warp sets the barriers up while the others allocate and look at the mask
  if (warp == 17 && lane == 0) {
    mbar_init(xy_full, 1);
    mbar_init(s_full, 1);
    mbar_init(dp_full, 1);
    mbar_init(ds_full, BWD_SOFTMAX / 32);
    mbar_init(p_full, BWD_SOFTMAX / 32);
    mbar_init(s_free, BWD_SOFTMAX / 32);
    mbar_init(out_full, 1);
    for (int k = 0; k < C::UST + C::WST; ++k) mbar_init(&raw[k], 1);
    mbar_init(drain, 1);
    for (int s = 0; s < 2; ++s) {
      mbar_init(&l_full[s], 1);
      mbar_init(&l_empty[s], BWD_SOFTMAX / 32);
    }
    for (int s = 0; s < C::UST; ++s) {
      mbar_init(&u_full[s], 1);
      mbar_init(&u_empty[s], 1);
    }
    for (int s = 0; s < C::WST; ++s) {
      mbar_init(&w_full[s], 1);
      mbar_init(&w_empty[s], 1);
    }
    fence_barrier_init();
  }
  if (warp == 16) tmem_alloc(tmem_slot, 512);
  const AttnBlocks tb = DKV ? attn_key_blocks(seq, r0) : attn_tile_blocks(seq, r0);
  const int ntile = tb.end - tb.first, steps = uniform(ntile * heads);
  if (warp == 17 && lane == 0 && steps > 0) {
    const int zx = (DKV ? kvh : h0) * (D / 64);
    mbar_arrive_expect_tx(xy_full, 2 * C::TILE);
    tma_load_3d(smem, &tx, xy_full, 0, seq.start + r0, zx);
    tma_load_3d(smem + C::OFF_Y, &ty, xy_full, 0, seq.start + r0, zx);
  }
  if (!DKV && warp < 16) {
#pragma unroll
    for (int i = 0; i < 8 / RPI; ++i) {
      const T* ot = reinterpret_cast<const T*>(&ov[i]);
      const T* gt = reinterpret_cast<const T*>(&gv[i]);
      float dot = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) dot = fmaf(to_f<T>(ot[e]), to_f<T>(gt[e]), dot);
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, o);
      if (lane % LPR == 0) sD[warp * 8 + i * RPI + lane / LPR] = dot;
    }
  }
  int sees = 0;  // rows that row threadIdx.x of the tile sees
  if (warp < 4 && r0 + (int)threadIdx.x < seq.len) {
    const int2 range = DKV ? attn_key_range(seq, r0 + threadIdx.x) : attn_row_range(seq, r0 + threadIdx.x);
    sees = range.y - range.x;
  }
  tc_fence_before();
  const bool parts = uniform(__syncthreads_or(sees > PARTS_ROWS)) == 0;
  tc_fence_after();
  const uint32_t tmem = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  if (warp == 17) {
    // ---- loads ----
    // U two steps ahead, W one. Tiles with rows that belong to no query or key land on a raw barrier and
    // are handed on when those rows have been zeroed, before any product reads them; what the waits
    // for room need is always handed on before them.
    bool ok = true;
    int un = 0, wn = 0;        // tiles sent for
    uint32_t raw_phase = 0;    // of raw[0 .. UST + WST)
    auto row_of = [&](int n) { return (tb.first + (DKV ? n % ntile : n)) * AM_T; };
    auto send = [&](int n, bool is_w, const DeadRows& d) {
      const int s = is_w ? n % C::WST : n % C::UST;
      const int z = (DKV ? h0 + n / ntile : kvh) * (D / 64);
      uint64_t* bar = d.any ? &raw[is_w ? C::UST + s : s] : is_w ? &w_full[s] : &u_full[s];
      if (lane == 0) {
        mbar_arrive_expect_tx(bar, C::TILE);
        tma_load_3d(smem + (is_w ? C::OFF_W : C::OFF_U) + s * C::TILE, is_w ? &tw : &tu, bar, 0,
                    seq.start + row_of(n), z);
      }
      if (is_w) wn = n + 1;
      else un = n + 1;
    };
    auto clean = [&](int n, bool is_w, const DeadRows& d) {
      if (!d.any) return true;
      const int s = is_w ? n % C::WST : n % C::UST, k = is_w ? C::UST + s : s;
      if (!warp_wait(&raw[k], (raw_phase >> k) & 1, err)) return false;
      raw_phase ^= 1u << k;
      attn_zero_rows<D / 64>(smem + (is_w ? C::OFF_W : C::OFF_U) + s * C::TILE, d);
      fence_proxy_async_smem();
      warp_arrive(is_w ? &w_full[s] : &u_full[s]);
      return true;
    };
    DeadRows d0{{0u, 0u, 0u, 0u}, false}, d1 = d0, d2 = d0;  // of steps n, n + 1, n + 2
    if (steps > 0) {
      d0 = attn_dead_rows(seq, row_of(0));
      send(0, false, d0);
      send(0, true, d0);
    }
    if (steps > 1) {
      d1 = attn_dead_rows(seq, row_of(1));
      send(1, false, d1);
      send(1, true, d1);
    }
    for (int n = 0; ok && n < steps; ++n) {
      float l[4], dv[4];
      if constexpr (DKV) {
        const int row = row_of(n);
        const int64_t at = (int64_t)(h0 + n / ntile) * a.n + seq.start + row;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t = u * 32 + lane;
          l[u] = row + t < seq.len ? a.lse[at + t] : -INFINITY;
          dv[u] = row + t < seq.len ? a.dvec[at + t] : 0.f;
        }
      }
      ok = clean(n, false, d0) && clean(n, true, d0);
      if constexpr (DKV) {
        if (ok && n >= 2) ok = warp_wait(&l_empty[n & 1], ((n >> 1) - 1) & 1, err);
        if (!ok) break;
        float* sl = sL + (n & 1) * 2 * AM_T;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
          const int t = u * 32 + lane;
          // a query that sees nothing (lse -inf) or lies past the end: probability 0
          sl[t] = l[u] == -INFINITY ? -INFINITY : fmaf(l[u], -1.4426950408889634f, P_SHIFT);
          sl[AM_T + t] = dv[u] * -P_BACK;
        }
        warp_arrive(&l_full[n & 1]);
      }
      if (n > 0 && n + 1 < steps) {
        ok = ok && warp_wait(&w_empty[(n + 1) % C::WST], ((n + 1) / C::WST - 1) & 1, err);
        if (ok) send(n + 1, true, d1);
      }
      if (n + 2 < steps) {
        d2 = attn_dead_rows(seq, row_of(n + 2));
        if (n + 2 >= C::UST) ok = ok && warp_wait(&u_empty[(n + 2) % C::UST], ((n + 2) / C::UST - 1) & 1, err);
        if (ok) send(n + 2, false, d2);
      }
      d0 = d1;
      d1 = d2;
    }
    if (!ok && lane == 0) {  // a wait ran out: let the copies in flight land before the CTA goes
      mbar_wait(xy_full, 0, nullptr, 100000000ull);
      for (int k = 0; k < C::UST + C::WST; ++k) mbar_wait(&raw[k], (raw_phase >> k) & 1, nullptr, 10000000ull);
      for (int n = max(0, un - C::UST); n < un; ++n)
        mbar_wait(&u_full[n % C::UST], (n / C::UST) & 1, nullptr, 10000000ull);
      for (int n = max(0, wn - C::WST); n < wn; ++n)
        mbar_wait(&w_full[n % C::WST], (n / C::WST) & 1, nullptr, 10000000ull);
    }
  } else if (warp == 16) {
    // ---- MMA ----
    if (steps > 0) {
      constexpr uint32_t id_s = umma_idesc_f16(IS_BF16, 128, AM_T, false);
      constexpr uint32_t id_o = umma_idesc_f16(IS_BF16, 128, D, true);
      constexpr uint32_t TILE16 = C::TILE >> 4;
      const uint32_t sx = desc_lo_k(smem_u32(smem)), sy = sx + TILE16;
      const uint32_t uk = desc_lo_k(smem_u32(smem + C::OFF_U)), um = desc_lo_mn(smem_u32(smem + C::OFF_U), BOX);
      const uint32_t wk = desc_lo_k(smem_u32(smem + C::OFF_W)), wm = desc_lo_mn(smem_u32(smem + C::OFF_W), BOX);
      auto u_landed = [&](int n) { return warp_wait(&u_full[n % C::UST], (n / C::UST) & 1, err); };
      auto w_landed = [&](int n) { return warp_wait(&w_full[n % C::WST], (n / C::WST) & 1, err); };
      auto score = [&](int n) {  // S = X U^T
        tc_fence_after();
        umma_score<D>(tmem, sx, uk + (n % C::UST) * TILE16, id_s);
        warp_commit(s_full);
      };
      auto dprob = [&](int n) {  // dP = Y W^T
        tc_fence_after();
        umma_score<D>(tmem + 128, sy, wk + (n % C::WST) * TILE16, id_s);
        warp_commit(dp_full);
        if (!DKV) warp_commit(&w_empty[n % C::WST]);
      };
      bool ok = warp_wait(xy_full, 0, err) && u_landed(0);
      if (ok) score(0);
      ok = ok && w_landed(0);
      if (ok) dprob(0);
      if (steps > 1 && !parts) {
        ok = ok && u_landed(1) && warp_wait(s_free, 0, err);
        if (ok) score(1);
      }
      // Copies are waited for ahead of the softmax warps: every instruction of this warp takes its turn
      // among those of four of them.
      for (int n = 0; ok && n < steps; ++n) {
        const uint32_t u0 = um + (n % C::UST) * TILE16, w0 = wm + (n % C::WST) * TILE16;
        const bool more = n + 1 < steps;
        ok = warp_wait(p_full, n & 1, err);
        if (!ok) break;
        tc_fence_after();
        umma_gather4(tmem + 256, tmem + 128, DKV ? w0 : u0, id_o, n > 0);
        if (parts) umma_gather4(tmem + 256, tmem, DKV ? w0 : u0, id_o, 1);
        if (DKV) warp_commit(&w_empty[n % C::WST]);
        if (more) ok = w_landed(n + 1);
        ok = ok && warp_wait(ds_full, n & 1, err);
        if (!ok) break;
        tc_fence_after();
        umma_gather4(tmem + 384, tmem + 128 + HC / 2, u0, id_o, n > 0);
        if (parts) {
          umma_gather4(tmem + 384, tmem + HC / 2, u0, id_o, 1);
          if (more) {
            ok = u_landed(n + 1);
            if (!ok) break;
            score(n + 1);
          }
        }
        if (more) dprob(n + 1);
        else warp_commit(out_full);
        warp_commit(&u_empty[n % C::UST]);
        if (n + 2 < steps && !parts) {
          ok = u_landed(n + 2) && warp_wait(s_free, (n + 1) & 1, err);
          if (ok) score(n + 2);
        }
      }
      if (!ok) {  // a wait ran out: the products already issued finish before TMEM is freed
        warp_commit(drain);
        if (lane == 0) mbar_wait(drain, 0, nullptr, 100000000ull);
        __syncwarp();
      }
    }
  } else {
    // ---- softmax ----
    const int part = warp >> 2, r = (warp & 3) * 32 + lane, ri = r0 + r;  // row ri of the sequence
    const uint32_t lane_base = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const bool live = ri < seq.len;
    const int2 range = !live ? make_int2(0, 0) : DKV ? attn_key_range(seq, ri) : attn_row_range(seq, ri);
    BwdConst c = bwd_const<MODE>(a, h0);
    float neg_lse = -INFINITY, neg_d = 0.f, rest = 0.f;
    if constexpr (!DKV) {
      if (range.y > range.x) {  // a row that sees nothing keeps probability 0 and Dvec 0
        neg_lse = a.lse[(int64_t)h0 * a.n + seq.start + ri] * -1.4426950408889634f;
        neg_d = -sD[r];
      }
    }
    bool ok = true;
    const uint32_t ts = lane_base + part * HC;
    for (int n = 0; n < steps; ++n) {
      const int s = n & 1, j = tb.first + (DKV ? n % ntile : n), i0 = j * AM_T + part * HC;
      if (DKV && (MODE & 2) != 0 && n > 0 && n % ntile == 0) c = bwd_const<MODE>(a, h0 + n / ntile);
      const bool masked = j < tb.ffirst || j >= tb.fend;
      const uint32_t seen = masked ? col_mask(range.x - i0, range.y - i0) : 0;
      const float dist0 = (float)(ri - i0);
      ok = warp_wait(s_full, n & 1, err);
      if (DKV && ok) ok = warp_wait(&l_full[s], (n >> 1) & 1, err);  // -lse2 and -Dvec are visible
      if (!ok) break;
      tc_fence_after();
      const float* nl = sL + s * 2 * AM_T + part * HC;
      uint32_t x[HC];
      float w[HC / 2], p[(MODE & 1) != 0 && !DKV ? HC : 1];
      tmem_ld32_nw(ts, x);
      tmem_wait_ld();
      tc_fence_before();
      warp_arrive(s_free);
      int form = 0;
      if constexpr ((MODE & 1) != 0) form = tanh_form<HC>(x, c.u);
#pragma unroll
      for (int g = 0; g < HC; g += 16) {
        float* pg = p + ((MODE & 1) != 0 && !DKV ? g : 0);
        if (masked) bwd_probs<T, MODE, true, DKV>(x + g, w + g / 2, pg, c, form, nl + g, neg_lse, dist0 - g, seen >> g, ts + g / 2, parts);
        else bwd_probs<T, MODE, false, DKV>(x + g, w + g / 2, pg, c, form, nl + g, neg_lse, dist0 - g, 0, ts + g / 2, parts);
      }
      if ((MODE & 1) == 0 || !DKV) {  // acc1 takes f itself
        if (parts) store_second<T>(x, ts);
      }
      ok = warp_wait(dp_full, n & 1, err);
      if (!ok) break;
      tc_fence_after();
      if constexpr ((MODE & 1) != 0 && !DKV) {
        // f and p both live: dP in two halves, or the registers spill (the backward of 8,192 capped
        // tokens then took 945 us, not 724; now 765)
        float ds[HC / 2];
#pragma unroll
        for (int g = 0; g < HC; g += 16) {
          float dh[16];
          tmem_ld16(ts + 128 + g, dh);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            w[g / 2 + e] = part_t2<T, false>(__uint_as_float(x[g + 2 * e]), __uint_as_float(x[g + 2 * e + 1]));
          const uint32_t* du = reinterpret_cast<const uint32_t*>(dh);
          if (masked) rest += bwd_ds<T, MODE, true, DKV, 16>(x + g, p + g, du, ds + g / 2, P_BACK, nl, neg_d, seen >> g);
          else rest += bwd_ds<T, MODE, false, DKV, 16>(x + g, p + g, du, ds + g / 2, P_BACK, nl, neg_d, 0);
        }
        tmem_st16(ts + 128, w);
        tmem_st16(ts + 128 + HC / 2, ds);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(p_full);
      } else {
        uint32_t dp[HC];
        tmem_ld32_nw(ts + 128, dp);
        tmem_wait_ld();
        if constexpr ((MODE & 1) == 0) {
#pragma unroll
          for (int e = 0; e < HC / 2; ++e)
            w[e] = part_t2<T, false>(__uint_as_float(x[2 * e]), __uint_as_float(x[2 * e + 1]));
        }
        tmem_st16(ts + 128, w);
        tmem_wait_st();
        tc_fence_before();
        warp_arrive(p_full);
        if (masked) rest += bwd_ds<T, MODE, true, DKV, HC>(x, p, dp, w, P_BACK, nl + AM_T, neg_d, seen);
        else rest += bwd_ds<T, MODE, false, DKV, HC>(x, p, dp, w, P_BACK, nl + AM_T, neg_d, 0);
        tmem_st16(ts + 128 + HC / 2, w);
      }
      if (parts) store_second<T>(x, ts + HC / 2);
      tmem_wait_st();
      tc_fence_before();
      if (DKV) warp_arrive(&l_empty[s]);
      warp_arrive(ds_full);
    }
    if (ok && steps > 0) {
      ok = warp_wait(out_full, 0, err);
      tc_fence_after();
    }
    // the results leave through X and Y, which every product has read
    constexpr int W = D / 2;          // bytes of a quarter row of 16-bit values
    const int col0 = part * (D / 4);  // this thread's columns
    const int row0 = ri - lane;       // the warp's first row
    uint8_t* stage = smem + warp * 32 * 2 * W;
    if constexpr (!DKV) {
      sR[part * AM_T + r] = rest;
      asm volatile("bar.sync 1, 512;" ::: "memory");
      rest = (sR[r] + sR[AM_T + r]) + (sR[2 * AM_T + r] + sR[3 * AM_T + r]);
      if (ok && live && part == 0) a.dvec[(int64_t)h0 * a.n + seq.start + ri] = rest - neg_d;
      if (ok) {
        const float sc = range.y - range.x == 1 ? 0.f : SIGN * a.scale;  // one key: the softmax is constant
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          float pk[16], v[16];
          if (steps > 0) {
            tmem_ld16(lane_base + 256 + col0 + u * 16, pk);
            tmem_ld16(lane_base + 384 + col0 + u * 16, v);
          }
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = steps > 0 ? (v[e] - rest * pk[e]) * sc : 0.f;
          stage16<T, W>(stage, lane, u, v);
        }
        T* dst = reinterpret_cast<T*>(a.dq) + ((int64_t)(seq.start + row0) * a.HQ + h0) * D + col0;
        stage_flush<W>(stage, reinterpret_cast<uint8_t*>(dst), (int64_t)a.HQ * D * 2, seq.len - row0);
      }
    } else if (ok) {
      const int64_t at = ((int64_t)(seq.start + row0) * a.HKV + kvh) * D + col0;
      const int64_t plane = (int64_t)a.n * a.HKV * D;
#pragma unroll
      for (int is_k = 0; is_k < 2; ++is_k) {
        const float sc = is_k ? SIGN * a.scale : P_BACK;
#pragma unroll
        for (int u = 0; u < D / 64; ++u) {
          float v[16];
          if (steps > 0) tmem_ld16(lane_base + (is_k ? 384 : 256) + col0 + u * 16, v);
#pragma unroll
          for (int e = 0; e < 16; ++e) v[e] = steps > 0 ? v[e] * sc : 0.f;
          if (a.splits == 1) {
            stage16<T, W>(stage, lane, u, v);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e)
              *reinterpret_cast<float4*>(stage_at<2 * W>(stage, lane, 4 * u + e)) =
                  make_float4(v[4 * e], v[4 * e + 1], v[4 * e + 2], v[4 * e + 3]);
          }
        }
        if (a.splits == 1)
          stage_flush<W>(stage, reinterpret_cast<uint8_t*>(reinterpret_cast<T*>(is_k ? a.dk : a.dv) + at),
                         (int64_t)a.HKV * D * 2, seq.len - row0);
        else
          stage_flush<2 * W>(stage, reinterpret_cast<uint8_t*>(a.parts + (2 * split + (is_k ? 0 : 1)) * plane + at),
                             (int64_t)a.HKV * D * 4, seq.len - row0);
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 16) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// dk and dv of every row of a sequence: the splits' partials added in split order, those of two splits
// on their way at a time, rounded once.
template <typename T>
__global__ void __launch_bounds__(256) attn_mod_sum_kernel(const AttnModArgs a, int D) {
  pdl_enter();
  const int64_t plane = (int64_t)a.n * a.HKV * D;
  const int64_t first = (int64_t)a.cu_seqlens[0] * a.HKV * D, end = (int64_t)a.cu_seqlens[a.B] * a.HKV * D;
  const int64_t i = first + (blockIdx.x * (int64_t)blockDim.x + threadIdx.x) * 4;
  if (i >= end) return;
  float4 s[2] = {make_float4(0.f, 0.f, 0.f, 0.f), make_float4(0.f, 0.f, 0.f, 0.f)};  // dk, dv
  for (int p = 0; p < a.splits; p += 2) {
    float4 v[2][2];
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w)
        v[k][w] = p + k < a.splits ? *reinterpret_cast<const float4*>(a.parts + (2 * (p + k) + w) * plane + i)
                                   : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int k = 0; k < 2; ++k)
#pragma unroll
      for (int w = 0; w < 2; ++w)
        s[w].x += v[k][w].x, s[w].y += v[k][w].y, s[w].z += v[k][w].z, s[w].w += v[k][w].w;
  }
#pragma unroll
  for (int w = 0; w < 2; ++w)
    *reinterpret_cast<uint2*>(reinterpret_cast<T*>(w == 0 ? a.dk : a.dv) + i) =
        make_uint2(pack_t2<T>(s[w].x, s[w].y), pack_t2<T>(s[w].z, s[w].w));
}

// How many CTAs share a KV head's query heads: as few as keep the longest CTA (a key block that
// every query tile sees) under this fraction of an SM's share of all tiles, because each split costs a
// write and a read of fp32 dk and dv (8,192 causal tokens, 12 + 2 heads: 3% longer with 0.5 than with 0.8).
constexpr double SPLIT_SHARE = 0.8;
int dkv_splits(const AttnModArgs& a) {
  const int group = a.HQ / a.HKV;
  const double tiles = (double)cdiv(a.max_len, AM_T);
  const double reach = a.window > 0 ? (a.causal ? 1.0 : 2.0) * a.window / AM_T + 1 : 1e30;
  const double longest = tiles < reach ? tiles : reach;               // query tiles per head and block
  const double mean = a.causal && longest == tiles ? tiles / 2 : longest;
  const double share = (double)cdiv(a.n, AM_T) * a.HQ * mean / sm_count();
  for (int s = 1; s < group; ++s)
    if (cdiv(group, s) * longest <= SPLIT_SHARE * share) return s;
  return group;
}

template <typename T, int D, int MODE>
int launch_bwd(const AttnModArgs& a, const CUtensorMap& mq, const CUtensorMap& mdo,
               const CUtensorMap& mk, const CUtensorMap& mv, cudaStream_t s) {
  static std::atomic<unsigned long long> done_q{0}, done_kv{0};
  auto kq = attn_mod_bwd_kernel<T, D, MODE, false>;
  auto kkv = attn_mod_bwd_kernel<T, D, MODE, true>;
  constexpr int smem = BwdCfg<D>::SMEM;
  int st = attn_smem_limit(reinterpret_cast<const void*>(kq), smem, done_q);
  if (st == QL_STATUS_OK) st = attn_smem_limit(reinterpret_cast<const void*>(kkv), smem, done_kv);
  if (st != QL_STATUS_OK) return st;
  const unsigned tiles = (unsigned)cdiv(a.max_len, AM_T);
  int* err = status_word();
  launch_k(kq, dim3((unsigned)(a.HQ * a.B), tiles), dim3(BWD_THREADS), smem, s, mq, mdo, mk, mv, a, err);
  launch_k(kkv, dim3((unsigned)(a.HKV * a.splits * a.B), tiles), dim3(BWD_THREADS), smem, s, mk, mv, mq,
           mdo, a, err);
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

int64_t attn_mod_bwd_workspace(int n, int max_len, int HQ, int HKV, int D, int causal, int window) {
  if (n <= 0 || max_len < 0 || HQ <= 0 || HKV <= 0 || HQ % HKV != 0 || D <= 0) return 0;
  AttnModArgs a{};
  a.n = n;
  a.max_len = max_len;
  a.HQ = HQ;
  a.HKV = HKV;
  a.causal = causal;
  a.window = window;
  const int splits = dkv_splits(a);
  return dvec_floats(a) + (splits > 1 ? 2 * (int64_t)splits * n * HKV * D : 0);
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
  const int64_t floats = attn_mod_bwd_workspace(a.n, a.max_len, a.HQ, a.HKV, m.D, a.causal, a.window);
  if (m.workspace == nullptr || m.workspace_floats < floats) return QL_STATUS_BAD_ARG;
  // the second launch reads the inputs when the first has written dq
  const int64_t rows = m.n, row = (int64_t)m.HQ * m.D, kv_row = (int64_t)m.HKV * m.D;
  if (outputs_overlap({{m.dq, rows * row * 2},
                       {m.dk, rows * kv_row * 2},
                       {m.dv, rows * kv_row * 2},
                       {m.workspace, floats * 4},
                       {m.doc_ids != nullptr ? m.ranges : nullptr, rows * 8}},
                      {{m.q, ((rows - 1) * m.ldq + row) * 2},
                       {m.k, ((rows - 1) * m.ldk + kv_row) * 2},
                       {m.v, ((rows - 1) * m.ldv + kv_row) * 2},
                       {m.out, rows * row * 2},
                       {m.dout, rows * row * 2},
                       {m.lse, rows * m.HQ * 4},
                       {m.cu_seqlens, ((int64_t)m.B + 1) * 4},
                       {m.slopes, (int64_t)m.HQ * 4},
                       {m.prefix_len, (int64_t)m.B * 4},
                       {m.doc_ids, rows * 4}}))
    return QL_STATUS_BAD_ARG;
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
