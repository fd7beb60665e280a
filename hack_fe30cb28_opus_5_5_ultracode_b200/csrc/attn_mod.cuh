// Shared pieces of the attention kernels with modified scores and masks (attn_mod_fwd.cu,
// attn_mod_bwd.cu).
//
// Score of query i and key j of one sequence, in units of log2 (so that the softmax is a power of
// two):  y = log2(e) * (cap(scale * q_i . k_j) - slope_h |i - j|),  cap(x) = c tanh(x / c).
// Every mask these kernels take - causal, a prefix seen in both directions, a window |i - j| < w,
// documents (runs of equal ids; negative ids are padding) - leaves query i an interval
// [lo_i, hi_i) of keys, and both ends never decrease with i. So the first and last row of a query
// tile give the key blocks it has to visit (the hull [lo_first, hi_last)) and those it can visit
// without looking at the mask (inside [lo_last, hi_first)). Read from the key's side the same
// conditions leave key j an interval of queries, so a block of keys finds its query tiles in the same
// way. Padding rows get the empty interval [i, i).
#pragma once
#include <atomic>

#include "common.cuh"
#include "gemm_common.cuh"
#include "ops.h"

namespace ql {

constexpr int AM_T = 128;  // rows of a query tile and of a key block

// Launch arguments of both directions (the public structs, checked and flattened).
struct AttnModArgs {
  const void* q;
  const void* k;
  const void* v;
  const void* out;
  const void* dout;
  const int32_t* cu_seqlens;
  const float* slopes;       // [HQ] or null
  const int32_t* prefix_len; // [B] or null
  const int2* docs;          // [n] (first, end) of the token's document in its sequence, or null
  float* lse;                // [HQ, n]
  float* dvec;               // [HQ, n] rowsum(dout * out), backward only
  void* out_w;               // forward: out
  void* dq;
  void* dk;
  void* dv;
  float* parts;              // backward: dk / dv per split of a head group, or null
  float scale, softcap;
  int n, B, max_len, HQ, HKV, causal, window;
  int splits;                // backward: CTAs that share a KV head's query heads
};

struct AttnSeq {
  int start, len, prefix, causal, window;
  const int2* docs;  // of this sequence's first token, or null
};

__device__ __forceinline__ AttnSeq attn_seq(const AttnModArgs& a, int b) {
  AttnSeq s;
  s.start = a.cu_seqlens[b];
  s.len = a.cu_seqlens[b + 1] - s.start;
  s.causal = a.causal;
  s.window = a.window;
  s.prefix = a.prefix_len != nullptr ? min(max(a.prefix_len[b], 0), s.len) : 0;
  s.docs = a.docs != nullptr ? a.docs + s.start : nullptr;
  return s;
}

// [lo, hi) of query row i (i < len)
__device__ __forceinline__ int2 attn_row_range(const AttnSeq& s, int i) {
  int lo = 0, hi = s.len;
  if (s.causal) hi = max(i + 1, s.prefix);
  if (s.window > 0) {
    lo = max(0, i - s.window + 1);
    hi = min(hi, i + s.window);
  }
  if (s.docs != nullptr) {
    const int2 d = s.docs[i];
    lo = max(lo, d.x);
    hi = min(hi, d.y);
  }
  return make_int2(lo, hi);
}

// [lo, hi) of the query rows that see key j (j < len): the same conditions read from the key's
// side; again both ends never decrease with j.
__device__ __forceinline__ int2 attn_key_range(const AttnSeq& s, int j) {
  int lo = 0, hi = s.len;
  if (s.causal && j >= s.prefix) lo = j;
  if (s.window > 0) {
    lo = max(lo, j - s.window + 1);
    hi = min(hi, j + s.window);
  }
  if (s.docs != nullptr) {
    const int2 d = s.docs[j];
    lo = max(lo, d.x);
    hi = min(hi, d.y);
  }
  return make_int2(lo, hi);
}

// Blocks of 128 that the 128 rows from r0 on reach: visited [first, end), unmasked [ffirst, fend).
struct AttnBlocks {
  int first, end, ffirst, fend;
};
__device__ __forceinline__ AttnBlocks attn_blocks(int2 first_row, int2 last_row) {
  AttnBlocks t{0, 0, 0, 0};
  if (last_row.y <= first_row.x) return t;
  t.first = first_row.x / AM_T;
  t.end = (last_row.y + AM_T - 1) / AM_T;
  t.ffirst = (last_row.x + AM_T - 1) / AM_T;
  t.fend = first_row.y / AM_T;
  return t;
}
// Key blocks of a query tile, and query tiles of a key block.
__device__ __forceinline__ AttnBlocks attn_tile_blocks(const AttnSeq& s, int r0) {
  if (r0 >= s.len) return AttnBlocks{0, 0, 0, 0};
  return attn_blocks(attn_row_range(s, r0), attn_row_range(s, min(r0 + AM_T, s.len) - 1));
}
__device__ __forceinline__ AttnBlocks attn_key_blocks(const AttnSeq& s, int r0) {
  if (r0 >= s.len) return AttnBlocks{0, 0, 0, 0};
  return attn_blocks(attn_key_range(s, r0), attn_key_range(s, min(r0 + AM_T, s.len) - 1));
}

// ---- packed pairs of floats ------------------------------------------------------------------
__device__ __forceinline__ uint64_t pk2(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void up2(uint64_t v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// The arithmetic below runs on groups of independent pairs, one operation for the whole group before the
// next: a softmax warp shares its scheduler with at most three others, so the distance between
// dependent instructions has to come from the order they are written in.

template <int N>
__device__ __forceinline__ void ex2_2(uint64_t* x) {
  float a[N], b[N];
#pragma unroll
  for (int i = 0; i < N; ++i) up2(x[i], a[i], b[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    a[i] = ex2(a[i]);
    b[i] = ex2(b[i]);
  }
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = pk2(a[i], b[i]);
}

// tanh(u) = u P(u^2) for |u| <= 0.75, in place: coefficients of this library's own fit (reweighted least
// squares in relative error; 6.6e-8, 1.6e-7 in fp32 Horner evaluation).
constexpr float TANH_POLY_MAX = 0.75f;
template <int N>
__device__ __forceinline__ void tanh_poly2(uint64_t* u) {
  uint64_t w[N], p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = mul2(u[i], u[i]);
#pragma unroll
  for (int i = 0; i < N; ++i)
    p[i] = fma2(w[i], pk2(-0.004716250579804182f, -0.004716250579804182f), pk2(0.019582899287343025f, 0.019582899287343025f));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(-0.053344424813985825f, -0.053344424813985825f));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(0.1332540661096573f, 0.1332540661096573f));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(-0.33332958817481995f, -0.33332958817481995f));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(1.f, 1.f));
#pragma unroll
  for (int i = 0; i < N; ++i) u[i] = mul2(p[i], u[i]);
}
// c tanh(u x) = x (k0 + k1 x^2 + k2 x^4 + k3 x^6) for |u x| <= 0.4, in place: the fit with u and c in
// its coefficients (1.2e-7 relative, 2.3e-7 in fp32), five operations a pair where tanh_poly2 with
// its two scalings takes nine. Scores of a model trained with a cap rarely leave this range.
constexpr float TANH_SHORT_MAX = 0.4f;
struct TanhShort {
  float k[4];
};
__device__ __forceinline__ TanhShort tanh_short(float u, float c) {
  const float t[4] = {0.9999998807907104f, -0.33331361413002014f, 0.13270977139472961f, -0.04755359888076782f};
  TanhShort r;
  float m = c * u;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r.k[i] = m * t[i];
    m *= u * u;
  }
  return r;
}
template <int N>
__device__ __forceinline__ void tanh_short2(uint64_t* x, const TanhShort& t) {
  uint64_t w[N], p[N];
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = mul2(x[i], x[i]);
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(w[i], pk2(t.k[3], t.k[3]), pk2(t.k[2], t.k[2]));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(t.k[1], t.k[1]));
#pragma unroll
  for (int i = 0; i < N; ++i) p[i] = fma2(p[i], w[i], pk2(t.k[0], t.k[0]));
#pragma unroll
  for (int i = 0; i < N; ++i) x[i] = mul2(p[i], x[i]);
}
// Largest |x| of N raw words.
template <int N>
__device__ __forceinline__ float abs_max(const uint32_t* x) {
  float m[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < N; i += 8)
#pragma unroll
    for (int k = 0; k < 4; ++k)
      m[k] = max3(m[k], fabsf(__uint_as_float(x[i + 2 * k])), fabsf(__uint_as_float(x[i + 2 * k + 1])));
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// Which form a warp's block of scores takes: 0 tanh_short2, 1 tanh_poly2, 2 tanhf.
template <int N>
__device__ __forceinline__ int tanh_form(const uint32_t* x, float u) {
  const float m = abs_max<N>(x) * u;
  if (__all_sync(0xffffffffu, m <= TANH_SHORT_MAX)) return 0;
  return __all_sync(0xffffffffu, m <= TANH_POLY_MAX) ? 1 : 2;
}
__device__ __forceinline__ uint64_t pair_of(const uint32_t* x) {
  return pk2(__uint_as_float(x[0]), __uint_as_float(x[1]));
}
__device__ __forceinline__ void unpair(uint64_t v, uint32_t* x) {
  float a, b;
  up2(v, a, b);
  x[0] = __float_as_uint(a);
  x[1] = __float_as_uint(b);
}

// 16 consecutive fp32 columns of this thread's TMEM lane (with the wait), and into it (tmem_wait_st()
// before they are read).
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];\n\ttcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const float* v) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const float* v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(taddr), "f"(v[0]),
               "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

// ---- whole products, issued by a converged warp -----------------------------------------------
// The MMA warp runs its loop with all 32 lanes and elects the issuing one inside each instruction
// sequence, and the operand descriptors differ from step to step by a constant in their low word. So
// the compiler can keep descriptors and addresses in uniform registers: issued by `if (lane == 0)`
// from descriptors built per step, the 16 MMAs of a tile and block took 1,400-2,000 cycles of this
// warp, longer than the tensor core needs for them (forward of 8,192 causal tokens, 12 heads: 10%).
__device__ __forceinline__ int uniform_warp() { return __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0); }

// A value every lane holds, as one the compiler knows to be the same (what comes from memory it takes to
// differ, and then moves every descriptor from a vector register for every MMA).
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// High words of the operand descriptors (128-byte swizzle, version 1): stride 1024 B between groups of
// 8 rows. Low words: start address / 16, and for MN-major operands the distance of 64-element chunks.
constexpr uint32_t DESC_HI = (1024 >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_lo_k(uint32_t smem_addr) { return ((smem_addr >> 4) & 0x3FFFu) | (1u << 16); }
__device__ __forceinline__ uint32_t desc_lo_mn(uint32_t smem_addr, uint32_t chunk) {
  return ((smem_addr >> 4) & 0x3FFFu) | ((chunk >> 4) << 16);
}

// D (+)= A . B^T over a head of D_ elements, both operands K-major tiles of 64-column boxes
#define QL_AM_SS(OFF)                                                                              \
  "add.u32 x, %1, " OFF "; add.u32 y, %2, " OFF ";\n\t"                                            \
  "mov.b64 a, {x, %4}; mov.b64 b, {y, %4};\n\t"                                                   \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t"                                  \
  "setp.eq.u32 p, 0, 0;\n\t"
template <int D_>
__device__ __forceinline__ void umma_score(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc) {
  static_assert(D_ == 64 || D_ == 128, "one or two 64-column boxes");
  if constexpr (D_ == 64) {
    asm volatile("{\n\t.reg .pred p, e; .reg .b32 x, y; .reg .b64 a, b;\n\t"
                 "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, 0, 0;\n\t"
                 QL_AM_SS("0") QL_AM_SS("2") QL_AM_SS("4") QL_AM_SS("6") "}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(DESC_HI) : "memory");
  } else {  // the second box: 128 rows x 128 bytes further on
    asm volatile("{\n\t.reg .pred p, e; .reg .b32 x, y; .reg .b64 a, b;\n\t"
                 "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, 0, 0;\n\t"
                 QL_AM_SS("0") QL_AM_SS("2") QL_AM_SS("4") QL_AM_SS("6")
                 QL_AM_SS("1024") QL_AM_SS("1026") QL_AM_SS("1028") QL_AM_SS("1030") "}"
                 ::"r"(d), "r"(a_lo), "r"(b_lo), "r"(idesc), "n"(DESC_HI) : "memory");
  }
}
#undef QL_AM_SS

// D (+)= A . B over 128 rows of the MN-major tile B: A [128 x 128] 16-bit in TMEM, two elements per
// 32-bit column.
#define QL_AM_TS(AOFF, BOFF)                                                                       \
  "add.u32 x, %1, " AOFF "; add.u32 y, %2, " BOFF ";\n\t"                                          \
  "mov.b64 b, {y, %4};\n\t"                                                                       \
  "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [x], b, %3, p;\n\t"                                \
  "setp.eq.u32 p, 0, 0;\n\t"
// A's 64 columns in one piece
__device__ __forceinline__ void umma_gather1(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t more) {
  asm volatile("{\n\t.reg .pred p, e; .reg .b32 x, y; .reg .b64 b;\n\t"
               "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %5, 0;\n\t"
               QL_AM_TS("0", "0") QL_AM_TS("8", "128") QL_AM_TS("16", "256") QL_AM_TS("24", "384")
               QL_AM_TS("32", "512") QL_AM_TS("40", "640") QL_AM_TS("48", "768") QL_AM_TS("56", "896") "}"
               ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "n"(DESC_HI), "r"(more) : "memory");
}
// four parts of 16 columns, 32 apart (four softmax threads per row)
__device__ __forceinline__ void umma_gather4(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, uint32_t more) {
  asm volatile("{\n\t.reg .pred p, e; .reg .b32 x, y; .reg .b64 b;\n\t"
               "elect.sync _|e, 0xffffffff;\n\tsetp.ne.u32 p, %5, 0;\n\t"
               QL_AM_TS("0", "0") QL_AM_TS("8", "128") QL_AM_TS("32", "256") QL_AM_TS("40", "384")
               QL_AM_TS("64", "512") QL_AM_TS("72", "640") QL_AM_TS("96", "768") QL_AM_TS("104", "896") "}"
               ::"r"(d), "r"(a), "r"(b_lo), "r"(idesc), "n"(DESC_HI), "r"(more) : "memory");
}
#undef QL_AM_TS

// umma_commit by the lane that issues the MMAs
__device__ __forceinline__ void warp_commit(uint64_t* bar) {
  asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
               "@e tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
               ::"r"(smem_u32(bar)) : "memory");
}

// Which of the 128 rows [j0, j0 + 128) of a tile hold no key or query of the sequence (past its
// end, or padding), as bits: word u covers rows 32 u .. 32 u + 31 (every lane gets the same words).
// Their tile rows are zeroed before a tensor-core product, because a masked probability of 0 times a
// NaN or infinity left in such a row would not be 0.
struct DeadRows {
  uint32_t w[4];
  bool any;
};
__device__ __forceinline__ DeadRows attn_dead_rows(const AttnSeq& s, int j0) {
  DeadRows d{{0u, 0u, 0u, 0u}, false};
  if (j0 + AM_T <= s.len && s.docs == nullptr) return d;
  const int lane = threadIdx.x & 31;
  bool dead[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int r = j0 + u * 32 + lane;
    dead[u] = r >= s.len;
    if (!dead[u] && s.docs != nullptr) {
      const int2 e = s.docs[r];
      dead[u] = e.x >= e.y;
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    d.w[u] = __ballot_sync(0xffffffffu, dead[u]);
    d.any |= d.w[u] != 0;
  }
  return d;
}
// Zeroes those rows of a [boxes][128 rows][128 bytes] tile (whole rows, so the swizzle inside a
// row does not matter), by one warp: two or four rows a store.
template <int BOXES>
__device__ __forceinline__ void attn_zero_rows(uint8_t* tile, const DeadRows& d) {
  constexpr int ROWS = 4 / BOXES;
  const int lane = threadIdx.x & 31, sub = lane / (8 * BOXES);
  uint8_t* at = tile + (lane >> 3) % BOXES * (AM_T * 128) + sub * 128 + (lane & 7) * 16;
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (d.w[u] == 0) continue;
#pragma unroll
    for (int i = 0; i < 32; i += ROWS)
      if (d.w[u] >> (i + sub) & 1) *reinterpret_cast<uint4*>(at + (u * 32 + i) * 128) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// A wait of a whole warp (bounded, see mbar_wait): every lane gets the same answer, so a warp whose
// wait ran out leaves together.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, int* err) {
  return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// One arrival for the warp, after every lane's work before it (TMEM loads and stores completed and
// fenced by each lane). Arrivals of single lanes would be serialised on the barrier's word: 512 of them
// a step held the backward's chain up by about a thousand cycles.
__device__ __forceinline__ void warp_arrive(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Columns c of 32 with lo <= c < hi, as bits.
__device__ __forceinline__ uint32_t col_mask(int lo, int hi) {
  const int a = max(lo, 0), b = min(hi, 32);
  return b <= a ? 0u : (0xffffffffu >> (32 - (b - a))) << a;
}

// A warp's 32 result rows of W bytes (32, 64 or 128) through shared memory, so that they leave as whole
// lines: one thread holds one row, and its 16-byte stores straight to global memory touched 32 lines
// each (the epilogue of a 256-query CTA took 4,500 cycles). 16-byte chunk c of row r is kept at chunk
// c ^ (r / rows per 128 bytes): eight neighbouring rows in eight different bank groups.
template <int W>
__device__ __forceinline__ uint8_t* stage_at(uint8_t* stage, int row, int chunk) {
  return stage + row * W + ((chunk ^ ((row / (128 / W)) & (W / 16 - 1))) << 4);
}
// Rows [0, live) of the stage to dst, row pitch ld bytes.
template <int W>
__device__ __forceinline__ void stage_flush(uint8_t* stage, uint8_t* dst, int64_t ld, int live) {
  const int lane = threadIdx.x & 31;
  __syncwarp();
#pragma unroll
  for (int i = 0; i < W / 16; ++i) {
    const int row = (i * 32 + lane) / (W / 16), chunk = lane % (W / 16);
    if (row < live)
      *reinterpret_cast<uint4*>(dst + row * ld + chunk * 16) = *reinterpret_cast<const uint4*>(stage_at<W>(stage, row, chunk));
  }
  __syncwarp();
}

// Host: raises a kernel's dynamic shared-memory limit on the current device, once per device (host threads
// may race to it: the limit is the same).
inline int attn_smem_limit(const void* kernel, int bytes, std::atomic<unsigned long long>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return QL_STATUS_CUDA;
  if (dev < 64 && ((done.load(std::memory_order_acquire) >> dev) & 1)) return QL_STATUS_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
    return QL_STATUS_CUDA;
  if (dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
  return QL_STATUS_OK;
}

// Host: a [n, heads * D] 16-bit matrix with row stride ld as boxes of 128 rows of one head.
inline int attn_head_map(CUtensorMap* map, const void* ptr, int64_t n, int heads, int D, int64_t ld,
                         bool bf16) {
  return encode_chunked_map(map, ptr, n, (int64_t)heads * D, ld, AM_T, D / 64, bf16);
}

// Writes (first, end) of each token's document in its sequence (attn_mod_fwd.cu).
int attn_doc_ranges(const int32_t* doc_ids, const int32_t* cu_seqlens, int B, int n, int2* ranges,
                    cudaStream_t s);
// Checks the public arguments (both directions) and flattens them.
int attn_mod_check(const ql_attn_mod_args& m, AttnModArgs& a);
// The mode bits of the score: 1 capped, 2 distance bias.
inline int attn_mode(const AttnModArgs& a) { return (a.softcap > 0.f ? 1 : 0) | (a.slopes != nullptr ? 2 : 0); }

}  // namespace ql
