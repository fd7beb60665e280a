// qkv + LoRA + rotary embedding with several position axes (time, height, width, ...), forward and
// backward. Each of the D / 2 frequencies belongs to one axis; the angle of frequency f at token t
// is the table's at row pos[axis(f)][t], so a text token (all positions equal) rotates as in
// rope.cu and a picture's tokens by their row and column.
//
// A tile is 16 tokens (8 in the backward of short batches, see mrope_bwd). The tile's cosines and
// sines are gathered once into shared memory (a gather of single floats where neighbouring
// frequencies belong to different axes) and serve every head. Then each warp takes units of 32
// columns of a head together with their 32 partners D / 2 further on. The LoRA-B product of a unit is formed on the tensor cores in the layout the data
// is moved in: the eight columns of an m16n8k16 step can be any eight outputs, and with output
// 8 t + 2 j + e in column 2 t + e of step j, thread t of a row ends up with eight consecutive
// columns after four steps - one 16-byte load and store. The product stays in fp32 (nothing is
// rounded between the factors and the output). The backward uses the same ordering for the K
// dimension of dx_lo = s g B, with g split into 16-bit parts (fp16: brought to one size by a power of
// two per token and unit first) and the units' sums added up in fp32, so dx_lo is good to fp32 whatever the
// gradients' size.
//
// Bound: HBM for long batches (2 bytes read and 2 written per element in each direction), launch and
// L2 latency for short ones.
#include "common.cuh"
#include "ops.h"
#include "profile.h"

namespace ql {

namespace {

constexpr int MR_RANK = 16;
constexpr int MR_MAXHALF = 128;  // head sizes up to 256
constexpr int MR_UNIT = 32;      // columns of a unit (and as many partners)

struct MropeArgs {
  const void* qkv;       // forward
  const void* xq;
  const void* xv;
  const void* Bq;
  const void* Bv;
  void* q;
  void* k;
  void* v;
  const void* dq;        // backward
  const void* dk;
  const void* dv;
  void* dqkv;
  float* dxlo_q;
  float* dxlo_v;
  const float* cos;
  const float* sin;
  const int32_t* pos;
  int64_t ld_pos;
  int32_t positions;
  float lora_scale;
  int n, HQ, HKV, D;
  int* err;
  uint8_t axis[MR_MAXHALF];
};

// cos / sin of the tile's tokens, [rows][half + 4] floats each
__device__ __forceinline__ void stage_angles(const MropeArgs& a, float* sc, float* ss, int tok0, int rows) {
  const int half = a.D / 2, pitch = half + 4;
#pragma unroll 4
  for (int i = threadIdx.x; i < rows * half; i += blockDim.x) {
    const int r = i / half, f = i % half, tok = tok0 + r;
    float c = 0.f, s = 0.f;
    if (tok < a.n) {
      const int p = a.pos[a.axis[f] * a.ld_pos + tok];
      if (p >= 0 && p < a.positions) {
        c = __ldg(a.cos + (int64_t)p * half + f);
        s = __ldg(a.sin + (int64_t)p * half + f);
      } else {
        raise_status(a.err, QL_STATUS_BAD_ARG);
      }
    }
    sc[r * pitch + f] = c;
    ss[r * pitch + f] = s;
  }
}

// 8 consecutive values of a row, as loaded and as floats
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
};
template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T* p) {
  Raw8<T> r;
#pragma unroll
  for (int i = 0; i < (int)sizeof(T) / 2; ++i) r.w[i] = __ldcs(reinterpret_cast<const uint4*>(p) + i);
  return r;
}
template <typename T>
__device__ __forceinline__ float2 unpack2(uint32_t u) {
  if constexpr (std::is_same<T, __half>::value) {
    return __half22float2(*reinterpret_cast<const __half2*>(&u));
  } else {
    return make_float2(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
  }
}
template <typename T>
__device__ __forceinline__ void floats8(const Raw8<T>& r, float* v) {
  const uint32_t* u = reinterpret_cast<const uint32_t*>(&r);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = __uint_as_float(u[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = unpack2<T>(u[j]);
      v[2 * j] = f.x;
      v[2 * j + 1] = f.y;
    }
  }
}
template <typename T>
__device__ __forceinline__ void store8(T* p, const float* v) {
  *reinterpret_cast<uint4*>(p) = make_uint4(pack_t2<T>(v[0], v[1]), pack_t2<T>(v[2], v[3]),
                                            pack_t2<T>(v[4], v[5]), pack_t2<T>(v[6], v[7]));
}

// acc[rh][8] += s x_lo . B^T for the 32 outputs from row o0 of B on: this thread's eight columns
// 8 t .. 8 t + 7 of tokens g and g + 8 of the tile
template <typename T>
__device__ __forceinline__ void lora_out(const uint32_t* af, const void* B, int64_t o0, float s, float (*acc)[8]) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  // step j: column n of the step is output 8 (n / 2) + 2 j + n % 2; the K indices of thread t
  // (2 t, 2 t + 1, 2 t + 8, 2 t + 9) are ranks 4 t .. 4 t + 3, in both operands
  const uint2* base = reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(B) +
                      (o0 + (g >> 1) * 8 + (g & 1)) * MR_RANK) + t;
  uint2 b[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) b[j] = __ldg(base + j * (2 * MR_RANK / 4));
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float c[4] = {0.f, 0.f, 0.f, 0.f};
    mma16816<T>(c, af, b[j].x, b[j].y);
    acc[0][2 * j] += c[0] * s;
    acc[0][2 * j + 1] += c[1] * s;
    acc[1][2 * j] += c[2] * s;
    acc[1][2 * j + 1] += c[3] * s;
  }
}

// A fragment of x_lo [n, 16] for the tile's tokens
template <typename T>
__device__ __forceinline__ void lora_in(const void* x, int tok0, int rows, int n, uint32_t* af) {
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
#pragma unroll
  for (int rh = 0; rh < 2; ++rh) {
    const int r = g + rh * 8, tok = tok0 + r;
    uint2 v = make_uint2(0u, 0u);
    if (r < rows && tok < n)
      v = __ldg(reinterpret_cast<const uint2*>(reinterpret_cast<const T*>(x) + (int64_t)tok * MR_RANK) + t);
    af[rh] = v.x;
    af[2 + rh] = v.y;
  }
}

// (o1, o2) = (x1 c -+ x2 s, x2 c +- x1 s) with the row's angles from shared memory; BACK: the inverse
template <bool BACK>
__device__ __forceinline__ void turn8(float* x1, float* x2, const float* cr, const float* sr) {
#pragma unroll
  for (int q = 0; q < 2; ++q) {
    const float4 c4 = reinterpret_cast<const float4*>(cr)[q], s4 = reinterpret_cast<const float4*>(sr)[q];
    const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = x1[4 * q + e], r = x2[4 * q + e];
      x1[4 * q + e] = BACK ? p * c[e] + r * s[e] : p * c[e] - r * s[e];
      x2[4 * q + e] = BACK ? r * c[e] - p * s[e] : r * c[e] + p * s[e];
    }
  }
}

// A unit: 32 columns of one head and their 32 partners; v's heads come after the rotated ones.
struct Unit {
  int head, d0;  // head of the [q | k | v] row, first column
};
__device__ __forceinline__ Unit unit_of(int u, int per_head) { return {u / per_head, (u % per_head) * MR_UNIT}; }

constexpr int MR_THREADS = 256, MR_CTAS = 3;  // 24 warps per SM at 80 registers (16 at 110: 136 us
                                              // against 113 for 24 k tokens of 28 + 8 heads)

template <typename T, int ROWS>
__global__ void __launch_bounds__(MR_THREADS, MR_CTAS) mrope_fwd_kernel(const __grid_constant__ MropeArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float angle_smem[];
  const int half = a.D / 2, pitch = half + 4;
  float* sc = angle_smem;
  float* ss = angle_smem + ROWS * pitch;
  const int tok0 = blockIdx.x * ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int per_head = half / MR_UNIT, units = (a.HQ + 2 * a.HKV) * per_head;
  const int64_t C = (int64_t)(a.HQ + 2 * a.HKV) * a.D;
  stage_angles(a, sc, ss, tok0, ROWS);
  uint32_t aq[4], av[4];
  if (a.xq != nullptr) lora_in<T>(a.xq, tok0, ROWS, a.n, aq);
  if (a.xv != nullptr) lora_in<T>(a.xv, tok0, ROWS, a.n, av);
  __syncthreads();
  const int step = gridDim.y * (blockDim.x >> 5);
  for (int u = blockIdx.y * (blockDim.x >> 5) + warp; u < units; u += step) {
    const Unit un = unit_of(u, per_head);
    const int d = un.d0 + t * 8;
    const bool is_q = un.head < a.HQ, is_v = un.head >= a.HQ + a.HKV;
    Raw8<T> raw[2][2];  // [row g / g + 8][first / partner]
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      const int r = g + rh * 8, tok = tok0 + r;
      const T* row = reinterpret_cast<const T*>(a.qkv) + tok * C + un.head * a.D + d;
      raw[rh][0] = r < ROWS && tok < a.n ? load8<T>(row) : Raw8<T>{};
      raw[rh][1] = r < ROWS && tok < a.n ? load8<T>(row + half) : Raw8<T>{};
    }
    float x1[2][8], x2[2][8];
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      floats8<T>(raw[rh][0], x1[rh]);
      floats8<T>(raw[rh][1], x2[rh]);
    }
    if (is_q && a.xq != nullptr) {
      const int64_t o = (int64_t)un.head * a.D + un.d0;
      lora_out<T>(aq, a.Bq, o, a.lora_scale, x1);
      lora_out<T>(aq, a.Bq, o + half, a.lora_scale, x2);
    } else if (is_v && a.xv != nullptr) {
      const int64_t o = (int64_t)(un.head - a.HQ - a.HKV) * a.D + un.d0;
      lora_out<T>(av, a.Bv, o, a.lora_scale, x1);
      lora_out<T>(av, a.Bv, o + half, a.lora_scale, x2);
    }
    T* dst = is_q ? reinterpret_cast<T*>(a.q) + un.head * a.D
                  : is_v ? reinterpret_cast<T*>(a.v) + (un.head - a.HQ - a.HKV) * a.D
                         : reinterpret_cast<T*>(a.k) + (un.head - a.HQ) * a.D;
    const int64_t ld = (int64_t)(is_q ? a.HQ : a.HKV) * a.D;
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      const int r = g + rh * 8, tok = tok0 + r;
      if (r >= ROWS || tok >= a.n) continue;
      if (!is_v) turn8<false>(x1[rh], x2[rh], sc + r * pitch + d, ss + r * pitch + d);
      store8<T>(dst + tok * ld + d, x1[rh]);
      store8<T>(dst + tok * ld + d + half, x2[rh]);
    }
  }
}

// The power of two that brings a token's largest of 32 gradients to [2^14, 2^15), and its inverse. fp16
// has no number below 2^-24 and none above 65,504: unscaled, the second part of a gradient of 10^-3
// lost all but 2^-16 of it (10^-5: 2^-9), and fp32 gradients above 65,504 had none. A token's scale is
// its own, as sizes differ from token to token; 0 (and what fp32 holds as a subnormal), infinities and NaN
// keep a scale of 1.
struct TokenScale {
  float up, down;
};
__device__ __forceinline__ TokenScale token_scale(const float* v) {
  float m = 0.f;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = fmaxf(m, fabsf(v[e]));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 2));
  int e = __float_as_int(m) >> 23;           // biased exponent
  if (e == 0 || e == 255) return {1.f, 1.f};
  e = max(e, 15);
  return {__int_as_float((268 - e) << 23), __int_as_float((e - 14) << 23)};
}

// acc[2 tiles of N][4] += g . B for 32 columns of g (this thread: 8 t .. 8 t + 7 of tokens g and g + 8)
// and the 32 rows of B from o0 on. Column n of N tile nt is rank 2 n + nt, so one 32-bit load of a
// row of B serves both tiles; K index 2 t + e (8 + 2 t + e) of step s is row 8 t + 4 s + e (+ 2).
template <typename T>
__device__ __forceinline__ void lora_back(const float (*gv)[8], const void* B, int64_t o0, float (*acc)[4]) {
  constexpr bool SCALED = std::is_same<T, __half>::value;
  const int lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const uint32_t* base = reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(B) + (o0 + t * 8) * MR_RANK) + g;
  float own[2][4] = {};
  float (*c)[4] = SCALED ? own : acc;
  TokenScale sc[2];
  if constexpr (SCALED) {
    sc[0] = token_scale(gv[0]);
    sc[1] = token_scale(gv[1]);
  }
#pragma unroll
  for (int s = 0; s < 2; ++s) {
    uint32_t w[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) w[e] = __ldg(base + (4 * s + e) * (MR_RANK / 2));
    // g in PARTS 16-bit pieces, each the rounding of what the ones before left: 2^-24 (bf16) or
    // 2^-22 (fp16) of g stays behind, or 2^-39 of the token's largest
    constexpr int PARTS = std::is_same<T, __nv_bfloat16>::value ? 3 : 2;
    float left[2][4];
#pragma unroll
    for (int rh = 0; rh < 2; ++rh)
#pragma unroll
      for (int k = 0; k < 4; ++k) left[rh][k] = SCALED ? gv[rh][4 * s + k] * sc[rh].up : gv[rh][4 * s + k];
#pragma unroll
    for (int part = 0; part < PARTS; ++part) {
      uint32_t af[4];
#pragma unroll
      for (int rh = 0; rh < 2; ++rh)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const uint32_t h = pack_t2<T>(left[rh][2 * k], left[rh][2 * k + 1]);
          const float2 f = unpack2<T>(h);
          af[rh + 2 * k] = h;
          left[rh][2 * k] -= f.x;
          left[rh][2 * k + 1] -= f.y;
        }
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) {
        const uint32_t sel = nt == 0 ? 0x5410 : 0x7632;
        mma16816<T>(c[nt], af, __byte_perm(w[0], w[1], sel), __byte_perm(w[2], w[3], sel));
      }
    }
  }
  if constexpr (SCALED) {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[nt][e] = fmaf(own[nt][e], sc[e >> 1].down, acc[nt][e]);
  }
}

template <typename T, typename TG, int ROWS>
__global__ void __launch_bounds__(MR_THREADS, MR_CTAS) mrope_bwd_kernel(const __grid_constant__ MropeArgs a) {
  pdl_enter();
  extern __shared__ __align__(16) float angle_smem[];
  const int half = a.D / 2, pitch = half + 4;
  float* sc = angle_smem;
  float* ss = angle_smem + ROWS * pitch;
  const int tok0 = blockIdx.x * ROWS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int warps = blockDim.x >> 5;
  const int per_head = half / MR_UNIT, units = (a.HQ + 2 * a.HKV) * per_head;
  const int64_t C = (int64_t)(a.HQ + 2 * a.HKV) * a.D;
  stage_angles(a, sc, ss, tok0, ROWS);
  __syncthreads();
  const bool lq = a.dxlo_q != nullptr, lv = a.dxlo_v != nullptr;
  float cq[2][4] = {}, cv[2][4] = {};
  // The tensor core cuts its sums off where fp32 addition rounds them: running sums over a token's 56 units
  // (28 heads of 128) were off by 1.5e-6, sums of one unit each, added up here, by 2.7e-7. fp16's are added
  // unit by unit for their scales; a bf16 unit's (c) when the next one's loads are on their way
  // (24 k tokens of 28 + 4 heads: 131 -> 134 us, at once 144).
  constexpr bool LATER = std::is_same<T, __nv_bfloat16>::value;
  float c[2][4] = {};
  bool of_q = true;  // whose unit c is
  auto add_unit = [&]() {
#pragma unroll
    for (int nt = 0; nt < 2; ++nt)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (of_q) cq[nt][e] += c[nt][e];
        else cv[nt][e] += c[nt][e];
        c[nt][e] = 0.f;
      }
  };
  for (int u = blockIdx.y * warps + warp; u < units; u += gridDim.y * warps) {
    const Unit un = unit_of(u, per_head);
    const int d = un.d0 + t * 8;
    const bool is_q = un.head < a.HQ, is_v = un.head >= a.HQ + a.HKV;
    const TG* src = is_q ? reinterpret_cast<const TG*>(a.dq) + un.head * a.D
                         : is_v ? reinterpret_cast<const TG*>(a.dv) + (un.head - a.HQ - a.HKV) * a.D
                                : reinterpret_cast<const TG*>(a.dk) + (un.head - a.HQ) * a.D;
    const int64_t ld = (int64_t)(is_q ? a.HQ : a.HKV) * a.D;
    Raw8<TG> raw[2][2];
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      const int r = g + rh * 8, tok = tok0 + r;
      raw[rh][0] = r < ROWS && tok < a.n ? load8<TG>(src + tok * ld + d) : Raw8<TG>{};
      raw[rh][1] = r < ROWS && tok < a.n ? load8<TG>(src + tok * ld + d + half) : Raw8<TG>{};
    }
    if (LATER && (lq || lv)) add_unit();
    float x1[2][8], x2[2][8];
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      floats8<TG>(raw[rh][0], x1[rh]);
      floats8<TG>(raw[rh][1], x2[rh]);
    }
#pragma unroll
    for (int rh = 0; rh < 2; ++rh) {
      const int r = g + rh * 8, tok = tok0 + r;
      if (r >= ROWS || tok >= a.n) continue;
      if (!is_v) turn8<true>(x1[rh], x2[rh], sc + r * pitch + d, ss + r * pitch + d);
      T* out = reinterpret_cast<T*>(a.dqkv) + tok * C + un.head * a.D + d;
      store8<T>(out, x1[rh]);
      store8<T>(out + half, x2[rh]);
    }
    if (is_q && lq) {
      const int64_t o = (int64_t)un.head * a.D + un.d0;
      lora_back<T>(x1, a.Bq, o, LATER ? c : cq);
      lora_back<T>(x2, a.Bq, o + half, LATER ? c : cq);
      of_q = true;
    } else if (is_v && lv) {
      const int64_t o = (int64_t)(un.head - a.HQ - a.HKV) * a.D + un.d0;
      lora_back<T>(x1, a.Bv, o, LATER ? c : cv);
      lora_back<T>(x2, a.Bv, o + half, LATER ? c : cv);
      of_q = false;
    }
  }
  if (!lq && !lv) return;
  if (LATER) add_unit();
  // the warps' partial sums, added in warp order
  float* red = angle_smem + 2 * ROWS * pitch;  // [warps][2][16 tokens][16]
#pragma unroll
  for (int nt = 0; nt < 2; ++nt)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int r = g + (e >> 1) * 8, rank = 2 * (2 * t + (e & 1)) + nt;
      red[((warp * 2 + 0) * 16 + r) * MR_RANK + rank] = cq[nt][e];
      red[((warp * 2 + 1) * 16 + r) * MR_RANK + rank] = cv[nt][e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * ROWS * MR_RANK; i += blockDim.x) {
    const int ad = i / (ROWS * MR_RANK), r = (i / MR_RANK) % ROWS, rank = i % MR_RANK;
    if (tok0 + r >= a.n || !(ad == 0 ? lq : lv)) continue;
    float sum = 0.f;
    for (int w = 0; w < warps; ++w) sum += red[((w * 2 + ad) * 16 + r) * MR_RANK + rank];
    (ad == 0 ? a.dxlo_q : a.dxlo_v)[(int64_t)(tok0 + r) * MR_RANK + rank] = sum * a.lora_scale;
  }
}

// The frequencies' axes: blocks of the sections, or dealt to the axes in turn while an axis has some
// left. False if the sections do not make up D / 2.
bool mrope_axes(const int32_t* sec, int axes, int interleaved, int half, uint8_t* axis) {
  int64_t sum = 0;
  for (int x = 0; x < axes; ++x) {
    if (sec[x] < 0) return false;
    sum += sec[x];
  }
  if (sum != half) return false;
  int left[4] = {0, 0, 0, 0};
  for (int x = 0; x < axes; ++x) left[x] = sec[x];
  for (int f = 0, x = 0; f < half; ++f) {
    if (interleaved) {
      while (left[x] == 0) x = (x + 1) % axes;
      axis[f] = (uint8_t)x;
      --left[x];
      x = (x + 1) % axes;
    } else {
      while (left[x] == 0) ++x;
      axis[f] = (uint8_t)x;
      --left[x];
    }
  }
  return true;
}

int mrope_check(const ql_mrope_args& m, MropeArgs& a) {
  if (m.n < 0 || m.HKV <= 0 || m.HQ <= 0 || m.D <= 0 || m.axes < 1 || m.axes > 4) return QL_STATUS_BAD_ARG;
  if (m.D % 64 != 0 || m.D > 2 * MR_MAXHALF) return QL_STATUS_UNSUPPORTED;
  if (m.dtype != QL_F16 && m.dtype != QL_BF16) return QL_STATUS_BAD_ARG;
  a = MropeArgs{};
  const int32_t sec[4] = {m.sec0, m.sec1, m.sec2, m.sec3};
  if (!mrope_axes(sec, m.axes, m.interleaved, m.D / 2, a.axis)) return QL_STATUS_BAD_ARG;
  if (m.n > 0 && (m.cos == nullptr || m.sin == nullptr || m.pos == nullptr || m.positions < 0 ||
                  (m.axes > 1 && m.ld_pos < m.n)))
    return QL_STATUS_BAD_ARG;
  a.Bq = m.Bq;
  a.Bv = m.Bv;
  a.cos = m.cos;
  a.sin = m.sin;
  a.pos = m.pos;
  a.ld_pos = m.ld_pos;
  a.positions = m.positions;
  a.lora_scale = m.lora_scale;
  a.n = m.n;
  a.HQ = m.HQ;
  a.HKV = m.HKV;
  a.D = m.D;
  a.err = status_word();
  return QL_STATUS_OK;
}

// What both directions read: the tables and positions (by the call's own sizes).
MemSpan table_span(const ql_mrope_args& m, const float* t) { return {t, (int64_t)m.positions * (m.D / 2) * 4}; }
MemSpan pos_span(const ql_mrope_args& m) { return {m.pos, ((m.axes - 1) * m.ld_pos + m.n) * 4}; }

bool misaligned(std::initializer_list<const void*> ps, uintptr_t to) {
  uintptr_t bits = 0;
  for (const void* p : ps) bits |= reinterpret_cast<uintptr_t>(p);
  return (bits & (to - 1)) != 0;
}

}  // namespace

int mrope_fwd(const ql_mrope_args& m, cudaStream_t s) {
  MropeArgs a;
  const int st = mrope_check(m, a);
  if (st != QL_STATUS_OK) return st;
  if (m.n == 0) return QL_STATUS_OK;
  if (m.qkv == nullptr || m.q == nullptr || m.k == nullptr || m.v == nullptr ||
      (m.xq != nullptr && m.Bq == nullptr) || (m.xv != nullptr && m.Bv == nullptr) ||
      misaligned({m.qkv, m.q, m.k, m.v}, 16) || misaligned({m.xq, m.xv, m.Bq, m.Bv}, 8))
    return QL_STATUS_BAD_ARG;
  const int64_t qb = (int64_t)m.HQ * m.D * 2, kvb = (int64_t)m.HKV * m.D * 2;  // bytes of a token's heads
  if (outputs_overlap({{m.q, m.n * qb}, {m.k, m.n * kvb}, {m.v, m.n * kvb}},
                      {{m.qkv, m.n * (qb + 2 * kvb)},
                       {m.xq, (int64_t)m.n * MR_RANK * 2},
                       {m.xv, (int64_t)m.n * MR_RANK * 2},
                       {m.xq != nullptr ? m.Bq : nullptr, qb * MR_RANK},
                       {m.xv != nullptr ? m.Bv : nullptr, kvb * MR_RANK},
                       table_span(m, m.cos),
                       table_span(m, m.sin),
                       pos_span(m)}))
    return QL_STATUS_BAD_ARG;
  a.qkv = m.qkv;
  a.xq = m.xq;
  a.xv = m.xv;
  a.q = m.q;
  a.k = m.k;
  a.v = m.v;
  const double elems = (double)m.n * (m.HQ + 2 * m.HKV) * m.D;
  ProfScope prof(PK_ROPE_FWD, 0, elems * 4, s);
  const int units = (m.HQ + 2 * m.HKV) * (m.D / 2 / MR_UNIT);
  const int warps = units < MR_THREADS / 32 ? units : MR_THREADS / 32;
  const int tiles = (int)cdiv(m.n, 16);
  const int most = (int)cdiv(units, warps);
  int gy = (int)cdiv(2 * sm_count(), tiles);  // short batches: the columns over several CTAs
  gy = gy > most ? most : gy;
#define QL_MROPEF(TT)                                                                       \
  launch_k(mrope_fwd_kernel<TT, 16>, dim3(tiles, gy), dim3(32 * warps), 2 * 16 * (m.D / 2 + 4) * 4, s, a)
  if (m.dtype == QL_F16) QL_MROPEF(__half); else QL_MROPEF(__nv_bfloat16);
#undef QL_MROPEF
  return launched(1);
}

int mrope_bwd(const ql_mrope_args& m, cudaStream_t s) {
  MropeArgs a;
  const int st = mrope_check(m, a);
  if (st != QL_STATUS_OK) return st;
  if (m.grad_dtype != QL_F32 && m.grad_dtype != m.dtype) return QL_STATUS_BAD_ARG;
  if (m.n == 0) return QL_STATUS_OK;
  if (m.dq == nullptr || m.dk == nullptr || m.dv == nullptr || m.dqkv == nullptr ||
      (m.dxlo_q != nullptr && m.Bq == nullptr) || (m.dxlo_v != nullptr && m.Bv == nullptr) ||
      misaligned({m.dq, m.dk, m.dv, m.dqkv}, 16) || misaligned({m.Bq, m.Bv}, 8))
    return QL_STATUS_BAD_ARG;
  const int64_t qc = (int64_t)m.HQ * m.D, kvc = (int64_t)m.HKV * m.D, size = m.grad_dtype == QL_F32 ? 4 : 2;
  if (outputs_overlap({{m.dqkv, m.n * (qc + 2 * kvc) * 2},
                       {m.dxlo_q, (int64_t)m.n * MR_RANK * 4},
                       {m.dxlo_v, (int64_t)m.n * MR_RANK * 4}},
                      {{m.dq, m.n * qc * size},
                       {m.dk, m.n * kvc * size},
                       {m.dv, m.n * kvc * size},
                       {m.dxlo_q != nullptr ? m.Bq : nullptr, qc * MR_RANK * 2},
                       {m.dxlo_v != nullptr ? m.Bv : nullptr, kvc * MR_RANK * 2},
                       table_span(m, m.cos),
                       table_span(m, m.sin),
                       pos_span(m)}))
    return QL_STATUS_BAD_ARG;
  a.dq = m.dq;
  a.dk = m.dk;
  a.dv = m.dv;
  a.dqkv = m.dqkv;
  a.dxlo_q = m.dxlo_q;
  a.dxlo_v = m.dxlo_v;
  const bool lora = m.dxlo_q != nullptr || m.dxlo_v != nullptr;
  const double elems = (double)m.n * (m.HQ + 2 * m.HKV) * m.D;
  ProfScope prof(PK_ROPE_BWD, 0, elems * (m.grad_dtype == QL_F32 ? 6 : 4), s);
  const int units = (m.HQ + 2 * m.HKV) * (m.D / 2 / MR_UNIT);
  const int warps = units < MR_THREADS / 32 ? units : MR_THREADS / 32;
#define QL_MROPEB(TT, TG, ROWS)                                                                   \
  do {                                                                                            \
    const int tiles = (int)cdiv(m.n, ROWS);                                                       \
    int gy = lora ? 1 : (int)cdiv(2 * sm_count(), tiles);                                         \
    const int most = (int)cdiv(units, warps);                                                     \
    gy = gy < 1 ? 1 : gy > most ? most : gy;                                                      \
    const int smem = 2 * ROWS * (m.D / 2 + 4) * 4 + (lora ? warps * 2 * 16 * MR_RANK * 4 : 0);    \
    launch_k(mrope_bwd_kernel<TT, TG, ROWS>, dim3(tiles, gy), dim3(32 * warps), smem, s, a);      \
  } while (0)
#define QL_MROPEB2(ROWS)                                                                          \
  do {                                                                                            \
    if (m.dtype == QL_F16) {                                                                      \
      if (m.grad_dtype == QL_F32) QL_MROPEB(__half, float, ROWS);                                 \
      else QL_MROPEB(__half, __half, ROWS);                                                       \
    } else {                                                                                      \
      if (m.grad_dtype == QL_F32) QL_MROPEB(__nv_bfloat16, float, ROWS);                          \
      else QL_MROPEB(__nv_bfloat16, __nv_bfloat16, ROWS);                                         \
    }                                                                                             \
  } while (0)
  // 8 tokens per CTA while all CTAs are resident at once (3,552 tokens on 148 SMs): B is read twice as
  // often, but by twice as many CTAs. 8 against 16 tokens, us: 61 tokens of 12 + 2 heads 7.6 / 10.5, 1,090
  // 9.0 / 11.6, 3,000 13.0 / 16.6, 4,000 20.8 / 18.8, 24 k of 28 + 4 heads 160 / 137.
  if (m.n > 8 * MR_CTAS * sm_count()) QL_MROPEB2(16); else QL_MROPEB2(8);
#undef QL_MROPEB2
#undef QL_MROPEB
  return launched(1);
}

}  // namespace ql
