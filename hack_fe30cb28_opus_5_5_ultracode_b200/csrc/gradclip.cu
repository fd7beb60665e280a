// Global 2-norm of a list of gradient tensors, and clipping by it.
//
// Two passes and no meeting of the CTAs inside a kernel: the first writes one sum of squares per
// CTA; in the second every CTA adds those sums in the same order (fp64), so all arrive at the same
// factor, and rescales its part. A gradient list that fits in L2 is read from HBM once. Squares are
// summed in fp32 over eight loads of a thread (four sums of 8 to 16 values; over thousands of them the
// norm was off by 1.5e-6), from there on in fp64; loads whose squares leave fp32's range (gradients above
// 1.8e19, or all below 1e-15) are looked at once more and squared in fp64 unless they are zeros (0.28 G
// fp32 zeros, or 5% nonzero values: 157 -> 211 us).
//
// The tensors' addresses and sizes travel as kernel parameters (up to 1,024 tensors a launch), so a
// call copies nothing to the device and can be captured. Work is cut into chunks of 32 KB of one
// tensor, and each CTA takes one stretch of them: it searches the list once and then walks it. Where
// addresses are 16-byte aligned a thread moves up to 16 bytes at a time, eight loads in flight; other
// spans go element by element.
//
// Bound: HBM (one read for the norm; one read and one write for the rescale) for large lists, two
// launch latencies for small ones. 0.9 G bf16 gradients: norm 256 us (7.0 TB/s), norm and rescale into
// fp32 1,205 us (6.0 TB/s of the bytes both passes move).
#include <algorithm>
#include <exception>
#include <utility>
#include <vector>

#include "common.cuh"
#include "ops.h"
#include "profile.h"

namespace ql {

namespace {

constexpr int GC_THREADS = 256;
constexpr int GC_CHUNK = 32768;      // bytes of gradient per chunk
constexpr int GC_CTAS_PER_SM = 4;

template <int MAX>
struct GradList {
  const void* grad[MAX];
  void* out[MAX];
  int64_t n[MAX];
  int32_t first[MAX + 1];  // first chunk of each tensor; [count]: all chunks
  uint8_t dtype[MAX], out_dtype[MAX];
  int32_t count;
};

__device__ __forceinline__ int chunk_elems(int dtype) { return dtype == QL_F32 ? GC_CHUNK / 4 : GC_CHUNK / 2; }

template <int MAX>
__device__ __forceinline__ int tensor_of(const GradList<MAX>& l, int chunk) {
  int lo = 0, hi = l.count;  // first[lo] <= chunk < first[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (l.first[mid] <= chunk) lo = mid; else hi = mid;
  }
  return lo;
}

template <typename T>
__device__ __forceinline__ void square16(const uint4& u, float* s) {
  if constexpr (sizeof(T) == 4) {
    const float* f = reinterpret_cast<const float*>(&u);
#pragma unroll
    for (int e = 0; e < 4; ++e) s[e] = fmaf(f[e], f[e], s[e]);
  } else {
    const T* h = reinterpret_cast<const T*>(&u);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float f = to_f<T>(h[e]);
      s[e & 3] = fmaf(f, f, s[e & 3]);
    }
  }
}

__device__ __forceinline__ double sum4(const float* s) {
  return ((double)s[0] + (double)s[1]) + ((double)s[2] + (double)s[3]);
}

// Whether fp32 sums of squares are in a range where no square that counts was lost: a square above 2^128
// makes its sum infinite, those below 2^-126 matter only where all of them together are below about 2^-100
// (zeros too: their squares may have vanished). fp16's never leave the range.
template <typename T>
__device__ __forceinline__ bool squares_fit(const float* s) {
  if constexpr (std::is_same<T, __half>::value) return true;
  const float most = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));  // a NaN stays in their sum
  return most > 1e-30f && most <= 3e38f;
}
// The bits, but for signs, of 16 bytes of gradients: 0 if all are zeros
template <typename T>
__device__ __forceinline__ uint32_t bits16(const uint4& u) {
  return (u.x | u.y | u.z | u.w) & (sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu);
}
// Squares in fp64 of p[i], p[i + GC_THREADS], ... before end, up to eight places of V values, read once more
// (from the caches), so that the loads in flight of the usual case keep their registers.
template <typename T, int V>
__device__ __noinline__ double squares_wide(const T* p, int64_t i, int64_t end) {
  double s = 0.0;
  if constexpr (V > 1) {  // nothing but zeros, in gradients that are not used or sparse ones
    uint32_t any = 0;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int64_t at = i + k * GC_THREADS;
      any |= at < end ? bits16<T>(reinterpret_cast<const uint4*>(p)[at]) : 0u;
    }
    if (any == 0) return s;
  }
#pragma unroll 1
  for (; i < end; i += GC_THREADS)
#pragma unroll 1
    for (int e = 0; e < V; ++e) {
      const double f = (double)to_f<T>(p[i * V + e]);
      s = fma(f, f, s);
    }
  return s;
}

template <typename T>
__device__ __forceinline__ double span_squares(const T* p, int64_t n) {
  constexpr int V = 16 / sizeof(T);
  double all = 0.0;
  int64_t done = 0;
  if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
    const uint4* v = reinterpret_cast<const uint4*>(p);
    const int64_t nv = n / V;
    int64_t i = threadIdx.x;
    for (; i + 7 * GC_THREADS < nv; i += 8 * GC_THREADS) {
      uint4 u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = v[i + k * GC_THREADS];
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) square16<T>(u[k], s);
      all += squares_fit<T>(s) ? sum4(s) : squares_wide<T, V>(p, i, i + 7 * GC_THREADS + 1);
    }
    const int64_t rest = i;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    for (; i < nv; i += GC_THREADS) square16<T>(v[i], s);
    if (rest < nv) all += squares_fit<T>(s) ? sum4(s) : squares_wide<T, V>(p, rest, nv);
    done = nv * V;
  }
  // up to seven values of an aligned span, all of another one
  for (int64_t i0 = done + threadIdx.x; i0 < n; i0 += 16 * GC_THREADS) {
    float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int64_t i = i0 + k * GC_THREADS;
      const float f = i < n ? to_f<T>(p[i]) : 0.f;
      s[k & 3] = fmaf(f, f, s[k & 3]);
    }
    const int64_t end = i0 + 16 * GC_THREADS;
    all += squares_fit<T>(s) ? sum4(s) : squares_wide<T, 1>(p, i0, end < n ? end : n);
  }
  return all;
}

// The CTA's stretch of the list's chunks, cut at the tensors' ends: f(tensor, first element, elements).
template <int MAX, typename F>
__device__ __forceinline__ void walk(const GradList<MAX>& l, F f) {
  const int64_t chunks = l.first[l.count];
  const int c0 = (int)(chunks * blockIdx.x / gridDim.x), c1 = (int)(chunks * (blockIdx.x + 1) / gridDim.x);
  if (c0 >= c1) return;
  int t = tensor_of(l, c0);
  for (int c = c0; c < c1; ++t) {
    const int f0 = l.first[t], to = min(c1, l.first[t + 1]);
    if (to > c) {
      const int64_t per = chunk_elems(l.dtype[t]), at = (c - f0) * per;
      f(t, at, min((to - c) * per, l.n[t] - at));
      c = to;
    }
  }
}

// Sum over the CTA in a fixed order; every thread gets it.
__device__ __forceinline__ double cta_sum(double v) {
  __shared__ double part[GC_THREADS / 32];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
  __syncthreads();
  double t = 0.0;
#pragma unroll
  for (int w = 0; w < GC_THREADS / 32; ++w) t += part[w];
  return t;
}

template <int MAX>
__global__ void __launch_bounds__(GC_THREADS) grad_squares_kernel(const __grid_constant__ GradList<MAX> l,
                                                                  double* partial) {
  pdl_enter();
  double all = 0.0;
  walk(l, [&](int t, int64_t at, int64_t n) {
    const int dt = l.dtype[t];
    if (dt == QL_F32) all += span_squares(static_cast<const float*>(l.grad[t]) + at, n);
    else if (dt == QL_F16) all += span_squares(static_cast<const __half*>(l.grad[t]) + at, n);
    else all += span_squares(static_cast<const __nv_bfloat16*>(l.grad[t]) + at, n);
  });
  const double sum = cta_sum(all);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

// The norm from the partial sums (the same in every CTA).
__device__ __forceinline__ float total_norm(const double* partial, int partials, float inv_scale) {
  double v = 0.0;
  for (int i = threadIdx.x; i < partials; i += GC_THREADS) v += partial[i];
  return (float)(sqrt(cta_sum(v)) * (double)inv_scale);
}

__global__ void __launch_bounds__(GC_THREADS) grad_norm_kernel(const double* partial, int partials,
                                                               float inv_scale, const float* inv_scale_dev,
                                                               float* norm) {
  pdl_enter();
  const float n = total_norm(partial, partials, inv_scale_dev != nullptr ? *inv_scale_dev : inv_scale);
  if (threadIdx.x == 0) *norm = n;
}

// V consecutive values as one access of 8 or 16 bytes
template <typename T, int V>
struct alignas(V * sizeof(T)) Vec {
  T e[V];
};

template <typename T, typename TO>
__device__ __forceinline__ void span_scale(const T* p, TO* o, int64_t n, float factor) {
  // 16 bytes of the wider type per access, so that a warp's stores are whole lines: with 16 bytes of
  // 16-bit gradients a thread's 32 bytes of fp32 went out as two half-filled sets of sectors
  constexpr int V = 16 / (sizeof(T) > sizeof(TO) ? sizeof(T) : sizeof(TO));
  int64_t done = 0;
  if (((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(o)) & 15) == 0) {
    const Vec<T, V>* v = reinterpret_cast<const Vec<T, V>*>(p);
    Vec<TO, V>* w = reinterpret_cast<Vec<TO, V>*>(o);
    const int64_t nv = n / V;
    auto put = [&](const Vec<T, V>& u, int64_t at) {
      Vec<TO, V> r;
#pragma unroll
      for (int e = 0; e < V; ++e) r.e[e] = from_f<TO>(to_f<T>(u.e[e]) * factor);
      w[at] = r;
    };
    int64_t i = threadIdx.x;
    for (; i + 7 * GC_THREADS < nv; i += 8 * GC_THREADS) {
      Vec<T, V> u[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) u[k] = v[i + k * GC_THREADS];
#pragma unroll
      for (int k = 0; k < 8; ++k) put(u[k], i + k * GC_THREADS);
    }
    for (; i < nv; i += GC_THREADS) put(v[i], i);
    done = nv * V;
  }
#pragma unroll 8
  for (int64_t i = done + threadIdx.x; i < n; i += GC_THREADS) o[i] = from_f<TO>(to_f<T>(p[i]) * factor);
}
template <typename T>
__device__ __forceinline__ void span_scale_to(const T* p, void* o, int out_dtype, int64_t at, int64_t n, float factor) {
  if (out_dtype == QL_F32) span_scale(p, static_cast<float*>(o) + at, n, factor);
  else if (out_dtype == QL_F16) span_scale(p, static_cast<__half*>(o) + at, n, factor);
  else span_scale(p, static_cast<__nv_bfloat16*>(o) + at, n, factor);
}

template <int MAX>
__global__ void __launch_bounds__(GC_THREADS, GC_CTAS_PER_SM) grad_scale_kernel(const __grid_constant__ GradList<MAX> l,
                                                                const double* partial, int partials,
                                                                float max_norm, float inv_scale,
                                                                const float* inv_scale_dev, float* norm,
                                                                int in_place, int write_norm) {
  pdl_enter();
  if (inv_scale_dev != nullptr) inv_scale = *inv_scale_dev;
  const float total = total_norm(partial, partials, inv_scale);
  if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  const float ratio = max_norm / (total + 1e-6f);
  const float factor = (ratio > 1.f ? 1.f : ratio) * inv_scale;  // a NaN stays one
  if (in_place && factor == 1.f) return;                         // every gradient stays as it is
  walk(l, [&](int t, int64_t at, int64_t n) {
    const int dt = l.dtype[t], odt = l.out_dtype[t];
    if (dt == QL_F32) span_scale_to(static_cast<const float*>(l.grad[t]) + at, l.out[t], odt, at, n, factor);
    else if (dt == QL_F16) span_scale_to(static_cast<const __half*>(l.grad[t]) + at, l.out[t], odt, at, n, factor);
    else span_scale_to(static_cast<const __nv_bfloat16*>(l.grad[t]) + at, l.out[t], odt, at, n, factor);
  });
}
constexpr int GC_SMALL = 128, GC_MAX = 1024;

int elem_bytes(int dtype) { return dtype == QL_F32 ? 4 : 2; }
bool dtype_ok(int dtype) { return dtype == QL_F16 || dtype == QL_BF16 || dtype == QL_F32; }

// Tensors [begin, end) of the call as kernel parameters; false if there are too many chunks.
template <int MAX>
bool fill_list(const GradTensors& t, int begin, int end, GradList<MAX>& l) {
  int64_t chunks = 0;
  l.count = end - begin;
  for (int i = begin; i < end; ++i) {
    const int k = i - begin;
    l.grad[k] = reinterpret_cast<const void*>(t.grads[i]);
    l.out[k] = t.outs != nullptr ? reinterpret_cast<void*>(t.outs[i]) : nullptr;
    l.n[k] = t.elements[i];
    l.dtype[k] = (uint8_t)t.dtypes[i];
    l.out_dtype[k] = t.outs != nullptr ? (uint8_t)t.out_dtypes[i] : 0;
    l.first[k] = (int32_t)chunks;
    chunks += cdiv(t.elements[i] * elem_bytes(t.dtypes[i]), GC_CHUNK);
    if (chunks > 0x3fffffff) return false;
  }
  l.first[l.count] = (int32_t)chunks;
  return true;
}

int grid_of(int chunks) { return (int)std::max<int64_t>(1, std::min<int64_t>(chunks, (int64_t)sm_count() * GC_CTAS_PER_SM)); }

struct ClipCall {
  float max_norm, inv_scale;
  const float* inv_scale_dev;
  float* norm;
  int in_place, partials;
  double* partial;
};

template <int MAX>
int squares(const GradTensors& t, int begin, int end, ClipCall& c, cudaStream_t s) {
  GradList<MAX> l;
  if (!fill_list(t, begin, end, l)) return QL_STATUS_UNSUPPORTED;
  const int grid = grid_of(l.first[l.count]);
  launch_k(grad_squares_kernel<MAX>, dim3(grid), dim3(GC_THREADS), 0, s, l, c.partial + c.partials);
  c.partials += grid;
  return launched(1);
}
template <int MAX>
int rescale(const GradTensors& t, int begin, int end, const ClipCall& c, cudaStream_t s) {
  GradList<MAX> l;
  if (!fill_list(t, begin, end, l)) return QL_STATUS_UNSUPPORTED;
  launch_k(grad_scale_kernel<MAX>, dim3(grid_of(l.first[l.count])), dim3(GC_THREADS), 0, s, l,
           (const double*)c.partial, c.partials, c.max_norm, c.inv_scale, c.inv_scale_dev, c.norm,
           c.in_place, begin == 0 ? 1 : 0);
  return launched(1);
}

int clip_check(const GradTensors& t, const float* norm, const double* ws, int64_t ws_bytes) {
  if (t.count < 0 || (t.count > 0 && (t.grads == nullptr || t.elements == nullptr || t.dtypes == nullptr)) ||
      norm == nullptr || ws == nullptr || (reinterpret_cast<uintptr_t>(ws) & 7) ||
      ws_bytes < grad_norm_workspace(t.count))
    return QL_STATUS_BAD_ARG;
  for (int i = 0; i < t.count; ++i)
    if (t.elements[i] < 0 || t.elements[i] > (int64_t)1 << 40 || (t.elements[i] > 0 && t.grads[i] == 0) ||
        !dtype_ok(t.dtypes[i]) || (t.grads[i] & (elem_bytes(t.dtypes[i]) - 1)))
      return QL_STATUS_BAD_ARG;
  return QL_STATUS_OK;
}

// Refuses a call where any two of the tensors written (or read beside one that is) share memory; an output
// that is its own gradient counts once.
int check_overlap(const GradTensors& t) {
  std::vector<std::pair<uint64_t, uint64_t>> spans;  // [first byte, end)
  try {
    spans.reserve(2 * (size_t)t.count);  // all that this function allocates
  } catch (const std::exception&) {
    return QL_STATUS_CUDA;  // no memory for it: an exception must not cross the C entry
  }
  for (int i = 0; i < t.count; ++i) {
    if (t.elements[i] == 0) continue;
    spans.emplace_back(t.grads[i], t.grads[i] + (uint64_t)t.elements[i] * elem_bytes(t.dtypes[i]));
    if (t.outs[i] != t.grads[i])
      spans.emplace_back(t.outs[i], t.outs[i] + (uint64_t)t.elements[i] * elem_bytes(t.out_dtypes[i]));
  }
  std::sort(spans.begin(), spans.end());
  for (size_t k = 1; k < spans.size(); ++k)
    if (spans[k].first < spans[k - 1].second) return QL_STATUS_BAD_ARG;
  return QL_STATUS_OK;
}

int all_squares(const GradTensors& t, ClipCall& c, cudaStream_t s) {
  const int count = t.count;
  for (int b = 0; b < count || b == 0; b += GC_MAX) {
    const int e = std::min(count, b + GC_MAX);
    const int st = e - b <= GC_SMALL ? squares<GC_SMALL>(t, b, e, c, s) : squares<GC_MAX>(t, b, e, c, s);
    if (st != QL_STATUS_OK) return st;
  }
  return QL_STATUS_OK;
}

}  // namespace

int64_t grad_norm_workspace(int count) {
  return std::max<int64_t>(1, cdiv(count, GC_MAX)) * sm_count() * GC_CTAS_PER_SM * (int64_t)sizeof(double);
}

int grad_norm(const GradTensors& t, float inv_scale, const float* inv_scale_dev, float* norm, double* ws,
              int64_t ws_bytes, cudaStream_t s) {
  int st = clip_check(t, norm, ws, ws_bytes);
  if (st != QL_STATUS_OK) return st;
  ProfScope prof(PK_OTHER, 0, 0, s);
  ClipCall c{0.f, inv_scale, inv_scale_dev, norm, 0, 0, ws};
  st = all_squares(t, c, s);
  if (st != QL_STATUS_OK) return st;
  launch_k(grad_norm_kernel, dim3(1), dim3(GC_THREADS), 0, s, (const double*)ws, c.partials, inv_scale,
           inv_scale_dev, norm);
  return launched(1);
}

int clip_grads(const GradTensors& t, float max_norm, float inv_scale, const float* inv_scale_dev, float* norm,
               double* ws, int64_t ws_bytes, cudaStream_t s) {
  int st = clip_check(t, norm, ws, ws_bytes);
  if (st != QL_STATUS_OK) return st;
  if (!(max_norm >= 0.f) || (t.count > 0 && (t.outs == nullptr || t.out_dtypes == nullptr)))
    return QL_STATUS_BAD_ARG;
  int in_place = 1;
  for (int i = 0; i < t.count; ++i) {
    if (t.elements[i] == 0) continue;
    if (t.outs[i] == 0 || !dtype_ok(t.out_dtypes[i]) || (t.outs[i] & (elem_bytes(t.out_dtypes[i]) - 1)) ||
        (t.outs[i] == t.grads[i] && t.out_dtypes[i] != t.dtypes[i]))
      return QL_STATUS_BAD_ARG;
    in_place &= t.outs[i] == t.grads[i];
  }
  st = check_overlap(t);
  if (st != QL_STATUS_OK) return st;
  ProfScope prof(PK_OTHER, 0, 0, s);
  ClipCall c{max_norm, inv_scale, inv_scale_dev, norm, in_place, 0, ws};
  st = all_squares(t, c, s);
  if (st != QL_STATUS_OK) return st;
  for (int b = 0; b < t.count || b == 0; b += GC_MAX) {
    const int e = std::min(t.count, b + GC_MAX);
    st = e - b <= GC_SMALL ? rescale<GC_SMALL>(t, b, e, c, s) : rescale<GC_MAX>(t, b, e, c, s);
    if (st != QL_STATUS_OK) return st;
  }
  return QL_STATUS_OK;
}

}  // namespace ql
