// AdamW over many tensors at once, moments in 32 bits or in 8:
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        (g: the gradient times a factor on the device)
//   w -= lr ( (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + weight_decay w )
// The tensors' addresses and lengths travel as the kernel's argument, so that a step is one launch for a few
// hundred tensors, copies nothing to the device and can be captured; CTAs walk over chunks of all of them.
//
// 8-bit moments: blocks of 256 values of a tensor are e4m3 numbers and one power of two, the smallest with which
// the block's largest value fits (448), at least 2^-126.  Numbers with an exponent of their own need no finer factor:
// dividing by a power of two is exact, so that a value is rounded once, by at most 2^-4 of itself, down to 2^-15 of
// the block's largest.  The second moment is held as its square root (twice the range in v), which does not
// become zero by rounding: a divisor of zero would turn the next small first moment into a huge step.
// The step itself uses the moments before they are rounded.  Products and sums of the moments are rounded to 32
// bits one by one, never fused: inputs of few bits lie on the borders between two 8-bit numbers often (0.9 m + 0.1 g:
// some 0.4 % of them), and which side is taken is then a property of the formula, not of the compiler.
//
// Bound by memory: 28 bytes per element with 16-bit weights, 32-bit masters and moments, 16 with 8-bit moments,
// 10 without masters.
#include <cuda_fp8.h>

#include "common.cuh"
#include "kernels.h"

namespace slapo {

constexpr int kAdamBlock = 256;                       // values per factor: a warp's 32 x 8
constexpr int kAdamThreads = 256;
constexpr int kAdamChunk = kAdamThreads * kVec;       // elements of a CTA's step

template <int N>
struct AdamBatch {
  AdamwTensor t[N];
  int first[N + 1];      // chunks before each tensor, and in all
  int count;
  AdamwScalars s;
};

// eight values from p on, of which `left` exist; whole: they do, on the boundaries that Vec8 needs
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int left, bool whole, float (&v)[8]) {
  if (whole) {
    Vec8<T>::load(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? static_cast<float>(p[i]) : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int left, bool whole, const float (&v)[8]) {
  if (whole) {
    Vec8<T>::store(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = static_cast<T>(v[i]);
  }
}

__device__ __forceinline__ void load_codes(const uint8_t* p, int left, bool whole, float scale, float (&v)[8]) {
  uint2 w = make_uint2(0u, 0u);
  if (whole) {
    w = *reinterpret_cast<const uint2*>(p);
  } else {
    uint8_t* b = reinterpret_cast<uint8_t*>(&w);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) b[i] = p[i];
  }
  const uint32_t words[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
        static_cast<__nv_fp8x2_storage_t>(words[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    v[2 * i] = f.x * scale;
    v[2 * i + 1] = f.y * scale;
  }
}

// The block's factor from its values (a warp's), and its codes.  A NaN stays one, in its own place.
template <bool kAboveZero>
__device__ __forceinline__ void store_codes(uint8_t* p, float* scale, int lane, int left, bool whole,
                                            const float (&v)[8]) {
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < 8; ++i) top = fmaxf(top, fabsf(v[i]));
  // (non-negative floats are ordered as their bits)
  const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));
  // largest = f 2^E with 1/2 <= f < 1: the factor is 2^(E - 9) for f <= 448 / 512, else 2^(E - 8)
  int e = static_cast<int>(bits >> 23) - 126 - 9;
  if ((bits & 0x7fffffu) > 0x600000u) ++e;
  e = max(e, -126);
  const float inv = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
  uint32_t words[2] = {0u, 0u};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    uint32_t c = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i] * inv, v[2 * i + 1] * inv), __NV_SATFINITE,
                                          __NV_E4M3);
    if (kAboveZero) {
      if ((c & 0x00ffu) == 0u && v[2 * i] > 0.f) c |= 0x0001u;
      if ((c & 0xff00u) == 0u && v[2 * i + 1] > 0.f) c |= 0x0100u;
    }
    words[i >> 1] |= c << (16 * (i & 1));
  }
  if (whole) {
    *reinterpret_cast<uint2*>(p) = make_uint2(words[0], words[1]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = static_cast<uint8_t>(words[i >> 2] >> (8 * (i & 3)));
  }
  if (lane == 0 && left > 0) *scale = __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

template <bool k8, typename T, int N>
__global__ void __launch_bounds__(kAdamThreads) adamw_multi_kernel(const __grid_constant__ AdamBatch<N> b) {
  float inv_bc1 = b.s.inv_bc1, inv_sqrt_bc2 = b.s.inv_sqrt_bc2;
  if (b.s.step != nullptr) {
    // the step's number on the device: a captured launch goes on counting
    __shared__ float bias[2];
    if (threadIdx.x < 2) {
      const double left = 1.0 - pow(threadIdx.x == 0 ? b.s.beta1_d : b.s.beta2_d, static_cast<double>(*b.s.step));
      bias[threadIdx.x] = static_cast<float>(threadIdx.x == 0 ? 1.0 / left : 1.0 / sqrt(left));
    }
    __syncthreads();
    inv_bc1 = bias[0];
    inv_sqrt_bc2 = bias[1];
  }
  const float gs = b.s.grad_scale != nullptr ? *b.s.grad_scale : 1.f;
  const int chunks = b.first[b.count], lane = threadIdx.x & 31;
  for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
    int lo = 0, hi = b.count;       // the tensor with first[lo] <= chunk < first[lo + 1]
    while (hi - lo > 1) {
      const int mid = (lo + hi) >> 1;
      if (b.first[mid] <= chunk) lo = mid;
      else hi = mid;
    }
    const AdamwTensor& t = b.t[lo];
    const int64_t at = static_cast<int64_t>(chunk - b.first[lo]) * kAdamChunk + threadIdx.x * kVec;
    const int64_t rest = t.n - at;
    const int left = rest < 0 ? 0 : (rest > kVec ? kVec : static_cast<int>(rest));
    const bool whole = t.aligned && left == kVec;
    float g[8], w[8], m[8], v[8];
    load_some(static_cast<const T*>(t.grad) + at, left, whole, g);
    if (t.master != nullptr) load_some(t.master + at, left, whole, w);
    else load_some(static_cast<const T*>(t.param) + at, left, whole, w);
    if constexpr (k8) {
      const int64_t block = at / kAdamBlock;      // (one per warp)
      const bool any = rest > -static_cast<int64_t>(lane * kVec);     // (the warp's first value exists)
      const float ms = any ? t.m_scale[block] : 0.f, vs = any ? t.v_scale[block] : 0.f;
      load_codes(static_cast<const uint8_t*>(t.m) + at, left, whole, ms, m);
      load_codes(static_cast<const uint8_t*>(t.v) + at, left, whole, vs, v);
    } else {
      load_some(static_cast<const float*>(t.m) + at, left, whole, m);
      load_some(static_cast<const float*>(t.v) + at, left, whole, v);
    }
    float u[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float x = __fmul_rn(g[i], gs);
      if (k8) v[i] = __fmul_rn(v[i], v[i]);
      m[i] = __fadd_rn(__fmul_rn(m[i], b.s.beta1), __fmul_rn(x, b.s.one_beta1));
      v[i] = __fadd_rn(__fmul_rn(v[i], b.s.beta2), __fmul_rn(__fmul_rn(x, x), b.s.one_beta2));
      u[i] = __fsqrt_rn(v[i]);
      const float step = __fdividef(m[i] * inv_bc1, fmaf(u[i], inv_sqrt_bc2, b.s.eps));
      w[i] = fmaf(-t.lr, fmaf(t.weight_decay, w[i], step), w[i]);
    }
    if (t.master != nullptr) store_some(t.master + at, left, whole, w);
    store_some(static_cast<T*>(t.param) + at, left, whole, w);
    if constexpr (k8) {
      const int64_t block = at / kAdamBlock;
      store_codes<false>(static_cast<uint8_t*>(t.m) + at, t.m_scale + block, lane, left, whole, m);
      store_codes<true>(static_cast<uint8_t*>(t.v) + at, t.v_scale + block, lane, left, whole, u);
    } else {
      store_some(static_cast<float*>(t.m) + at, left, whole, m);
      store_some(static_cast<float*>(t.v) + at, left, whole, v);
    }
  }
}

template <bool k8, typename T, int N>
static int launch_batch(const AdamwTensor* t, int n, const AdamwScalars& s, cudaStream_t stream) {
  AdamBatch<N> b;
  int64_t chunks = 0;
  for (int i = 0; i < n; ++i) {
    b.t[i] = t[i];
    b.first[i] = static_cast<int>(chunks);
    chunks += (t[i].n + kAdamChunk - 1) / kAdamChunk;
    if (chunks > 0x7fffffff) return 1;
  }
  b.first[n] = static_cast<int>(chunks);
  b.count = n;
  b.s = s;
  if (chunks == 0) return 0;
  const int64_t cap = static_cast<int64_t>(sm_count()) * 8;
  count_launch();
  adamw_multi_kernel<k8, T, N><<<static_cast<int>(chunks < cap ? chunks : cap), kAdamThreads, 0, stream>>>(b);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

#define DISPATCH_DTYPE(dtype, ...)                                   \
  switch (dtype) {                                                   \
    case 0: { using T = __nv_bfloat16; __VA_ARGS__; break; }         \
    case 1: { using T = __half; __VA_ARGS__; break; }                \
    default: { using T = float; __VA_ARGS__; break; }                \
  }

// A kernel's arguments end at 32764 bytes.
constexpr int kAdamMany = 360, kAdamFew = 48;
static_assert(sizeof(AdamBatch<kAdamMany>) <= 32764, "more tensors than a kernel's arguments hold");

int launch_adamw_multi(const AdamwTensor* t, int n, const AdamwScalars& s, bool bits8, int dtype,
                       cudaStream_t stream) {
  for (int at = 0; at < n; at += kAdamMany) {
    const int m = n - at < kAdamMany ? n - at : kAdamMany;
    int rc = 1;
#define ADAMW_MULTI_CASE(K8_)                                                                                     \
  DISPATCH_DTYPE(dtype, rc = m <= kAdamFew ? (launch_batch<K8_, T, kAdamFew>(t + at, m, s, stream))               \
                                           : (launch_batch<K8_, T, kAdamMany>(t + at, m, s, stream)))
    if (bits8) { ADAMW_MULTI_CASE(true); }
    else { ADAMW_MULTI_CASE(false); }
#undef ADAMW_MULTI_CASE
    if (rc != 0) return rc;
  }
  return 0;
}

}  // namespace slapo
