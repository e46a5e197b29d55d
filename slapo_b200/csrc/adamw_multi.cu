// AdamW over many tensors at once, moments in 32 bits or in 8:
//   m = b1 m + (1 - b1) g        v = b2 v + (1 - b2) g^2        (g: the gradient times a factor on the device)
//   w -= lr ( (m / (1 - b1^t)) / (sqrt(v / (1 - b2^t)) + eps) + weight_decay w )
// The tensors' addresses and lengths travel as the kernel's argument, so that a step is one launch for a few
// hundred tensors, copies nothing to the device and can be captured; warps walk over all of them together.
//
// 8-bit moments: blocks of 256 values of a tensor are e4m3 numbers and one power of two, the smallest with which
// the block's largest value fits (448), at least 2^-126.  Numbers with an exponent of their own need no finer factor:
// dividing by a power of two is exact, so that a value is rounded once, by at most 2^-4 of itself, down to 2^-15 of
// the block's largest.  The second moment is held as its square root (twice the range in v), which does not
// become zero by rounding: a divisor of zero would turn the next small first moment into a huge step.
// The step itself uses the moments before they are rounded.  Products and sums of the moments are rounded to 32
// bits one by one, never fused: inputs of few bits lie on the borders between two 8-bit numbers often (0.9 m + 0.1 g:
// some 0.4 % of them), and which side is taken is then a property of the formula, not of the compiler.  (The square
// root is within a unit in the last place: next to a border, 2^-20 of all, either side.)
//
// Bound by memory: 28 bytes per element with 16-bit weights, 32-bit masters and moments, 16 with 8-bit moments,
// 10 without masters; with 8-bit moments by instructions too, some 45 per element (a scheduler's slots are three
// quarters full at 10 bytes).
// Measured: 183 M elements, 12 layers of 1024: 32-bit moments and masters 812 - 820 us (96 % of the copy
// rate), 8-bit moments 490 - 499 us (90 - 92 %); 304 M elements, 8-bit, no masters: 560 - 588 us (80 - 84 %), from box to box.
#include <cuda_fp8.h>

#include <type_traits>

#include "common.cuh"
#include "kernels.h"

namespace slapo {

constexpr int kAdamBlock = 256;                       // values per factor: a warp's 32 x 8
constexpr int kAdamUnit = 2, kAdamUnitSize = kAdamUnit * kAdamBlock;      // blocks that a warp takes at a time
constexpr int kAdamThreads = 256, kAdamWarps = kAdamThreads / 32;

constexpr int kAdam32Unit = kAdamThreads * kVec;      // elements of a CTA's step in the other kernel

template <int N>
struct AdamBatch {
  AdamwTensor t[N];
  int first[N + 1];      // units before each tensor, and in all
  int count;
  AdamwScalars s;
};

// Eight values of a tensor as they are in memory; stored as whole words where a block is whole, else element by element
// (`left` of them)
template <typename T>
struct Raw {
  static constexpr int kWords = 8 * sizeof(T) / 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kWords == 2) {
      const uint2 x = *reinterpret_cast<const uint2*>(p);
      w[0] = x.x; w[1] = x.y;
    } else {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 x = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint32_t*>(p) + i);
        w[i] = x.x; w[i + 1] = x.y; w[i + 2] = x.z; w[i + 3] = x.w;
      }
    }
  }
  __device__ __forceinline__ void store(T* p, int left, bool whole) const {
    if (whole) {
      if constexpr (kWords == 2) {
        *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
      } else {
#pragma unroll
        for (int i = 0; i < kWords; i += 4)
          *reinterpret_cast<uint4*>(reinterpret_cast<uint32_t*>(p) + i) = make_uint4(w[i], w[i + 1], w[i + 2], w[i + 3]);
      }
    } else {
      const T* e = reinterpret_cast<const T*>(w);
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < left) p[i] = e[i];
    }
  }
  __device__ __forceinline__ float2 get(int i) const {      // values 2 i and 2 i + 1
    if constexpr (sizeof(T) == 4) return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
    else return pair_floats(w[i], T());
  }
  __device__ __forceinline__ void set(int i, float a, float b) {
    if constexpr (sizeof(T) == 4) {
      w[2 * i] = __float_as_uint(a);
      w[2 * i + 1] = __float_as_uint(b);
    } else {
      w[i] = pair_word(a, b, T());
    }
  }
};

__device__ __forceinline__ float2 codes_get(const Raw<uint8_t>& r, int i) {
  const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(
      static_cast<__nv_fp8x2_storage_t>(r.w[i >> 1] >> (16 * (i & 1))), __NV_E4M3);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// A block's codes from its values (a warp's), and its factor.  A NaN stays one, in its own place.
template <bool kAboveZero>
__device__ __forceinline__ float codes_set(Raw<uint8_t>& r, const float (&v)[8]) {
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
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const float* x = v + 4 * i;
    const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(x[0] * inv, x[1] * inv), __NV_SATFINITE, __NV_E4M3);
    const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(x[2] * inv, x[3] * inv), __NV_SATFINITE, __NV_E4M3);
    uint32_t c = low | high << 16;
    if (kAboveZero && ((c - 0x01010101u) & ~c & 0x80808080u) != 0u) {      // (some byte is zero)
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if ((c >> (8 * k) & 0xffu) == 0u && x[k] > 0.f) c |= 1u << (8 * k);
    }
    r.w[i] = c;
  }
  return __uint_as_float(static_cast<uint32_t>(127 + e) << 23);
}

// A unit's operands in shared memory
template <bool kMaster, typename T>
struct alignas(16) AdamStage {
  using Weight = typename std::conditional<kMaster, float, T>::type;
  T g[kAdamUnitSize];
  Weight w[kAdamUnitSize];
  uint8_t m[kAdamUnitSize], v[kAdamUnitSize];
  float scale[2][kAdamUnit];
};

// A CTA's ring, how many of them an SM holds, and how many launches' worth of resident CTAs the units are dealt out to.
// 16-bit weights: three CTAs and one sweep (324 us for 183 M elements; two sweeps 332).  With masters two CTAs fit, and
// four sweeps, each by CTAs that start as those before end, beat one: 490 for 545 us, 24 layers 900 for 1008, 4 layers of 2048
// 820 for 936 (eight: 474, 875, 777, but 12 layers of 768 372 for 357).  fp32 weights: one CTA, and a unit more on its way:
// 480 for 525 us with three in the ring, two CTAs of two each 568.
template <bool kMaster, typename T>
struct AdamRing {
  using Stage = AdamStage<kMaster, T>;
  static constexpr int kDepth = sizeof(T) == 4 ? 4 : 3;                   // units of a warp in shared memory
  static constexpr int kSmem = kAdamWarps * kDepth * static_cast<int>(sizeof(Stage));
  static constexpr int kCtas = sizeof(T) == 4 ? 1 : kMaster ? 2 : 3, kSweeps = kMaster ? 4 : 1;
  static_assert(kCtas * (kSmem + 1024 + 16) <= 228 * 1024, "8-bit AdamW: shared memory of the CTAs on an SM");
};

__device__ __forceinline__ void copy_async16(void* dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
__device__ __forceinline__ void copy_async4(void* dst, const void* src) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(static_cast<uint32_t>(__cvta_generic_to_shared(dst))),
               "l"(src)
               : "memory");
}
// a warp's copy of kBytes, 16 bytes to a lane
template <int kBytes>
__device__ __forceinline__ void copy_block(void* dst, const void* src, int lane) {
#pragma unroll
  for (int i = 0; i < kBytes; i += 512)
    copy_async16(static_cast<uint8_t*>(dst) + i + lane * 16, static_cast<const uint8_t*>(src) + i + lane * 16);
}

// Unit `unit` of a tensor on its way to shared memory, where it is whole and on the boundaries that copies need
template <bool kMaster, typename T>
__device__ __forceinline__ void fetch_unit(const AdamwTensor& t, int unit, AdamStage<kMaster, T>& to) {
  const int lane = threadIdx.x & 31;
  const int64_t at = static_cast<int64_t>(unit) * kAdamUnitSize;
  copy_block<kAdamUnitSize * sizeof(T)>(to.g, static_cast<const T*>(t.grad) + at, lane);
  if constexpr (kMaster) copy_block<kAdamUnitSize * 4>(to.w, t.master + at, lane);
  else copy_block<kAdamUnitSize * sizeof(T)>(to.w, static_cast<const T*>(t.param) + at, lane);
  copy_block<kAdamUnitSize>(to.m, static_cast<const uint8_t*>(t.m) + at, lane);
  copy_block<kAdamUnitSize>(to.v, static_cast<const uint8_t*>(t.v) + at, lane);
  if (lane < 2 * kAdamUnit)
    copy_async4(&to.scale[0][0] + lane,
                (lane < kAdamUnit ? t.m_scale : t.v_scale - kAdamUnit) + static_cast<int64_t>(unit) * kAdamUnit + lane);
}
// ... and element by element where not, zeros behind the tensor's end
template <bool kMaster, typename T>
__device__ __noinline__ void gather_unit(const AdamwTensor& t, int unit, AdamStage<kMaster, T>& to) {
  const int lane = threadIdx.x & 31;
  for (int i = lane; i < kAdamUnitSize; i += 32) {
    const int64_t at = static_cast<int64_t>(unit) * kAdamUnitSize + i;
    const bool ok = at < t.n;
    to.g[i] = ok ? static_cast<const T*>(t.grad)[at] : static_cast<T>(0.f);
    if constexpr (kMaster) to.w[i] = ok ? t.master[at] : 0.f;
    else to.w[i] = ok ? static_cast<const T*>(t.param)[at] : static_cast<T>(0.f);
    to.m[i] = ok ? static_cast<const uint8_t*>(t.m)[at] : static_cast<uint8_t>(0);
    to.v[i] = ok ? static_cast<const uint8_t*>(t.v)[at] : static_cast<uint8_t>(0);
  }
  const int64_t block = static_cast<int64_t>(unit) * kAdamUnit + lane % kAdamUnit;
  if (lane < 2 * kAdamUnit && block * kAdamBlock < t.n)
    to.scale[lane / kAdamUnit][lane % kAdamUnit] = (lane < kAdamUnit ? t.m_scale : t.v_scale)[block];
}

// The quotients and roots of the two kernels.  With 32-bit moments denormals count, so that eps may be as small as one likes,
// 0 included; both are within two units in the last place.  (Rounded correctly they cost 1 % of the time: 823 us for
// 815.)  With 8-bit moments instructions count: a second moment below 2^-126 is zero and the divisor never that small (the
// caller has looked at eps).
template <bool k8> __device__ __forceinline__ float square_root(float x) {
  float r;
  if constexpr (k8) asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  else asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
template <bool k8> __device__ __forceinline__ float quotient(float x, float y) {
  float r;
  if constexpr (k8) {
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(y));
    r *= x;
  } else {
    asm("div.full.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(y));
  }
  return r;
}

// What does not change over a launch
struct AdamStepScalars {
  float beta1, one_beta1, beta2, one_beta2, eps, inv_bc1, inv_sqrt_bc2, grad_scale;
};
__device__ __forceinline__ AdamStepScalars adam_scalars(const AdamwScalars& s) {
  AdamStepScalars c{s.beta1, s.one_beta1, s.beta2, s.one_beta2, s.eps, s.inv_bc1, s.inv_sqrt_bc2,
                    s.grad_scale != nullptr ? *s.grad_scale : 1.f};
  if (s.step != nullptr) {
    // the step's number on the device: a captured launch goes on counting
    __shared__ float bias[2];
    if (threadIdx.x < 2) {
      const double left = 1.0 - pow(threadIdx.x == 0 ? s.beta1_d : s.beta2_d, static_cast<double>(*s.step));
      bias[threadIdx.x] = static_cast<float>(threadIdx.x == 0 ? 1.0 / left : 1.0 / sqrt(left));
    }
    __syncthreads();
    c.inv_bc1 = bias[0];
    c.inv_sqrt_bc2 = bias[1];
  }
  return c;
}

// One element: its moments m and v brought up to date, u = sqrt(v), and the new weight
template <bool k8>
__device__ __forceinline__ float adam_value(float g, float w, float& m, float& v, float& u, const AdamwTensor& t,
                                            const AdamStepScalars& c) {
  const float x = __fmul_rn(g, c.grad_scale);
  m = __fadd_rn(__fmul_rn(m, c.beta1), __fmul_rn(x, c.one_beta1));
  v = __fadd_rn(__fmul_rn(v, c.beta2), __fmul_rn(__fmul_rn(x, x), c.one_beta2));
  u = square_root<k8>(v);
  const float step = quotient<k8>(m * c.inv_bc1, fmaf(u, c.inv_sqrt_bc2, c.eps));
  return fmaf(-t.lr, fmaf(t.weight_decay, w, step), w);
}

// The step of a block that has come to shared memory, eight elements to a lane
template <bool kMaster, typename T>
__device__ __forceinline__ void adam_block(const AdamwTensor& t, const AdamStepScalars& c, int unit, int sub, bool whole,
                                           const AdamStage<kMaster, T>& from) {
  const int lane = threadIdx.x & 31;
  const int64_t block = static_cast<int64_t>(unit) * kAdamUnit + sub, at = block * kAdamBlock + lane * kVec;
  Raw<T> g, p_new;
  Raw<typename AdamStage<kMaster, T>::Weight> w, w_new;
  Raw<uint8_t> m_codes, v_codes;
  g.load(from.g + sub * kAdamBlock + lane * kVec);
  w.load(from.w + sub * kAdamBlock + lane * kVec);
  m_codes.load(from.m + sub * kAdamBlock + lane * kVec);
  v_codes.load(from.v + sub * kAdamBlock + lane * kVec);
  const float m_scale = from.scale[0][sub], v_scale = from.scale[1][sub];
  const int left = whole ? kVec : static_cast<int>(max(int64_t(0), min(int64_t(kVec), t.n - at)));
  float m[8], u[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 g2 = g.get(i), w2 = w.get(i), m2 = codes_get(m_codes, i), u2 = codes_get(v_codes, i);
    const float x[2] = {g2.x, g2.y};
    float y[2] = {w2.x, w2.y};
    m[2 * i] = m2.x; m[2 * i + 1] = m2.y;
    u[2 * i] = u2.x; u[2 * i + 1] = u2.y;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const int e = 2 * i + k;
      m[e] = __fmul_rn(m[e], m_scale);
      u[e] = __fmul_rn(u[e], v_scale);
      float v = __fmul_rn(u[e], u[e]);
      y[k] = adam_value<true>(x[k], y[k], m[e], v, u[e], t, c);
    }
    if constexpr (kMaster) w_new.set(i, y[0], y[1]);
    p_new.set(i, y[0], y[1]);
  }
  if constexpr (kMaster) w_new.store(t.master + at, left, whole);
  p_new.store(static_cast<T*>(t.param) + at, left, whole);
  const float ms = codes_set<false>(m_codes, m);
  m_codes.store(static_cast<uint8_t*>(t.m) + at, left, whole);
  const float vs = codes_set<true>(v_codes, u);
  v_codes.store(static_cast<uint8_t*>(t.v) + at, left, whole);
  if (lane == 0 && left > 0) {
    t.m_scale[block] = ms;
    t.v_scale[block] = vs;
  }
}

// 8-bit moments.  A warp's units come into its part of shared memory some ahead of the one that it is at: bytes on
// their way take no registers, which the arithmetic needs.  (us for the two cases above.  Loads straight into registers,
// 40 warps per SM: 616 and 905; 16 warps that fetch a block ahead into registers: 636 and 737.  Through shared memory with a
// stretch of 16 blocks for each warp: 665 and 766 - thousands of places in memory at a time -, one sweep of all
// warps: 583 and 660, two blocks at a time: 564 and 593.)
template <bool kMaster, typename T, int N>
__global__ void __launch_bounds__(kAdamThreads, AdamRing<kMaster, T>::kCtas)
adamw8_kernel(const __grid_constant__ AdamBatch<N> b) {
  extern __shared__ uint4 adam_smem[];
  using Stage = AdamStage<kMaster, T>;
  constexpr int kAdamDepth = AdamRing<kMaster, T>::kDepth;
  Stage* ring = reinterpret_cast<Stage*>(adam_smem) + (threadIdx.x >> 5) * kAdamDepth;
  const AdamStepScalars c = adam_scalars(b.s);
  // Neighbouring warps take neighbouring units, the resident ones a sweep over the tensors: memory is read page by page.
  const int units = b.first[b.count], first = blockIdx.x * kAdamWarps + (threadIdx.x >> 5);
  const int stride = gridDim.x * kAdamWarps;
  auto seek = [&](int at, int tensor) {      // the tensor with first[tensor] <= at < first[tensor + 1], from there on
    while (b.first[tensor + 1] <= at) ++tensor;
    return tensor;
  };
  auto in_copies = [&](int unit, int tensor) {
    return b.t[tensor].aligned && static_cast<int64_t>(unit + 1) * kAdamUnitSize <= b.t[tensor].n;
  };
  int ahead = first, ahead_tensor = 0, slot = 0;
  auto fetch = [&](Stage& to) {
    if (ahead < units) {
      ahead_tensor = seek(ahead, ahead_tensor);
      const int unit = ahead - b.first[ahead_tensor];
      if (in_copies(unit, ahead_tensor)) fetch_unit(b.t[ahead_tensor], unit, to);
      else gather_unit(b.t[ahead_tensor], unit, to);
      ahead += stride;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kAdamDepth - 1; ++i) fetch(ring[i]);
  for (int at = first, tensor = 0; at < units; at += stride) {
    fetch(ring[slot == 0 ? kAdamDepth - 1 : slot - 1]);       // (read before the last __syncwarp)
    asm volatile("cp.async.wait_group %0;" ::"n"(kAdamDepth - 1) : "memory");
    __syncwarp();
    tensor = seek(at, tensor);
    const int unit = at - b.first[tensor];
    const bool whole = in_copies(unit, tensor);
#pragma unroll 2
    for (int sub = 0; sub < kAdamUnit; ++sub)
      adam_block(b.t[tensor], c, unit, sub, whole, ring[slot]);
    __syncwarp();
    slot = slot + 1 == kAdamDepth ? 0 : slot + 1;
  }
}

// Eight values that are read or written once: 32 bytes of fp32 in one request (two of 16 hold such a kernel at 84 % of
// the copy rate, elementwise.cu), 16 of 16-bit ones
__device__ __forceinline__ void load_once(const float* p, float (&v)[8]) {
  asm volatile("ld.global.cs.v8.f32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}
__device__ __forceinline__ void store_once(float* p, const float (&v)[8]) {
  asm volatile("st.global.cs.v8.f32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}
template <typename T> __device__ __forceinline__ void load_once(const T* p, float (&v)[8]) { Vec8<T>::load(p, v); }
template <typename T> __device__ __forceinline__ void store_once(T* p, const float (&v)[8]) { Vec8<T>::store(p, v); }

// Moments in 32 bits: bytes alone, a CTA's 2048 elements at a time straight from memory.
template <bool kMaster, typename T, int N>
__global__ void __launch_bounds__(kAdamThreads) adamw32_kernel(const __grid_constant__ AdamBatch<N> b) {
  const AdamStepScalars c = adam_scalars(b.s);
  const int units = b.first[b.count];
  for (int unit = blockIdx.x, tensor = 0; unit < units; unit += gridDim.x) {
    while (b.first[tensor + 1] <= unit) ++tensor;
    const AdamwTensor& t = b.t[tensor];
    const int64_t begin = static_cast<int64_t>(unit - b.first[tensor]) * kAdam32Unit;
    T* param = static_cast<T*>(t.param);
    const T* grad = static_cast<const T*>(t.grad);
    float* exp_avg = static_cast<float*>(t.m);
    float* exp_avg_sq = static_cast<float*>(t.v);
    if (t.aligned && begin + kAdam32Unit <= t.n) {
      const int64_t at = begin + threadIdx.x * kVec;
      float g[8], w[8], m[8], v[8];
      load_once(grad + at, g);
      if constexpr (kMaster) load_once(t.master + at, w);
      else load_once(param + at, w);
      load_once(exp_avg + at, m);
      load_once(exp_avg_sq + at, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float u;
        w[i] = adam_value<false>(g[i], w[i], m[i], v[i], u, t, c);
      }
      if constexpr (kMaster) store_once(t.master + at, w);
      store_once(param + at, w);
      store_once(exp_avg + at, m);
      store_once(exp_avg_sq + at, v);
    } else {      // a tensor's end, or one that begins anywhere: element by element
      const int64_t end = min(t.n, begin + kAdam32Unit);
#pragma unroll 2
      for (int64_t at = begin + threadIdx.x; at < end; at += kAdamThreads) {
        float m = exp_avg[at], v = exp_avg_sq[at], u;
        float w = kMaster ? t.master[at] : static_cast<float>(param[at]);
        w = adam_value<false>(static_cast<float>(grad[at]), w, m, v, u, t, c);
        if constexpr (kMaster) t.master[at] = w;
        param[at] = static_cast<T>(w);
        exp_avg[at] = m;
        exp_avg_sq[at] = v;
      }
    }
  }
}

template <bool k8, bool kMaster, typename T, int N>
static int launch_batch(const AdamwTensor* t, int n, const AdamwScalars& s, cudaStream_t stream) {
  constexpr int kUnit = k8 ? kAdamUnitSize : kAdam32Unit;
  AdamBatch<N> b;
  int64_t units = 0;
  for (int i = 0; i < n; ++i) {
    b.t[i] = t[i];
    b.first[i] = static_cast<int>(units);
    units += (t[i].n + kUnit - 1) / kUnit;
    if (units > 0x3fffffff) return 1;
  }
  b.first[n] = static_cast<int>(units);
  b.count = n;
  b.s = s;
  if (units == 0) return 0;
  count_launch();
  if constexpr (k8) {
    using Ring = AdamRing<kMaster, T>;
    constexpr int kSmem = Ring::kSmem;
    auto kernel = adamw8_kernel<kMaster, T, N>;
    // (of the current device; cheap beside a launch)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem) != cudaSuccess) return 3;
    const int64_t ctas = (units + kAdamWarps - 1) / kAdamWarps;
    const int64_t cap = static_cast<int64_t>(sm_count()) * Ring::kCtas * Ring::kSweeps;
    kernel<<<static_cast<int>(ctas < cap ? ctas : cap), kAdamThreads, kSmem, stream>>>(b);
  } else {
    const int64_t cap = static_cast<int64_t>(sm_count()) * 16;
    adamw32_kernel<kMaster, T, N><<<static_cast<int>(units < cap ? units : cap), kAdamThreads, 0, stream>>>(b);
  }
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

// A kernel's arguments end at 32764 bytes.
constexpr int kAdamMany = 360, kAdamFew = 60;
static_assert(sizeof(AdamBatch<kAdamMany>) <= 32764, "more tensors than a kernel's arguments hold");

template <bool k8, bool kMaster, typename T>
static int launch_many(const AdamwTensor* t, int n, const AdamwScalars& s, cudaStream_t stream) {
  for (int at = 0; at < n; at += kAdamMany) {
    const int m = n - at < kAdamMany ? n - at : kAdamMany;
    const int rc = m <= kAdamFew ? launch_batch<k8, kMaster, T, kAdamFew>(t + at, m, s, stream)
                                 : launch_batch<k8, kMaster, T, kAdamMany>(t + at, m, s, stream);
    if (rc != 0) return rc;
  }
  return 0;
}

template <bool k8, typename T>
static int launch_typed(const AdamwTensor* t, int n, const AdamwScalars& s, bool master, cudaStream_t stream) {
  if constexpr (sizeof(T) == 2)
    if (master) return launch_many<k8, true, T>(t, n, s, stream);
  return master ? 1 : launch_many<k8, false, T>(t, n, s, stream);
}

// (all tensors have masters, or none)
int launch_adamw_multi(const AdamwTensor* t, int n, const AdamwScalars& s, bool bits8, int dtype, cudaStream_t stream) {
  if (n <= 0) return 0;
  const bool master = t[0].master != nullptr;
  switch (dtype) {
    case 0: return bits8 ? launch_typed<true, __nv_bfloat16>(t, n, s, master, stream)
                         : launch_typed<false, __nv_bfloat16>(t, n, s, master, stream);
    case 1: return bits8 ? launch_typed<true, __half>(t, n, s, master, stream)
                         : launch_typed<false, __half>(t, n, s, master, stream);
    default: return bits8 ? launch_typed<true, float>(t, n, s, master, stream)
                          : launch_typed<false, float>(t, n, s, master, stream);
  }
}

}  // namespace slapo
