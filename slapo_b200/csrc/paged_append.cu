// New tokens' keys and values into a paged cache in 8 bits, keys rotated by their positions on the way, and their
// queries rotated beside them.
//
// A page holds `page` tokens of a sequence; for each side (keys, values) and head it has its tokens' values as e4m3
// numbers and one scale, a power of two: the smallest with which the largest value fits (448), at least 2^-100.  e4m3
// has an exponent of its own, so that a power of two costs none of its precision; and a page whose scale has to grow
// because a token's values are larger than all before has its codes multiplied by a power of two, which rounds only
// those that become denormal.  A page's first token starts its scale anew.
//
// Rounding: rotation in fp32, then once to e4m3 (at most 2^-4 of the value, the halves of its steps).  Values that are
// not finite are held as NaN and do not count for the scale.
//
// Bound by HBM for prompts (16 bits in, 8 bits out), by latency for a token.  A CTA takes one page of one side of one
// head: its new values stay in registers between the maximum and their codes.  Other CTAs of the launch rotate queries.
#include <cuda_fp8.h>

#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

constexpr int kThreads = 256;
constexpr int kLeast = -100;      // the least scale's exponent

// Eight values of a head from d0 on, to be rotated: cosine and sine of each, or none where nothing is rotated
struct Turn8 {
  float2 cs[8];
  int mode;        // 0: as they are; 1: halves, whole vectors; 2: halves, value by value; 3: neighbours
  int half, rotary, d0;
  __device__ __forceinline__ Turn8(int d0_, int rotary_, bool interleaved) : half(rotary_ / 2), rotary(rotary_), d0(d0_) {
    mode = d0 >= rotary ? 0 : interleaved ? 3 : half % 8 == 0 ? 1 : 2;
  }
  __device__ __forceinline__ void read(const float* table, int64_t pos) {
    if (mode == 0) return;
    const float2* row = reinterpret_cast<const float2*>(table) + pos * half;
    if (mode == 3) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        cs[j] = d0 + 2 * j < rotary ? row[d0 / 2 + j] : make_float2(1.f, 0.f);
      return;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int d = d0 + j;
      cs[j] = d < rotary ? row[d < half ? d : d - half] : make_float2(1.f, 0.f);
      if (d < half) cs[j].y = -cs[j].y;
    }
  }
  // from a token's entries in shared memory, `stride` float4 between those of a place (modes 1 and 3)
  __device__ __forceinline__ void take(const float4* token, int stride) {
    if (mode == 0) return;
    const int place = (mode == 3 || d0 < half ? d0 : d0 - half) / 8;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (mode == 3 && q >= 2) break;
      const float4 e = token[q * stride + place];
      cs[2 * q] = make_float2(e.x, e.y);
      cs[2 * q + 1] = make_float2(e.z, e.w);
    }
    if (mode == 1 && d0 < half) {
#pragma unroll
      for (int j = 0; j < 8; ++j) cs[j].y = -cs[j].y;
    }
  }
  // v: the values at d0 of the head `x`
  template <typename T>
  __device__ __forceinline__ void apply(const T* x, float (&v)[8]) const {
    if (mode == 0) return;
    if (mode == 3) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float a = v[2 * j], b = v[2 * j + 1];
        v[2 * j] = turned_value(a, cs[j].x, b, -cs[j].y);
        v[2 * j + 1] = turned_value(b, cs[j].x, a, cs[j].y);
      }
      return;
    }
    float o[8];
    if (mode == 1) {
      Vec8<T>::load(x + (d0 < half ? d0 + half : d0 - half), o);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        o[j] = d < rotary ? static_cast<float>(x[d < half ? d + half : d - half]) : 0.f;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = turned_value(v[j], cs[j].x, o[j], cs[j].y);
  }
};

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The exponent of the smallest power of two that holds `top` in 448 times
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 126 - ((bits & 0x7fffffu) <= 0x600000u ? 9 : 8);   // 448 = 0.875 * 2^9
  return e < kLeast ? kLeast : e;
}

__device__ __forceinline__ uint2 to_codes(const float (&v)[8], float factor) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    uint32_t parts[2];
#pragma unroll
    for (int p = 0; p < 2; ++p) {
      const int j = 4 * h + 2 * p;
      // (an infinity as a NaN: saturation would make a number of it)
      const float a = fabsf(v[j]) <= 3.402823466e38f ? v[j] * factor : __uint_as_float(0x7fffffffu);
      const float b = fabsf(v[j + 1]) <= 3.402823466e38f ? v[j + 1] * factor : __uint_as_float(0x7fffffffu);
      parts[p] = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
    }
    w[h] = parts[0] | (parts[1] << 16);
  }
  return make_uint2(w[0], w[1]);
}
__device__ __forceinline__ void from_codes(uint2 raw, float (&v)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = j < 2 ? raw.x : raw.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> (16 * (j & 1))), __NV_E4M3);
    const float2 f = __half22float2(__half2(h));
    v[2 * j] = f.x;
    v[2 * j + 1] = f.y;
  }
}

// How many new tokens a sequence brings and where its first one is
__device__ __forceinline__ void new_tokens(const PagedCache& c, int b, int64_t& start, int& count) {
  count = c.counts != nullptr ? min(max(c.counts[b], 0), c.n) : c.n;
  start = static_cast<int64_t>(c.lengths[b]) - count;
}

// Eight values as they are in memory
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void values(float (&v)[8]) const { Vec8<T>::load(reinterpret_cast<const T*>(w), v); }
};

// The heads [h0, h1) of a side of a page.  More than one row to a thread: the rotation's rows of the page's tokens go
// through shared memory, in the order in which lanes read them (16 bytes of each of the places of a token side by side).
template <typename T, int kRows>
__device__ __forceinline__ void append_page(const PagedAppend& a, int64_t tile, int per_cta) {
  const PagedCache& c = a.cache;
  extern __shared__ __align__(16) float4 s_rot[];
  __shared__ float s_top[2][kThreads / 32];
  const int side = static_cast<int>(tile & 1);
  tile >>= 1;
  const int groups = (c.heads + per_cta - 1) / per_cta;
  const int h0 = static_cast<int>(tile % groups) * per_cta, h1 = min(c.heads, h0 + per_cta);
  tile /= groups;
  const int spans = (c.n + c.page - 2) / c.page + 1;
  const int b = static_cast<int>(tile / spans);
  int64_t start;
  int count;
  new_tokens(c, b, start, count);
  const int64_t from = start > 0 ? start : 0, end = start + count;      // positions that are written
  const int64_t number = from / c.page + tile % spans;
  if (from >= end || number * c.page >= end || number >= c.table_pages) return;
  const int64_t id = c.table[static_cast<int64_t>(b) * c.table_pages + number];
  if (id < 0 || id >= c.n_pages) return;
  const int64_t first = number * c.page;
  const int held = static_cast<int>(from > first ? from - first : 0);             // the page's older tokens
  const int last = static_cast<int>(end - first < c.page ? end - first : c.page);
  const int places = c.pitch / 8, rows = kThreads / places;
  const int place = threadIdx.x % places, row = threadIdx.x / places;
  const int d0 = place * 8;
  const bool mine = row < rows, real = mine && d0 < c.dim;
  const int64_t* stride = side ? a.v_stride : a.k_stride;
  const T* x = static_cast<const T*>(side ? a.v : a.k) + b * stride[0] + (first - start) * stride[1] + d0;
  const int64_t head_bytes = static_cast<int64_t>(c.page) * c.pitch;
  uint8_t* codes = c.pages + (id * 2 + side) * c.heads * head_bytes + d0;
  float* scales = c.scales + (id * 2 + side) * c.heads;
  const bool turned = side == 0 && a.rot != nullptr;
  Turn8 turn(d0, turned ? a.rotary : 0, a.interleaved);
  const int half = a.rotary / 2, units = half / 2;                // float4 of a token's rotation
  const int parts = a.interleaved ? 2 : 4;                        // ... of a place
  const bool shared = kRows > 1 && turned && half % (2 * parts) == 0;
  if (shared) {
    for (int i = threadIdx.x; i < (last - held) * units; i += kThreads) {
      const int t = i / units, u = i - t * units;
      const int64_t pos = first + held + t;
      s_rot[t * units + (u % parts) * (units / parts) + u / parts] =
          pos < a.rot_rows ? reinterpret_cast<const float4*>(a.rot)[pos * units + u] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
  }
  auto slot_of = [&](int i) { return held + row + i * rows; };

  Raw8<T> next[kRows];
  auto fetch = [&](int h) {
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (real && slot_of(i) < last) next[i].load(x + h * stride[2] + slot_of(i) * stride[1]);
  };
  fetch(h0);
  for (int h = h0; h < h1; ++h) {
    const float old = held > 0 ? scales[h] : 0.f;
    float v[kRows][8];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
      const int slot = slot_of(i);
      if (!real || slot >= last) continue;
      next[i].values(v[i]);
      if (turned) {
        if (first + slot < a.rot_rows) {
          if (shared) turn.take(s_rot + (slot - held) * units, units / parts);
          else if (kRows > 1 || h == h0) turn.read(a.rot, first + slot);
          turn.apply(x + h * stride[2] + slot * stride[1] - d0, v[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float size = fabsf(v[i][j]);
        if (size <= 3.402823466e38f) top = fmaxf(top, size);
      }
    }
    if (h + 1 < h1) fetch(h + 1);
    top = warp_max(top);
    float* tops = s_top[h & 1];
    if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
    __syncthreads();      // (every thread has read the old scale, and is done with the tops of two heads before)
    top = tops[0];
#pragma unroll
    for (int w = 1; w < kThreads / 32; ++w) top = fmaxf(top, tops[w]);
    const int e = scale_exponent(top);
    const float need = power_of_two(e), scale = fmaxf(old, need);
    const float factor = scale == need ? power_of_two(-e) : 1.f / scale;
    if (threadIdx.x == 0) scales[h] = scale;
    uint8_t* to = codes + h * head_bytes;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (mine && slot_of(i) < last) *reinterpret_cast<uint2*>(to + slot_of(i) * c.pitch) = to_codes(v[i], factor);
    if (held > 0 && scale != old && mine) {
      const float ratio = old * factor;
      for (int slot = row; slot < held; slot += rows) {
        uint2* at = reinterpret_cast<uint2*>(to + slot * c.pitch);
        float w[8];
        from_codes(*at, w);
        *at = to_codes(w, ratio);
      }
    }
  }
}

// The queries of a token
template <typename T>
__device__ __forceinline__ void append_query(const PagedAppend& a, int64_t token) {
  const PagedCache& c = a.cache;
  const int b = static_cast<int>(token / c.n), t = static_cast<int>(token - static_cast<int64_t>(b) * c.n);
  int64_t start;
  int count;
  new_tokens(c, b, start, count);
  const int64_t pos = start + t;
  const bool turned = a.rot != nullptr;
  const bool known = t < count && pos >= 0 && (!turned || pos < a.rot_rows);
  const int places = c.dim / 8, rows = kThreads / places;
  const int place = threadIdx.x % places, row = threadIdx.x / places;
  if (row >= rows) return;
  Turn8 turn(place * 8, turned ? a.rotary : 0, a.interleaved);
  if (known && turned) turn.read(a.rot, pos);
  const T* x = static_cast<const T*>(a.q) + b * a.q_stride[0] + t * a.q_stride[1];
  T* y = static_cast<T*>(a.q_out) + token * a.q_heads * c.dim;
  for (int h = row; h < a.q_heads; h += rows) {
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (known) {
      const T* xh = x + h * a.q_stride[2];
      Vec8<T>::load(xh + place * 8, v);
      turn.apply(xh, v);
    }
    Vec8<T>::store(y + static_cast<int64_t>(h) * c.dim + place * 8, v);
  }
}

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads, kRows <= 2 ? 3 : kRows <= 4 ? 2 : 1) paged_append_kernel(const PagedAppend a, int64_t tiles, int per_cta) {
  if (blockIdx.x < tiles) append_page<T, kRows>(a, blockIdx.x, per_cta);
  else append_query<T>(a, blockIdx.x - tiles);
}

template <typename T, int kRows>
int launch_rows(const PagedAppend& a, int64_t tiles, int per_cta, unsigned grid, cudaStream_t stream) {
  auto kernel = paged_append_kernel<T, kRows>;
  int bytes = 0;
  if (kRows > 1 && a.rot != nullptr) {
    bytes = (a.cache.n < a.cache.page ? a.cache.n : a.cache.page) * a.rotary * 4;
    if (bytes > 48 * 1024) {
      int device = 0;
      if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 3;
      static bool configured[64] = {};
      if (!configured[device]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024) != cudaSuccess) return 3;
        configured[device] = true;
      }
    }
  }
  count_launch();
  kernel<<<grid, kThreads, bytes, stream>>>(a, tiles, per_cta);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

template <typename T>
int launch(const PagedAppend& a_in, cudaStream_t stream) {
  PagedAppend a = a_in;
  const PagedCache& c = a.cache;
  const int64_t spans = (c.n + c.page - 2) / c.page + 1, pages = c.B * spans * 2;
  // Many tokens: their queries by the rotation's own kernel, which has more bytes on their way.  (Few: one launch.)
  if (a.q != nullptr && a.rot != nullptr && static_cast<int64_t>(c.B) * c.n >= 4 * sm_count()) {
    RotaryCall r{};
    RotaryPart& p = r.part[0];
    p.x = a.q;
    p.y = a.q_out;
    for (int d = 0; d < 3; ++d) p.x_stride[d] = a.q_stride[d];
    p.y_stride[2] = c.dim;
    p.y_stride[1] = static_cast<int64_t>(a.q_heads) * c.dim;
    p.y_stride[0] = p.y_stride[1] * c.n;
    p.heads = a.q_heads;
    p.turn = true;
    r.parts = 1;
    r.table = a.rot;
    r.table_rows = a.rot_rows;
    r.at.lengths = c.lengths;
    r.at.counts = c.counts;
    r.B = c.B;
    r.S = c.n;
    r.D = c.dim;
    r.rotary = a.rotary;
    r.interleaved = a.interleaved;
    r.dtype = a.dtype;
    const int rc = launch_rotary(r, stream);
    if (rc != 0) return rc;
    a.q = nullptr;
  }
  // as many heads to a CTA as leave each SM some CTAs: they share the rotation's rows
  int per_cta = 8;
  while (per_cta > 1 && pages * ((c.heads + per_cta - 1) / per_cta) < 6 * sm_count()) per_cta /= 2;
  const int64_t tiles = pages * ((c.heads + per_cta - 1) / per_cta);
  const int64_t ctas = tiles + (a.q != nullptr ? static_cast<int64_t>(c.B) * c.n : 0);
  if (ctas > 0x7fffffff) return 5;
  if (ctas == 0) return 0;
  const unsigned grid = static_cast<unsigned>(ctas);
  const int rows = kThreads / (c.pitch / 8);
  const int most = c.n < c.page ? c.n : c.page;           // new tokens of a page
  const int per = (most + rows - 1) / rows;
  if (per <= 1) return launch_rows<T, 1>(a, tiles, per_cta, grid, stream);
  if (per <= 2) return launch_rows<T, 2>(a, tiles, per_cta, grid, stream);
  if (per <= 4) return launch_rows<T, 4>(a, tiles, per_cta, grid, stream);
  if (per <= 8) return launch_rows<T, 8>(a, tiles, per_cta, grid, stream);
  return 6;
}

}  // namespace

int launch_paged_append(const PagedAppend& a, cudaStream_t stream) {
  const PagedCache& c = a.cache;
  if (c.B == 0 || c.n == 0) return 0;
  if (c.dim < 8 || c.dim > 128 || c.dim % 8 != 0 || c.pitch != (c.dim + 15) / 16 * 16) return 1;
  if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128) return 2;
  if (a.rot != nullptr && (a.rotary < 2 || a.rotary % 2 != 0 || a.rotary > c.dim)) return 3;
  switch (a.dtype) {
    case 0: return launch<__nv_bfloat16>(a, stream);
    case 1: return launch<__half>(a, stream);
    case 2: return launch<float>(a, stream);
    default: return 7;
  }
}

}  // namespace slapo
