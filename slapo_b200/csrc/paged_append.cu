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
// Bound by HBM for prompts (16 bits in, 8 bits out), by latency for a token.  A CTA takes one page of one side, and of some
// heads one after the other: their new values stay in registers between the maximum and their codes, the next head's
// are read under the barrier.  Other CTAs of the launch rotate (or copy) queries, or, where tokens are many, rotary.cu's kernel
// beside it.
// 8 x 2048 tokens of 16 heads of 128, bf16, pages of 64: 55 us, with their queries 77 (floor 51); one token each 6.3, the host's time.
#include <cuda_fp8.h>

#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

constexpr int kThreads = 256;     // of a CTA, at most
constexpr int kLeast = -100;      // the least scale's exponent

// Eight values as they are in memory
template <typename T>
struct Raw8 {
  uint4 w[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) {
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) w[i] = reinterpret_cast<const uint4*>(p)[i];
  }
  __device__ __forceinline__ void flip(bool negative) {
    const uint32_t mask = negative ? (sizeof(T) == 2 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) / 2; ++i) {
      w[i].x ^= mask;
      w[i].y ^= mask;
      w[i].z ^= mask;
      w[i].w ^= mask;
    }
  }
  __device__ __forceinline__ void values(float (&v)[8]) const {
    if constexpr (sizeof(T) == 2) {
      const uint32_t x[4] = {w[0].x, w[0].y, w[0].z, w[0].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 f = pair_floats(x[i], T());
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
      }
    } else {
      Vec8<T>::load(reinterpret_cast<const T*>(w), v);
    }
  }
};

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
      if (mode == 2 && d < half) cs[j].y = -cs[j].y;
    }
  }
  // from a token's entries in shared memory, `stride` float4 between those of a place: neighbours', or halves'
  template <bool kNeighbours>
  __device__ __forceinline__ void take(const float4* token, int stride) {
    const int place = (kNeighbours || d0 < half ? d0 : d0 - half) / 8;
#pragma unroll
    for (int q = 0; q < (kNeighbours ? 2 : 4); ++q) {
      const float4 e = token[q * stride + place];
      cs[2 * q] = make_float2(e.x, e.y);
      cs[2 * q + 1] = make_float2(e.z, e.w);
    }
  }
  // the first `turned` values (those behind stay: a product with 0 would be NaN where one of them is infinite)
  __device__ __forceinline__ void neighbours(float (&v)[8], int turned = 8) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (2 * j >= turned) break;
      const float a = v[2 * j], b = v[2 * j + 1];
      v[2 * j] = turned_value(a, cs[j].x, b, -cs[j].y);
      v[2 * j + 1] = turned_value(b, cs[j].x, a, cs[j].y);
    }
  }
  // (the first half's partners count negatively: their signs are turned, two at a time where they have 16 bits)
  template <typename T>
  __device__ __forceinline__ void halves(const T* x, float (&v)[8]) const {
    Raw8<T> other;
    other.load(x + (d0 < half ? d0 + half : d0 - half));
    other.flip(d0 < half);
    float o[8];
    other.values(o);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = turned_value(v[j], cs[j].x, o[j], cs[j].y);
  }
  // v: the values at d0 of the head `x`
  template <typename T>
  __device__ __forceinline__ void apply(const T* x, float (&v)[8]) const {
    if (mode == 1) halves(x, v);
    else if (mode == 3) neighbours(v, rotary - d0);
    else if (mode == 2) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int d = d0 + j;
        const float o = d < rotary ? static_cast<float>(x[d < half ? d + half : d - half]) : 0.f;
        v[j] = turned_value(v[j], cs[j].x, o, cs[j].y);
      }
    }
  }
};

__device__ __forceinline__ float power_of_two(int e) { return __uint_as_float(static_cast<uint32_t>(e + 127) << 23); }

// The exponent of the smallest power of two that holds `top` in 448 times
__device__ __forceinline__ int scale_exponent(float top) {
  const uint32_t bits = __float_as_uint(top);
  const int e = static_cast<int>(bits >> 23) - 126 - ((bits & 0x7fffffu) <= 0x600000u ? 9 : 8);   // 448 = 0.875 * 2^9
  return e < kLeast ? kLeast : e;
}

constexpr float kFinite = 3.402823466e38f;

// finite: all of them are (else what is not is NaN: saturation would make a number of an infinity)
__device__ __forceinline__ uint2 to_codes(const float (&v)[8], float factor, bool finite) {
  float x[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = v[j] * factor;
  if (!finite) {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (!(fabsf(v[j]) <= kFinite)) x[j] = __uint_as_float(0x7fffffffu);
  }
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t low = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h], x[4 * h + 1]), __NV_SATFINITE, __NV_E4M3);
    const uint32_t high = __nv_cvt_float2_to_fp8x2(make_float2(x[4 * h + 2], x[4 * h + 3]), __NV_SATFINITE, __NV_E4M3);
    w[h] = low | (high << 16);
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

// The largest of all threads' (one barrier: `tops` is read until the next but one call, of the same)
__device__ __forceinline__ float block_top(float top, float* tops) {
  top = warp_max(top);
  if ((threadIdx.x & 31) == 0) tops[threadIdx.x >> 5] = top;
  __syncthreads();
  top = tops[0];
  const int warps = blockDim.x / 32;
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w)
    if (w < warps) top = fmaxf(top, tops[w]);
  return top;
}

// A page of one side, some of its heads, and the rows of it that a thread has
template <typename T>
struct PagePart {
  const PagedAppend& a;
  int h0, h1;
  int64_t first;                 // the page's first position
  int held, last;                // its older tokens, and where the new ones end
  int places, rows, row, d0;
  bool mine, real;               // whether the thread has rows, and values in them
  const T* x;                    // its first new row of head h0
  int64_t head_stride, step;     // ... to the next head, and to its next row
  uint8_t* codes;                // head h0's
  float* scales;
  bool turned, shared;
  int units, parts;              // float4 of a token's rotation, and of a place
};

// How a page's values are taken: row by row as they come (0), or all rows of all threads new ones: as they are (1), turned
// as halves (2) or as neighbours (3), whole vectors.
template <typename T, int kRows, int kForm>
__device__ __forceinline__ void append_heads(const PagePart<T>& p, Turn8 turn, const float4* s_rot, float (*s_top)[kThreads / 32]) {
  const PagedCache& c = p.a.cache;
  const T* x = p.x;
  uint8_t* to = p.codes + (p.held + p.row) * c.pitch;
  const int64_t head_bytes = static_cast<int64_t>(c.page) * c.pitch;
  auto new_row = [&](int i) { return kForm > 0 || p.held + p.row + i * p.rows < p.last; };
  Raw8<T> next[kRows];
  auto fetch = [&] {
#pragma unroll
    for (int i = 0; i < kRows; ++i) next[i].load(x + i * p.step);
  };
  if constexpr (kForm > 0) fetch();
  for (int h = p.h0; h < p.h1; ++h) {
    const float old = kForm == 0 && p.held > 0 ? p.scales[h] : 0.f;
    float v[kRows][8];
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < kRows; ++i) {
      if constexpr (kForm == 0) {
#pragma unroll
        for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        if (!p.real || !new_row(i)) continue;
        next[i].load(x + i * p.step);
      }
      next[i].values(v[i]);
      if constexpr (kForm >= 2) {
        if (turn.mode != 0) {
          if constexpr (kRows > 1) turn.take<kForm == 3>(s_rot + (p.row + i * p.rows) * p.units, p.units / p.parts);
          else if (h == p.h0) turn.read(p.a.rot, p.first + p.row);
          if constexpr (kForm == 2) turn.halves(x + i * p.step - p.d0, v[i]);
          else turn.neighbours(v[i]);
        }
      } else if (kForm == 0 && p.turned) {
        const int slot = p.held + p.row + i * p.rows;
        if (p.first + slot < p.a.rot_rows) {
          if (p.shared && turn.mode == 3) turn.take<true>(s_rot + (slot - p.held) * p.units, p.units / p.parts);
          else if (p.shared && turn.mode == 1) turn.take<false>(s_rot + (slot - p.held) * p.units, p.units / p.parts);
          else if (kRows > 1 || h == p.h0) turn.read(p.a.rot, p.first + slot);
          turn.apply(x + i * p.step - p.d0, v[i]);
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[i][j]));
    }
    x += p.head_stride;
    if (kForm > 0 && h + 1 < p.h1) fetch();        // under the barrier
    top = block_top(top, s_top[h & 1]);        // (every thread has read the old scale)
    const bool finite = top <= kFinite;
    if (!finite) {                             // the largest of those that are
      top = 0.f;
#pragma unroll
      for (int i = 0; i < kRows; ++i)
#pragma unroll
        for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(v[i][j]) <= kFinite ? fabsf(v[i][j]) : 0.f);
      __syncthreads();
      top = block_top(top, s_top[h & 1]);
    }
    const int e = scale_exponent(top);
    const float need = power_of_two(e), scale = kForm > 0 ? need : fmaxf(old, need);
    const float factor = kForm > 0 || scale == need ? power_of_two(-e) : 1.f / scale;
    if (threadIdx.x == 0) p.scales[h] = scale;
#pragma unroll
    for (int i = 0; i < kRows; ++i)
      if (kForm > 0 || (p.mine && new_row(i)))
        *reinterpret_cast<uint2*>(to + i * p.rows * c.pitch) = to_codes(v[i], factor, finite);
    if (kForm == 0 && p.held > 0 && scale != old && p.mine) {
      const float ratio = old * factor;
      for (int slot = p.row; slot < p.held; slot += p.rows) {
        uint2* at = reinterpret_cast<uint2*>(to + (slot - p.held - p.row) * c.pitch);
        float w[8];
        from_codes(*at, w);
        *at = to_codes(w, ratio, true);
      }
    }
    to += head_bytes;
  }
}

// Some heads of a side of a page.  More than one row to a thread: the rotation's rows of the page's tokens go
// through shared memory, in the order in which lanes read them (16 bytes of each of the places of a token side by side).
template <typename T, int kRows>
__device__ __forceinline__ void append_page(const PagedAppend& a, int tile, int per_cta, int rows) {
  const PagedCache& c = a.cache;
  extern __shared__ __align__(16) float4 s_rot[];
  __shared__ float s_top[2][kThreads / 32];
  const int side = tile & 1, groups = (c.heads + per_cta - 1) / per_cta, spans = (c.n + c.page - 2) / c.page + 1;
  int rest = tile >> 1, at = rest / groups;
  const int h0 = (rest - at * groups) * per_cta;
  rest = at;
  at = rest / spans;
  const int b = at, span = rest - at * spans;
  int64_t start;
  int count;
  new_tokens(c, b, start, count);
  const int64_t from = start > 0 ? start : 0, end = start + count;      // positions that are written (of 32 bits, but for start)
  const int64_t number = static_cast<int>(from) / c.page + static_cast<int64_t>(span);
  if (from >= end || number * c.page >= end || number >= c.table_pages) return;
  const int64_t id = c.table[static_cast<int64_t>(b) * c.table_pages + number];
  if (id < 0 || id >= c.n_pages) return;
  const int64_t first = number * c.page;
  const int held = static_cast<int>(from > first ? from - first : 0), last = static_cast<int>(end - first < c.page ? end - first : c.page);
  const int places = c.pitch / 8, place = threadIdx.x % places, row = threadIdx.x / places, d0 = place * 8;
  const int64_t* stride = side ? a.v_stride : a.k_stride;
  const bool turned = side == 0 && a.rot != nullptr;
  const int half = a.rotary / 2, units = half / 2, parts = a.interleaved ? 2 : 4;
  const bool whole_places = half % (2 * parts) == 0 && (reinterpret_cast<uintptr_t>(a.rot) & 15) == 0;      // rows as float4
  const PagePart<T> p{a, h0, min(c.heads, h0 + per_cta), first, held, last, places, rows, row, d0, row < rows, row < rows && d0 < c.dim,
                      static_cast<const T*>(side ? a.v : a.k) + b * stride[0] + (first + held + row - start) * stride[1] +
                          h0 * stride[2] + d0,
                      stride[2], rows * stride[1],
                      c.pages + ((id * 2 + side) * c.heads + h0) * static_cast<int64_t>(c.page) * c.pitch + d0,
                      c.scales + (id * 2 + side) * c.heads, turned, kRows > 1 && turned && whole_places, units, parts};
  if (p.shared) {
    const int u = threadIdx.x % units, t0 = threadIdx.x / units, tokens = blockDim.x / units;      // (at most 32 units)
    const int to = (u % parts) * (units / parts) + u / parts;
    const float4* from_row = reinterpret_cast<const float4*>(a.rot) + (first + held) * units + u;
    if (t0 < tokens) {
#pragma unroll 4
      for (int t = t0; t < last - held; t += tokens)
        s_rot[t * units + to] = first + held + t < a.rot_rows ? from_row[t * units] : make_float4(0.f, 0.f, 0.f, 0.f);
    }
    __syncthreads();
  }
  const Turn8 turn(d0, turned ? a.rotary : 0, a.interleaved);
  if (held == 0 && last == kRows * rows && places * rows == static_cast<int>(blockDim.x) && c.pitch == c.dim &&
      (!turned || (whole_places && first + last <= a.rot_rows))) {
    if (!turned) append_heads<T, kRows, 1>(p, turn, s_rot, s_top);
    else if (a.interleaved) append_heads<T, kRows, 3>(p, turn, s_rot, s_top);
    else append_heads<T, kRows, 2>(p, turn, s_rot, s_top);
    return;
  }
  append_heads<T, kRows, 0>(p, turn, s_rot, s_top);
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
  const int places = c.dim / 8, rows = blockDim.x / places;
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

// (CTAs of an SM, 8 x 1024 tokens of 16 heads of 128, us: 16-bit pages of 64 and 128 37 and 56 with two and one, 34 and 42 with three and
// two, for some spilling; fp32 44 with two, 53 with three.)
template <typename T, int kRows> constexpr int kCtas = (kRows <= 2 ? 3 : kRows <= 4 ? 2 : 1) + (sizeof(T) == 2 ? 1 : 0);

template <typename T, int kRows>
__global__ void __launch_bounds__(kThreads, kCtas<T, kRows>) paged_append_kernel(const PagedAppend a, int64_t tiles, int per_cta, int rows) {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");        // (the queries' kernel waits for nothing of this one)
  if (blockIdx.x < tiles) append_page<T, kRows>(a, static_cast<int>(blockIdx.x), per_cta, rows);
  else append_query<T>(a, blockIdx.x - tiles);
}

template <typename T, int kRows>
int launch_rows(const PagedAppend& a, int64_t tiles, int per_cta, int rows, unsigned grid, cudaStream_t stream) {
  auto kernel = paged_append_kernel<T, kRows>;
  int bytes = 0;
  if (kRows > 1 && a.rot != nullptr) {
    bytes = (a.cache.n < a.cache.page ? a.cache.n : a.cache.page) * a.rotary * 4;
    if (bytes > 47 * 1024) {             // (48 KB without it, the static part's bytes among them)
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
  const int threads = (rows * (a.cache.pitch / 8) + 31) / 32 * 32;
  kernel<<<grid, threads, bytes, stream>>>(a, tiles, per_cta, rows);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

template <typename T>
int launch(const PagedAppend& a_in, cudaStream_t stream) {
  PagedAppend a = a_in;
  const PagedCache& c = a.cache;
  const int64_t spans = (c.n + c.page - 2) / c.page + 1, pages = c.B * spans * 2;
  // Many tokens: their queries by the rotation's own kernel, which has more bytes on their way, beside this one's last CTAs.
  // (Few: one launch.)
  RotaryCall r{};
  const bool apart = a.q != nullptr && static_cast<int64_t>(c.B) * c.n >= 4 * sm_count();
  if (apart) {
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
    r.table_rows = a.rot != nullptr ? a.rot_rows : INT64_MAX;
    r.at.lengths = c.lengths;
    r.at.counts = c.counts;
    r.B = c.B;
    r.S = c.n;
    r.D = c.dim;
    r.rotary = a.rotary;
    r.interleaved = a.interleaved;
    r.dtype = a.dtype;
    r.beside = true;
    a.q = nullptr;
  }
  // as many heads to a CTA as leave each SM some CTAs: they share the rotation's rows.  (8 x 2048 tokens of 16 heads of 128 and four
  // ragged prompts of up to 1001 tokens of 32 heads of 80, us: up to four heads 55 and 29.5, eight 56 and 36, two 64 and 28.)
  int per_cta = 4;
  while (per_cta > 1 && pages * ((c.heads + per_cta - 1) / per_cta) < 6 * sm_count()) per_cta /= 2;
  const int64_t tiles = pages * ((c.heads + per_cta - 1) / per_cta);
  const int64_t ctas = tiles + (a.q != nullptr ? static_cast<int64_t>(c.B) * c.n : 0);
  if (ctas > 0x7fffffff) return 5;
  if (ctas == 0) {
    r.beside = false;
    return apart ? launch_rotary(r, stream) : 0;
  }
  const unsigned grid = static_cast<unsigned>(ctas);
  // as many rows of threads as there are new tokens in a page, in powers of two, or a share of that: up to kThreads, no fewer
  // than half of that where there are tokens enough or the queries' CTAs are in the launch
  const int places = c.pitch / 8;
  int rows = 1, per = 1;
  while (rows < c.n && rows < c.page) rows *= 2;
  while (rows * places > kThreads) {
    rows /= 2;
    per *= 2;
  }
  while (per == 1 && rows < c.page && rows * 2 * places <= kThreads / 2) rows *= 2;
  int rc = 6;
  if (per == 1) rc = launch_rows<T, 1>(a, tiles, per_cta, rows, grid, stream);
  else if (per == 2) rc = launch_rows<T, 2>(a, tiles, per_cta, rows, grid, stream);
  else if (per == 4) rc = launch_rows<T, 4>(a, tiles, per_cta, rows, grid, stream);
  else if (per == 8) rc = launch_rows<T, 8>(a, tiles, per_cta, rows, grid, stream);
  return rc == 0 && apart ? launch_rotary(r, stream) : rc;
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
