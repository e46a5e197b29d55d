// Rotation of queries and keys by their positions, and its gradient.
//
// A pair (a, b) of a head at position p becomes (a c - b s, b c + a s) with c and s from a table's row p; the gradient is
// the transposed rotation (s negated), which needs nothing but the positions.  Pairs are the halves of the rotated part
// of a head or neighbours; what lies behind it is copied.  Products and sums in fp32, one rounding.
//
// Bound by HBM: each value is read once and written once.  A CTA takes a token with all its heads: a thread has one
// place in the heads - 16 bytes, or for halves the two places of 16 bytes that belong together - and goes over the heads,
// so that the table's entries are read once per token and thread.  q, k (and v of a packed projection, copied) are
// parts of one launch.
#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

template <typename T, int V>
struct Values {
  float v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      v[0] = static_cast<float>(*p);
    } else {
      const uint4 raw = *reinterpret_cast<const uint4*>(p);
      const T* x = reinterpret_cast<const T*>(&raw);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = static_cast<float>(x[i]);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) {
      *p = static_cast<T>(v[0]);
    } else {
      uint4 raw;
      T* x = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (int i = 0; i < V; ++i) x[i] = static_cast<T>(v[i]);
      *reinterpret_cast<uint4*>(p) = raw;
    }
  }
};

// One place of a head for a thread: V values (16 bytes, or single ones) that are turned with V others, or copied.  Places
// that are turned come first.
template <typename T, int V, bool kPairs>
struct RotaryPlace {
  static constexpr bool kNeighbours = kPairs && V > 1;       // both of a pair in one vector
  static constexpr int kCs = kNeighbours ? V / 2 : V;
  bool copy;
  int first, second;          // where the values lie in a head (second: not with kNeighbours)
  int entry;                  // ... and their cosines and sines in a row of the table
  float2 cs[kCs];

  static __host__ __device__ __forceinline__ int turned(int rotary) {
    return kNeighbours ? rotary / V : rotary / 2 / V;
  }
  static __host__ __device__ __forceinline__ int places(int dim, int rotary) {
    return turned(rotary) + (dim - rotary) / V;
  }
  __device__ __forceinline__ RotaryPlace(int i, int rotary) {
    const int t = turned(rotary);
    copy = i >= t;
    first = copy ? rotary + (i - t) * V : (kPairs && !kNeighbours ? 2 * i : i * V);
    second = kPairs ? first + 1 : first + rotary / 2;
    entry = i * kCs;
  }
  // the table's row of a position that is in it
  __device__ __forceinline__ void read(const float* table, int64_t pos, int rotary, float sign) {
    if (copy) return;
    const float2* row = reinterpret_cast<const float2*>(table) + pos * (rotary / 2) + entry;
#pragma unroll
    for (int j = 0; j < kCs; ++j) {
      cs[j] = row[j];
      cs[j].y *= sign;
    }
  }
  // x to y, as it is
  __device__ __forceinline__ void move(const T* x, T* y) const {
    Values<T, V> m;
    m.load(x + first);
    m.store(y + first);
    if constexpr (!kNeighbours) {
      if (!copy) {
        m.load(x + second);
        m.store(y + second);
      }
    }
  }
  __device__ __forceinline__ void clear(T* y) const {
    Values<T, V> m{};
    m.store(y + first);
    if constexpr (!kNeighbours) {
      if (!copy) m.store(y + second);
    }
  }
  __device__ __forceinline__ void turn(const T* x, T* y) const {
    Values<T, V> m, n;
    m.load(x + first);
    if (copy) {
      m.store(y + first);
      return;
    }
    if constexpr (kNeighbours) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        n.v[2 * j] = turned_value(m.v[2 * j], cs[j].x, m.v[2 * j + 1], -cs[j].y);
        n.v[2 * j + 1] = turned_value(m.v[2 * j + 1], cs[j].x, m.v[2 * j], cs[j].y);
      }
      n.store(y + first);
    } else {
      n.load(x + second);
      Values<T, V> a, o;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        a.v[j] = turned_value(m.v[j], cs[j].x, n.v[j], -cs[j].y);
        o.v[j] = turned_value(n.v[j], cs[j].x, m.v[j], cs[j].y);
      }
      a.store(y + first);
      o.store(y + second);
    }
  }
};

template <typename T, int V, bool kPairs>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryCall c) {
  RotaryPlace<T, V, kPairs> place(threadIdx.x, c.rotary);
  for (int64_t token = blockIdx.x; token < c.B * c.S; token += gridDim.x) {
    const int64_t b = token / c.S, s = token - b * c.S;
    int64_t pos = c.at.start + s;
    if (c.at.ids != nullptr) {
      const int64_t at = b * c.at.batch_stride + s * c.at.token_stride;
      pos = c.at.ids64 ? static_cast<const int64_t*>(c.at.ids)[at] : static_cast<const int32_t*>(c.at.ids)[at];
    }
    const bool known = pos >= 0 && pos < c.table_rows;
    if (known) place.read(c.table, pos, c.rotary, c.transposed ? -1.f : 1.f);
#pragma unroll
    for (int p = 0; p < 3; ++p) {
      if (p >= c.parts) break;
      const RotaryPart& part = c.part[p];
      const T* x = static_cast<const T*>(part.x) + b * part.x_stride[0] + s * part.x_stride[1];
      T* y = static_cast<T*>(part.y) + b * part.y_stride[0] + s * part.y_stride[1];
      for (int h = threadIdx.y; h < part.heads; h += blockDim.y) {
        const T* xh = x + h * part.x_stride[2];
        T* yh = y + h * part.y_stride[2];
        if (!part.turn) place.move(xh, yh);
        else if (known) place.turn(xh, yh);
        else place.clear(yh);        // (a position outside of the table)
      }
    }
  }
}

bool vectors(const RotaryCall& c, int v, int bytes) {
  if (c.D % v != 0 || c.rotary % (c.interleaved ? v : 2 * v) != 0) return false;
  for (int p = 0; p < c.parts; ++p) {
    const RotaryPart& part = c.part[p];
    if (((reinterpret_cast<uintptr_t>(part.x) | reinterpret_cast<uintptr_t>(part.y)) & 15) != 0) return false;
    for (int d = 0; d < 3; ++d)
      if (part.x_stride[d] * bytes % 16 != 0 || part.y_stride[d] * bytes % 16 != 0) return false;
  }
  return true;
}

template <typename T>
int launch(const RotaryCall& c, cudaStream_t stream) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = vectors(c, V, sizeof(T));
  const int places = wide ? (c.interleaved ? RotaryPlace<T, V, true>::places(c.D, c.rotary)
                                           : RotaryPlace<T, V, false>::places(c.D, c.rotary))
                          : RotaryPlace<T, 1, false>::places(c.D, c.rotary);
  int heads = 0;
  for (int p = 0; p < c.parts; ++p) heads = c.part[p].heads > heads ? c.part[p].heads : heads;
  if (places > 256) return 2;
  int rows = 256 / places;
  if (rows > heads) rows = heads;
  const int64_t tokens = c.B * c.S;
  const unsigned grid = static_cast<unsigned>(tokens < 0x7fffffff ? tokens : 0x7fffffff);
  const dim3 block(places, rows);
  count_launch();
  if (wide && c.interleaved) rotary_kernel<T, V, true><<<grid, block, 0, stream>>>(c);
  else if (wide) rotary_kernel<T, V, false><<<grid, block, 0, stream>>>(c);
  else if (c.interleaved) rotary_kernel<T, 1, true><<<grid, block, 0, stream>>>(c);
  else rotary_kernel<T, 1, false><<<grid, block, 0, stream>>>(c);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace

int launch_rotary(const RotaryCall& c, cudaStream_t stream) {
  if (c.B == 0 || c.S == 0) return 0;
  if (c.D < 1 || c.D > 256 || c.rotary < 2 || c.rotary % 2 != 0 || c.rotary > c.D) return 1;
  switch (c.dtype) {
    case 0: return launch<__nv_bfloat16>(c, stream);
    case 1: return launch<__half>(c, stream);
    case 2: return launch<float>(c, stream);
    default: return 3;
  }
}

}  // namespace slapo
