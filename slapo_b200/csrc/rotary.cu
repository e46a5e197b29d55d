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

// V values as they are in memory: 16 bytes, or a single one
template <typename T, int V>
struct __align__(V == 1 ? sizeof(T) : 16) Values {
  T v[V];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      v[0] = *p;
    } else {
      *reinterpret_cast<uint4*>(v) = __ldcs(reinterpret_cast<const uint4*>(p));
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (V == 1) *p = v[0];
    else *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(v);
  }
  __device__ __forceinline__ float get(int i) const { return static_cast<float>(v[i]); }
  __device__ __forceinline__ void set(int i, float x) { v[i] = static_cast<T>(x); }
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
  __device__ __forceinline__ void load(const T* x, Values<T, V>& m, Values<T, V>& n) const {
    m.load(x + first);
    if constexpr (!kNeighbours) {
      if (!copy) n.load(x + second);
    }
  }
  __device__ __forceinline__ void store(T* y, const Values<T, V>& m, const Values<T, V>& n) const {
    m.store(y + first);
    if constexpr (!kNeighbours) {
      if (!copy) n.store(y + second);
    }
  }
  __device__ __forceinline__ void turn(Values<T, V>& m, Values<T, V>& n) const {
    if (copy) return;
#pragma unroll
    for (int j = 0; j < kCs; ++j) {
      float a[2];
      if constexpr (kNeighbours) { a[0] = m.get(2 * j); a[1] = m.get(2 * j + 1); }
      else { a[0] = m.get(j); a[1] = n.get(j); }
      const float x = turned_value(a[0], cs[j].x, a[1], -cs[j].y), y = turned_value(a[1], cs[j].x, a[0], cs[j].y);
      if constexpr (kNeighbours) { m.set(2 * j, x); m.set(2 * j + 1, y); }
      else { m.set(j, x); n.set(j, y); }
    }
  }
};

// Rows of heads that a thread has on their way at a time
constexpr int kRowsAhead = 3;

template <typename T, int V, bool kPairs>
__global__ void __launch_bounds__(256) rotary_kernel(const RotaryCall c, int rows) {
  using Place = RotaryPlace<T, V, kPairs>;
  Place place(threadIdx.x, c.rotary);
  for (int64_t token = blockIdx.x; token < c.B * c.S; token += gridDim.x) {
    const int64_t b = token / c.S, s = token - b * c.S;
    int64_t pos = c.at.start + s;
    if (c.at.ids != nullptr) {
      const int64_t at = b * c.at.batch_stride + s * c.at.token_stride;
      pos = c.at.ids64 ? static_cast<const int64_t*>(c.at.ids)[at] : static_cast<const int32_t*>(c.at.ids)[at];
    } else if (c.at.lengths != nullptr) {
      const int64_t count = c.at.counts != nullptr ? min(max(static_cast<int64_t>(c.at.counts[b]), int64_t{0}), c.S) : c.S;
      pos = s < count ? c.at.lengths[b] - count + s : -1;
    }
    const bool known = pos >= 0 && pos < c.table_rows;
    for (int row0 = threadIdx.y; row0 < rows; row0 += kRowsAhead * blockDim.y) {
      Values<T, V> m[kRowsAhead], n[kRowsAhead];
      T* y[kRowsAhead];
      bool turn[kRowsAhead];
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        int h = row0 + u * blockDim.y;
        y[u] = nullptr;
        if (h >= rows) continue;
        // the parts' heads are rows one after the other
        int p = 0;
        while (h >= c.part[p].heads) h -= c.part[p++].heads;
        const RotaryPart& part = c.part[p];
        turn[u] = part.turn;
        y[u] = static_cast<T*>(part.y) + b * part.y_stride[0] + s * part.y_stride[1] + h * part.y_stride[2];
        if (part.turn && !known) continue;
        place.load(static_cast<const T*>(part.x) + b * part.x_stride[0] + s * part.x_stride[1] + h * part.x_stride[2], m[u], n[u]);
      }
      if (known && row0 == threadIdx.y) place.read(c.table, pos, c.rotary, c.transposed ? -1.f : 1.f);
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        if (y[u] == nullptr) continue;
        if (turn[u]) {
          if (known) place.turn(m[u], n[u]);
          else m[u] = n[u] = Values<T, V>{};        // (a position outside of the table)
        }
        place.store(y[u], m[u], n[u]);
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
  for (int p = 0; p < c.parts; ++p) heads += c.part[p].heads;
  if (places > 256) return 2;
  if (heads == 0) return 0;
  // as few rounds over the heads as 256 threads take, with as few idle rows in the last one
  const int most = 256 / places, rounds = (heads + most - 1) / most;
  const int rows = (heads + rounds - 1) / rounds;
  const int64_t tokens = c.B * c.S;
  const unsigned grid = static_cast<unsigned>(tokens < 0x7fffffff ? tokens : 0x7fffffff);
  const dim3 block(places, rows);
  count_launch();
  if (wide && c.interleaved) rotary_kernel<T, V, true><<<grid, block, 0, stream>>>(c, heads);
  else if (wide) rotary_kernel<T, V, false><<<grid, block, 0, stream>>>(c, heads);
  else if (c.interleaved) rotary_kernel<T, 1, true><<<grid, block, 0, stream>>>(c, heads);
  else rotary_kernel<T, 1, false><<<grid, block, 0, stream>>>(c, heads);
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
