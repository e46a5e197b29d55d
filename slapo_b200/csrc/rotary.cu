// Rotation of queries and keys by their positions, and its gradient.
//
// A pair (a, b) of a head at position p becomes (a c - b s, b c + a s) with c and s from a table's row p; the gradient is
// the transposed rotation (s negated), which needs nothing but the positions.  Pairs are the halves of the rotated part
// of a head or neighbours; what lies behind it is copied.  Products and sums in fp32, one rounding.
//
// Bound by HBM: each value is read once and written once.  A CTA takes some tokens one after the other with all their heads: a
// thread has one place in the heads - 16 bytes, or for halves the two places of 16 bytes that belong together - and three
// heads on their way, so that the table's entries are read once per token and thread.  q, k (and v of a packed
// projection, copied) are parts of one launch.  Heads whose pairs do not fill 16 bytes go value by value.
// 4 x 2048 packed tokens of 16 heads of 128, bf16: 37 us a direction (5.4 TB/s of 201 MB); 12001 tokens of 32 and 4 heads of 80 with 40
// rotated as neighbours, fp16: 31, as halves (20 values: value by value) 97.
#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

// V values as they are in memory: 16 bytes, or a single one
template <typename T, int V>
struct Values {
  uint4 w;
  __device__ __forceinline__ void load(const T* p) { w = __ldcs(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = w; }
  __device__ __forceinline__ uint32_t& word(int i) { return i == 0 ? w.x : i == 1 ? w.y : i == 2 ? w.z : w.w; }
  // two values one after the other
  __device__ __forceinline__ float2 get2(int i) {
    if constexpr (sizeof(T) == 2) return pair_floats(word(i), T());
    else return make_float2(__uint_as_float(word(2 * i)), __uint_as_float(word(2 * i + 1)));
  }
  __device__ __forceinline__ void set2(int i, float a, float b) {
    if constexpr (sizeof(T) == 2) {
      word(i) = pair_word(a, b, T());
    } else {
      word(2 * i) = __float_as_uint(a);
      word(2 * i + 1) = __float_as_uint(b);
    }
  }
};
template <typename T>
struct Values<T, 1> {
  T v;
  __device__ __forceinline__ void load(const T* p) { v = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = v; }
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
    if constexpr (V > 1) {
#pragma unroll
      for (int j = 0; j < kCs; j += 2) {
        const float4 two = *reinterpret_cast<const float4*>(row + j);
        cs[j] = make_float2(two.x, two.y * sign);
        cs[j + 1] = make_float2(two.z, two.w * sign);
      }
    } else {
      cs[0] = make_float2(row[0].x, row[0].y * sign);
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
    if constexpr (V == 1) {
      const float a = static_cast<float>(m.v), b = static_cast<float>(n.v);
      m.v = static_cast<T>(turned_value(a, cs[0].x, b, -cs[0].y));
      n.v = static_cast<T>(turned_value(b, cs[0].x, a, cs[0].y));
    } else if constexpr (kNeighbours) {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 a = m.get2(j);
        m.set2(j, turned_value(a.x, cs[j].x, a.y, -cs[j].y), turned_value(a.y, cs[j].x, a.x, cs[j].y));
      }
    } else {
#pragma unroll
      for (int j = 0; j < V / 2; ++j) {
        const float2 a = m.get2(j), b = n.get2(j), c = cs[2 * j], d = cs[2 * j + 1];
        m.set2(j, turned_value(a.x, c.x, b.x, -c.y), turned_value(a.y, d.x, b.y, -d.y));
        n.set2(j, turned_value(b.x, c.x, a.x, c.y), turned_value(b.y, d.x, a.y, d.y));
      }
    }
  }
};

// Rows of heads that a thread has on their way at a time.  (4 x 2048 packed tokens of 16 heads of 128, and 8 x 2048 of 16 and 2
// heads, us: three rows and up to 128 registers 37.0 and 32.8, two and 64 38.7 and 35.4, three and 80 40.9 and 38.6, four and
// 128 36.9 and 36.8.)
constexpr int kRowsAhead = 3;

// A CTA has `tokens` tokens one after the other, all heads of each: what an address takes is computed once for all of them.
// (Addresses by token and head, 64 bits wide, were half of the instructions: 4 x 2048 tokens of 48 heads of 128 49 us.)
template <typename T, int V, bool kPairs>
__global__ void __launch_bounds__(256, 2) rotary_kernel(const RotaryCall c, int rows, int tokens) {
  using Place = RotaryPlace<T, V, kPairs>;
  Place place(threadIdx.x, c.rotary);
  const int64_t s0 = static_cast<int64_t>(blockIdx.x) * tokens;
  const int n = static_cast<int>(c.S - s0 < tokens ? c.S - s0 : tokens);
  for (int64_t b = blockIdx.y; b < c.B; b += gridDim.y) {
    int64_t start = c.at.start, count = c.S;       // positions that follow one another, of the first `count` tokens
    if (c.at.lengths != nullptr) {
      if (c.at.counts != nullptr) count = min(max(static_cast<int64_t>(c.at.counts[b]), int64_t{0}), c.S);
      start = c.at.lengths[b] - count;
    }
    for (int row0 = threadIdx.y; row0 < rows; row0 += kRowsAhead * blockDim.y) {
      const T* x[kRowsAhead];
      T* y[kRowsAhead];
      int x_step[kRowsAhead], y_step[kRowsAhead];        // (of more than one token: see launch)
      bool turn[kRowsAhead], mine[kRowsAhead];
#pragma unroll
      for (int u = 0; u < kRowsAhead; ++u) {
        int h = row0 + u * blockDim.y;
        mine[u] = h < rows;
        // the parts' heads are rows one after the other
        int p = 0;
        while (mine[u] && h >= c.part[p].heads) h -= c.part[p++].heads;
        const RotaryPart& part = c.part[p];
        turn[u] = part.turn;
        x[u] = static_cast<const T*>(part.x) + b * part.x_stride[0] + s0 * part.x_stride[1] + h * part.x_stride[2];
        y[u] = static_cast<T*>(part.y) + b * part.y_stride[0] + s0 * part.y_stride[1] + h * part.y_stride[2];
        x_step[u] = static_cast<int>(part.x_stride[1]);
        y_step[u] = static_cast<int>(part.y_stride[1]);
      }
      for (int t = 0; t < n; ++t) {
        int64_t pos = s0 + t < count ? start + s0 + t : -1;
        if (c.at.ids != nullptr) {
          const int64_t at = b * c.at.batch_stride + (s0 + t) * c.at.token_stride;
          pos = c.at.ids64 ? static_cast<const int64_t*>(c.at.ids)[at] : static_cast<const int32_t*>(c.at.ids)[at];
        }
        const bool known = pos >= 0 && pos < c.table_rows;
        Values<T, V> m[kRowsAhead], n[kRowsAhead];
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u)
          if (mine[u] && (known || !turn[u])) place.load(x[u], m[u], n[u]);
        if (known) place.read(c.table, pos, c.rotary, c.transposed ? -1.f : 1.f);
#pragma unroll
        for (int u = 0; u < kRowsAhead; ++u) {
          if (mine[u]) {
            if (turn[u]) {
              if (known) place.turn(m[u], n[u]);
              else m[u] = n[u] = Values<T, V>{};        // (a position outside of the table)
            }
            place.store(y[u], m[u], n[u]);
          }
          x[u] += x_step[u];
          y[u] += y_step[u];
        }
      }
    }
  }
  if (c.beside) asm volatile("griddepcontrol.wait;" ::: "memory");        // (what comes after has to find both done)
}

bool vectors(const RotaryCall& c, int v, int bytes) {
  if (c.D % v != 0 || c.rotary % (c.interleaved ? v : 2 * v) != 0 || (reinterpret_cast<uintptr_t>(c.table) & 15) != 0) return false;
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
  // as many rows to a thread as it has on their way at a time, in as few rounds as 256 threads take
  const int most = 256 / places, each = heads < kRowsAhead ? heads : kRowsAhead, rounds = (heads + most * each - 1) / (most * each);
  const int rows = (heads + each * rounds - 1) / (each * rounds);
  // some tokens to a CTA where that leaves each SM CTAs enough
  int tokens = 8;
  for (int p = 0; p < c.parts; ++p)
    for (const int64_t step : {c.part[p].x_stride[1], c.part[p].y_stride[1]})
      if (step > 0x7fffffff || step < -0x7fffffff) tokens = 1;
  while (tokens > 1 && c.B * ((c.S + tokens - 1) / tokens) < 12 * sm_count()) tokens /= 2;
  const int64_t stretches = (c.S + tokens - 1) / tokens;
  if (stretches > 0x7fffffff) return 5;
  const dim3 block(places, rows), grid(static_cast<unsigned>(stretches), static_cast<unsigned>(c.B < 65535 ? c.B : 65535));
  count_launch();
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = block;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = c.beside ? 1 : 0;
  const cudaError_t done =
      wide && c.interleaved ? cudaLaunchKernelEx(&config, rotary_kernel<T, V, true>, c, heads, tokens)
      : wide                ? cudaLaunchKernelEx(&config, rotary_kernel<T, V, false>, c, heads, tokens)
      : c.interleaved       ? cudaLaunchKernelEx(&config, rotary_kernel<T, 1, true>, c, heads, tokens)
                            : cudaLaunchKernelEx(&config, rotary_kernel<T, 1, false>, c, heads, tokens);
  return done == cudaSuccess ? 0 : 4;
}

}  // namespace

int launch_rotary(const RotaryCall& c, cudaStream_t stream) {
  if (c.B == 0 || c.S == 0) return 0;
  if (c.D < 1 || c.D > 256 || c.rotary < 0 || c.rotary % 2 != 0 || c.rotary > c.D) return 1;
  switch (c.dtype) {
    case 0: return launch<__nv_bfloat16>(c, stream);
    case 1: return launch<__half>(c, stream);
    case 2: return launch<float>(c, stream);
    default: return 3;
  }
}

}  // namespace slapo
