// Attention of a sequence's newest tokens over a paged cache in 8 bits.
//
// Row r of a cached head is query t = r / G of query head r % G of its G; it sees the keys up to its own position (and
// not before its window).  With codes k, v and a page's scales ks, vs: s = ks (q k) scale, o = sum p vs v / sum p.
//
// Bound by reading the cache.  A warp works alone, on units of 16 keys of one head: S^T = K Q^T by m16n8k16 (16 keys,
// 8 rows), O^T += V^T P^T (16 values of a head, 8 rows), codes converted to fp16 - exactly - on their way into the
// registers of the products.  The tensor core's order of the contraction is free as long as both operands share it, so
// that a lane's 16 bytes of a key are its operands of four products, and 16 bytes each of four values' rows, bytes
// interleaved, those of eight.  Lanes copy what they themselves read later, by cp.async, into a ring in shared memory: no
// barriers, and bytes enough on their way.  mma.sync and not tcgen05: a unit has one to eight rows of work, and the
// operands pass through registers, since they are converted.
//
// Keys are dealt out over all warps evenly, whatever the sequences' lengths, which are in device memory: each warp counts
// the units of all sequences and takes its share of their row, at least kLeastUnits; it writes an item (sequence, head,
// rows) that lies wholly in its share, and leaves its part of the first and the last else, which a second kernel adds up.
//
// Roundings: q to fp16 by a power of two per row (exact for bf16 values within 2^-28 of the row's largest, and for fp16's),
// probabilities to fp16 (2^-11), all else in fp32.
#include <cuda_fp8.h>

#include "flash_common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

constexpr int kWarps = 8;
constexpr int kUnit = 16;          // keys
constexpr int kLeastUnits = 4;     // of a warp's share

// What is known of the work before lengths are: the same in both kernels
struct Plan {
  PagedAttention a;
  int group, rows, tiles, tile_rows, warps, words;     // tiles of rows per head; words: of a row's part
  int page_units;                                      // log2 of a page's units
  float scale_log2;
};

__device__ __forceinline__ void keys_of(const PagedCache& c, int window, int b, int& first_unit, int& units, int& len,
                                        int& count) {
  count = c.counts != nullptr ? min(max(c.counts[b], 0), c.n) : c.n;
  const int64_t most = static_cast<int64_t>(c.table_pages) * c.page;
  len = c.lengths[b];
  const int seen = static_cast<int>(min(static_cast<int64_t>(max(len, 0)), most));
  const int64_t first = window > 0 ? static_cast<int64_t>(len) - count - window + 1 : 0;
  first_unit = first > 0 ? static_cast<int>(min(first, most)) / kUnit : 0;
  units = count > 0 ? max((seen + kUnit - 1) / kUnit - first_unit, 0) : 0;
}

// Sum of the units of all sequences' items, and (for one thread each of the warps) the sequence with the `at`-th one
struct Shares {
  int64_t total;       // units
  int64_t per;         // of a warp
  __device__ __forceinline__ int64_t begin(int warp) const { return min(warp * per, total); }
};
__device__ __forceinline__ Shares count_units(const Plan& p) {
  const PagedCache& c = p.a.cache;
  int64_t sum = 0;
  for (int b = threadIdx.x & 31; b < c.B; b += 32) {
    int first, units, len, count;
    keys_of(c, p.a.window, b, first, units, len, count);
    sum += units;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  Shares s;
  s.total = sum * c.heads * p.tiles;
  const int64_t even = (s.total + p.warps - 1) / p.warps;
  s.per = max(even, static_cast<int64_t>(kLeastUnits));
  return s;
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copy8(uint32_t to, const void* from, bool ok) {
  const int n = ok ? 8 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 8, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ uint4 read16(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ uint2 read8(uint32_t at) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float read4(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// four codes as two pairs in fp16
__device__ __forceinline__ uint2 halves(uint32_t w) {
  const __half2_raw lo = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w & 0xffffu), __NV_E4M3);
  const __half2_raw hi = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(w >> 16), __NV_E4M3);
  return make_uint2(*reinterpret_cast<const uint32_t*>(&lo), *reinterpret_cast<const uint32_t*>(&hi));
}
__device__ __forceinline__ uint32_t bytes(uint32_t a, uint32_t b, uint32_t selector) { return __byte_perm(a, b, selector); }
__device__ __forceinline__ void product(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// kWide: heads of 72 to 128, whose tokens are 80 to 128 bytes; else up to 64.  N: tiles of 8 rows.
template <bool kWide, int N, typename T>
struct Shape {
  static constexpr int kChunks = kWide ? 2 : 1;                   // of 64 values of a key
  static constexpr int kKey = kChunks * 2 * 16;                   // a lane's bytes of a unit
  static constexpr int kValue = 4 * (kWide ? 16 : 8);
  static constexpr int kStage = 32 * (kKey + kValue + 8);
  static constexpr int kStages = kWide ? 6 : 10;
  static constexpr int kSmem = kWarps * kStages * kStage;
  static constexpr int kTiles = kWide ? 8 : 4;                    // of 16 values of a head
  static constexpr int kValues = kWide ? 16 : 8;                  // consecutive ones that a lane has
};

// A place in the row of all units
struct Cursor {
  int b, item, unit, units, first_unit, len, count;
};
__device__ __forceinline__ void sequence(const Plan& p, Cursor& at) {
  while (at.b < p.a.cache.B) {
    keys_of(p.a.cache, p.a.window, at.b, at.first_unit, at.units, at.len, at.count);
    if (at.units > 0) return;
    ++at.b;
  }
}
// the `target`-th unit
__device__ __forceinline__ Cursor find(const Plan& p, int64_t target) {
  const PagedCache& c = p.a.cache;
  const int lane = threadIdx.x & 31;
  const int64_t items = static_cast<int64_t>(c.heads) * p.tiles;
  Cursor at{};
  int64_t before = 0;
  for (int b0 = 0; b0 < c.B; b0 += 32) {
    int first, units = 0, len, count;
    if (b0 + lane < c.B) keys_of(c, p.a.window, b0 + lane, first, units, len, count);
    int64_t sum = units * items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, sum, o);
      if (lane >= o) sum += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + sum > target);
    if (past != 0) {
      const int l = __ffs(past) - 1;
      at.b = b0 + l;
      const int64_t until = __shfl_sync(0xffffffffu, sum, l) + before;
      at.units = __shfl_sync(0xffffffffu, units, l);
      keys_of(c, p.a.window, at.b, at.first_unit, at.units, at.len, at.count);
      const int64_t in = target - (until - at.units * items);
      at.item = static_cast<int>(in / at.units);
      at.unit = static_cast<int>(in - static_cast<int64_t>(at.item) * at.units);
      return at;
    }
    before += __shfl_sync(0xffffffffu, sum, 31);
  }
  at.b = c.B;
  return at;
}

// what a warp leaves of the item that it begins with (0) or ends with (1): a row of `words` floats for each row of the tile
__device__ __forceinline__ float* part_of(const Plan& p, int warp, int which, int row) {
  return p.a.scratch + ((static_cast<int64_t>(warp) * 2 + which) * p.tile_rows + row) * p.words;
}

template <bool kWide, int N, typename T>
__global__ void __launch_bounds__(kWarps * 32, 1) paged_attention_kernel(const Plan p) {
  using S = Shape<kWide, N, T>;
  extern __shared__ __align__(128) uint8_t s_ring[];
  const PagedCache& c = p.a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int number = blockIdx.x * kWarps + warp;
  pdl_launch();
  const Shares shares = count_units(p);
  const int64_t begin = shares.begin(number), end = shares.begin(number + 1);
  if (begin >= end) return;
  int left = static_cast<int>(end - begin), to_issue = left;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(s_ring)) + warp * S::kStages * S::kStage;
  const int64_t head_bytes = static_cast<int64_t>(c.page) * c.pitch;

  Cursor in = find(p, begin), at = in;
  auto page_of = [&](const Cursor& x) {        // of the unit's keys; -1: none
    if (x.b >= c.B) return -1;
    const int id = c.table[static_cast<int64_t>(x.b) * c.table_pages + ((x.first_unit + x.unit) >> p.page_units)];
    return id >= 0 && id < c.n_pages ? id : -1;
  };
  auto step = [&](Cursor& x) {
    if (++x.unit < x.units) return;
    x.unit = 0;
    if (++x.item < c.heads * p.tiles) return;
    x.item = 0;
    ++x.b;
    sequence(p, x);
  };
  int page = page_of(in);
  unsigned missing = 0;        // the stages whose unit has no page
  // the unit's codes and scales on their way into a stage; the next unit's page is read ahead
  auto issue = [&](int stage) {
    if (to_issue > 0) {
      --to_issue;
      const int key0 = (in.first_unit + in.unit) * kUnit, h = in.item / p.tiles;
      const bool known = page >= 0;
      missing = (missing & ~(1u << stage)) | (known ? 0u : 1u << stage);
      const int64_t side = (static_cast<int64_t>(known ? page : 0) * 2) * c.heads + h;
      const uint8_t* k = c.pages + side * head_bytes + static_cast<int64_t>(key0 & (c.page - 1)) * c.pitch;
      const uint8_t* v = k + c.heads * head_bytes;
      const uint32_t to = ring + stage * S::kStage + lane * 16;
      // keys that no row sees are zeros: a hidden code may be a NaN
      const int until = in.len - key0;
      const int from = p.a.window > 0 ? in.len - in.count - p.a.window + 1 - key0 : 0;
#pragma unroll
      for (int j = 0; j < S::kChunks; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = g + 8 * r, d = 64 * j + 16 * t;
          const bool ok = known && key < until && key >= from && d < c.pitch;
          copy16(to + (j * 2 + r) * 512, ok ? k + key * c.pitch + d : c.pages, ok);
        }
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int key = 2 * t + (r & 1) + 8 * (r >> 1), d = S::kValues * g;
        const bool ok = known && key < until && key >= from && d < c.pitch;
        const uint8_t* src = ok ? v + key * c.pitch + d : c.pages;
        if constexpr (kWide) copy16(to + 32 * S::kKey + r * 512, src, ok);
        else copy8(ring + stage * S::kStage + 32 * S::kKey + r * 256 + lane * 8, src, ok);
      }
      const uint32_t scales = ring + stage * S::kStage + 32 * (S::kKey + S::kValue) + lane * 8;
      copy4(scales, c.scales + side, known);
      copy4(scales + 4, c.scales + side + c.heads, known);
      step(in);
      if (to_issue > 0) page = page_of(in);
    }
    commit_copies();
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);

  uint32_t q[N][S::kChunks][4][2];
  float factor[N][2], m[N][2], l[N][2], o[N][S::kTiles][4];
  int last[N][2];                      // the last key that a row sees (or less than 0), and with a window
  bool fresh = true;                   // an item begins here
  int begun = 0;                       // ... at this unit of it
  int stage = 0;
  while (left > 0) {
    if (fresh) {
      fresh = false;
      begun = at.unit;
      const int h = at.item / p.tiles, row0 = (at.item - h * p.tiles) * 8 * N;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const int row = row0 + i * 8 + g;
        const int token = row / p.group, head = h * p.group + row - token * p.group;
        const bool ok = row < p.rows;
        const T* src = static_cast<const T*>(p.a.q) + at.b * p.a.q_stride[0] + (ok ? token : 0) * p.a.q_stride[1] +
                       (ok ? head : 0) * p.a.q_stride[2];
        float x[S::kChunks][16], top = 0.f;
#pragma unroll
        for (int j = 0; j < S::kChunks; ++j)
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int d = 64 * j + 16 * t + 8 * half;
            float w[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
            if (ok && d < c.dim) Vec8<T>::load(src + d, w);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              x[j][8 * half + k] = w[k];
              top = fmaxf(top, fabsf(w[k]));
            }
          }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        // the row's largest value in [2^13, 2^14); what is not finite stays so
        const int e = min(max(static_cast<int>(__float_as_uint(top) >> 23) - 127 - 13, -100), 115);
        const float down = __uint_as_float(static_cast<uint32_t>(127 - e) << 23);
#pragma unroll
        for (int j = 0; j < S::kChunks; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const __half2 w = __floats2half2_rn(x[j][4 * k + 2 * half] * down, x[j][4 * k + 2 * half + 1] * down);
              q[i][j][k][half] = *reinterpret_cast<const uint32_t*>(&w);
            }
        // the two rows whose scores this lane has
        const float up = __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * p.scale_log2;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          factor[i][k] = __shfl_sync(0xffffffffu, up, (2 * t + k) * 4);
          const int r = row0 + i * 8 + 2 * t + k, tok = r / p.group;
          last[i][k] = r < p.rows && tok < at.count ? at.len - at.count + tok : -1;
          m[i][k] = -INFINITY;
          l[i][k] = 0.f;
        }
#pragma unroll
        for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][j][k] = 0.f;
      }
    }

    wait_copies<S::kStages - 2>();
    const uint32_t base = ring + stage * S::kStage + lane * 16;
    float s[N][4];
#pragma unroll
    for (int i = 0; i < N; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
#pragma unroll
    for (int j = 0; j < S::kChunks; ++j) {
      const uint4 k0 = read16(base + (j * 2) * 512), k1 = read16(base + (j * 2 + 1) * 512);
      const uint32_t w0[4] = {k0.x, k0.y, k0.z, k0.w}, w1[4] = {k1.x, k1.y, k1.z, k1.w};
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const uint2 a = halves(w0[k]), b = halves(w1[k]);
#pragma unroll
        for (int i = 0; i < N; ++i) product(s[i], a.x, b.x, a.y, b.y, q[i][j][k][0], q[i][j][k][1]);
      }
    }
    const uint32_t scales = ring + stage * S::kStage + 32 * (S::kKey + S::kValue) + lane * 8;
    const float k_scale = read4(scales), v_scale = read4(scales + 4);
    uint32_t w[4][S::kValues / 4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if constexpr (kWide) {
        const uint4 x = read16(base + 32 * S::kKey + r * 512);
        w[r][0] = x.x; w[r][1] = x.y; w[r][2] = x.z; w[r][3] = x.w;
      } else {
        const uint2 x = read8(ring + stage * S::kStage + 32 * S::kKey + r * 256 + lane * 8);
        w[r][0] = x.x; w[r][1] = x.y;
      }
    }
    const bool no_page = (missing >> stage) & 1;
    // (what the stage before held is in registers and used)
    issue(stage == 0 ? S::kStages - 1 : stage - 1);
    stage = stage + 1 == S::kStages ? 0 : stage + 1;

    const int key0 = (at.first_unit + at.unit) * kUnit;
    uint32_t pb[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float shrink[2];
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const float f = factor[i][k] * k_scale;
        const int from = p.a.window > 0 ? last[i][k] - p.a.window : -1;
        float x[2], top = m[i][k];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = key0 + g + 8 * r;
          x[r] = key <= last[i][k] && key > from && !no_page ? s[i][2 * r + k] * f : -INFINITY;
          top = fmaxf(top, x[r]);
        }
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float use = top == -INFINITY ? 0.f : top;
        shrink[k] = exp2f(m[i][k] - use);
        m[i][k] = top;
        const float p0 = exp2f(x[0] - use), p1 = exp2f(x[1] - use);
        l[i][k] = l[i][k] * shrink[k] + p0 + p1;
        s[i][k] = p0;
        s[i][2 + k] = p1;
      }
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const __half2 h2 = __floats2half2_rn(s[i][2 * r], s[i][2 * r + 1]);
        pb[i][r] = transposed(*reinterpret_cast<const uint32_t*>(&h2));
      }
#pragma unroll
      for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k) o[i][j][k] *= shrink[k & 1];
    }
#pragma unroll
    for (int j = 0; j < S::kTiles / 2; ++j) {
      // values 4 j .. 4 j + 3 of this lane's, of keys 2 t, 2 t + 1 and eight further
      const uint2 a = halves(bytes(w[0][j], w[1][j], 0x5140)), b = halves(bytes(w[2][j], w[3][j], 0x5140));
      const uint2 e = halves(bytes(w[0][j], w[1][j], 0x7362)), f = halves(bytes(w[2][j], w[3][j], 0x7362));
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
        product(x, a.x, a.y, b.x, b.y, pb[i][0], pb[i][1]);
        product(y, e.x, e.y, f.x, f.y, pb[i][0], pb[i][1]);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          o[i][2 * j][k] = fmaf(x[k], v_scale, o[i][2 * j][k]);
          o[i][2 * j + 1][k] = fmaf(y[k], v_scale, o[i][2 * j + 1][k]);
        }
      }
    }

    --left;
    const bool complete = at.unit + 1 == at.units;
    if (complete || left == 0) {
      const int h = at.item / p.tiles, row0 = (at.item - h * p.tiles) * 8 * N;
      const bool whole = complete && begun == 0;
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          float sum = l[i][k];
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
          const int in_tile = i * 8 + 2 * t + k, row = row0 + in_tile;
          if (row >= p.rows) continue;
          const float scale = whole ? (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)) : 1.f;
          float* part = part_of(p, number, begun == 0 ? 1 : 0, in_tile);
          const int token = row / p.group;
          T* out = static_cast<T*>(p.a.out) +
                   ((static_cast<int64_t>(at.b) * c.n + token) * p.a.q_heads + h * p.group + row - token * p.group) * c.dim;
#pragma unroll
          for (int j = 0; j < S::kValues / 8; ++j) {
            const int d = S::kValues * g + 8 * j;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = o[i][4 * j + e / 2][2 * (e & 1) + k] * scale;
            if (d >= c.dim) continue;
            if (whole) Vec8<T>::store(out + d, x);
            else Vec8<float>::store(part + d, x);
          }
          if (!whole && g == 0) {
            part[c.dim] = m[i][k];
            part[c.dim + 1] = sum;
          }
        }
      fresh = true;
    }
    step(at);
  }
}

// An item's parts added up, where more than one warp had it; zeros where none had
template <typename T>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Plan p) {
  const PagedCache& c = p.a.cache;
  __shared__ float s_m[8], s_l[8], s_o[8][128];
  const int items = c.heads * p.tiles;
  const int b = blockIdx.x / items, item = blockIdx.x - b * items;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const Shares shares = count_units(p);
  int64_t before = 0;
  for (int x = lane; x < b; x += 32) {
    int first, units, len, count;
    keys_of(c, p.a.window, x, first, units, len, count);
    before += units;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  int first, units, len, count;
  keys_of(c, p.a.window, b, first, units, len, count);
  const int64_t begin = before * items + static_cast<int64_t>(item) * units;
  const int w0 = static_cast<int>(begin / shares.per), w1 = static_cast<int>((begin + units - 1) / shares.per);
  pdl_wait();
  if (units > 0 && w0 == w1) return;
  const int h = item / p.tiles, row0 = (item - h * p.tiles) * p.tile_rows;
  const int rows = min(p.tile_rows, p.rows - row0);
  for (int r = 0; r < rows; ++r) {
    const int row = row0 + r, token = row / p.group;
    // each warp every eighth part, four values of a head to a lane
    float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
    const int d = lane * 4;
    if (units > 0) {
      for (int w = w0 + warp; w <= w1; w += 8) {
        const float* part = part_of(p, w, w == w0 ? 1 : 0, r);
        const float pm = part[c.dim], pl = part[c.dim + 1];
        const float top = fmaxf(m, pm), use = top == -INFINITY ? 0.f : top;
        const float f0 = exp2f(m - use), f1 = exp2f(pm - use);
        l = l * f0 + pl * f1;
        if (d < c.dim) {
          const float4 x = *reinterpret_cast<const float4*>(part + d);
          o[0] = o[0] * f0 + x.x * f1;
          o[1] = o[1] * f0 + x.y * f1;
          o[2] = o[2] * f0 + x.z * f1;
          o[3] = o[3] * f0 + x.w * f1;
        }
        m = top;
      }
    }
    __syncthreads();
    if (lane == 0) {
      s_m[warp] = m;
      s_l[warp] = l;
    }
    *reinterpret_cast<float4*>(&s_o[warp][d]) = make_float4(o[0], o[1], o[2], o[3]);
    __syncthreads();
    float top = -INFINITY;
#pragma unroll
    for (int w = 0; w < 8; ++w) top = fmaxf(top, s_m[w]);
    const float use = top == -INFINITY ? 0.f : top;
    if (threadIdx.x < c.dim) {
      float sum = 0.f, x = 0.f;
#pragma unroll
      for (int w = 0; w < 8; ++w) {
        const float f = exp2f(s_m[w] - use);
        sum += s_l[w] * f;
        x += s_o[w][threadIdx.x] * f;
      }
      T* out = static_cast<T*>(p.a.out) +
               ((static_cast<int64_t>(b) * c.n + token) * p.a.q_heads + h * p.group + row - token * p.group) * c.dim;
      out[threadIdx.x] = static_cast<T>(x * (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)));
    }
  }
}

Plan make_plan(const PagedAttention& a) {
  const PagedCache& c = a.cache;
  Plan p;
  p.a = a;
  p.group = a.q_heads / c.heads;
  p.rows = p.group * c.n;
  p.tile_rows = p.rows <= 8 ? 8 : p.rows <= 16 ? 16 : 32;
  p.tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  p.page_units = 0;
  while ((kUnit << p.page_units) < c.page) ++p.page_units;
  p.words = c.dim + 4;           // (rows on 16 bytes)
  p.scale_log2 = a.scale * kLog2e;
  // units if all sequences fill their rows of the table
  const int64_t units = static_cast<int64_t>(c.B) * c.heads * p.tiles * ((static_cast<int64_t>(c.table_pages) * c.page) / kUnit);
  const int64_t ctas = (units + kLeastUnits * kWarps - 1) / (kLeastUnits * kWarps);
  p.warps = static_cast<int>(ctas < sm_count() ? (ctas > 0 ? ctas : 1) : sm_count()) * kWarps;
  return p;
}

template <bool kWide, int N, typename T>
int launch_tiles(const Plan& p, cudaStream_t stream) {
  using S = Shape<kWide, N, T>;
  auto kernel = paged_attention_kernel<kWide, N, T>;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 3;
  static bool configured[64] = {};
  if (device < 0 || device >= 64) return 3;
  if (!configured[device]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return 3;
    configured[device] = true;
  }
  count_launch();
  kernel<<<p.warps / kWarps, kWarps * 32, S::kSmem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return 4;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(p.a.cache.B * p.a.cache.heads * p.tiles));
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&config, paged_combine_kernel<T>, p) == cudaSuccess ? 0 : 4;
}

template <bool kWide, typename T>
int launch_rows(const Plan& p, cudaStream_t stream) {
  if (p.tile_rows == 8) return launch_tiles<kWide, 1, T>(p, stream);
  if (p.tile_rows == 16) return launch_tiles<kWide, 2, T>(p, stream);
  return launch_tiles<kWide, 4, T>(p, stream);
}

}  // namespace

int64_t paged_attention_words(const PagedAttention& a) {
  const Plan p = make_plan(a);
  return static_cast<int64_t>(p.warps) * 2 * p.tile_rows * p.words;
}

int launch_paged_attention(const PagedAttention& a, cudaStream_t stream) {
  const PagedCache& c = a.cache;
  if (c.B == 0 || c.n == 0 || a.q_heads == 0) return 0;
  if (c.dim < 8 || c.dim > 128 || c.dim % 8 != 0 || c.pitch != (c.dim + 15) / 16 * 16) return 1;
  if (c.page != 16 && c.page != 32 && c.page != 64 && c.page != 128) return 2;
  const Plan p = make_plan(a);
  if (static_cast<int64_t>(c.B) * c.heads * p.tiles > 0x7fffffff) return 5;
  if (c.dim > 64) return a.bf16 ? launch_rows<true, __nv_bfloat16>(p, stream) : launch_rows<true, __half>(p, stream);
  return a.bf16 ? launch_rows<false, __nv_bfloat16>(p, stream) : launch_rows<false, __half>(p, stream);
}

}  // namespace slapo
