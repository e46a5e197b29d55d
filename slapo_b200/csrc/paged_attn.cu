// Attention of a sequence's newest tokens over a paged cache in 8 bits.
//
// Row r of a cached head is query t = r / G of query head r % G of its G; it sees the keys up to its own position (and
// not before its window).  With codes k, v and a page's scales ks, vs: s = ks (q k) scale, o = sum p vs v / sum p.
//
// Bound by reading the cache and, nearly as much, by the instructions around it.  A warp works alone, on units of 32 keys of
// one head: S^T = K Q^T by m16n8k16 of fp16 (16 keys, 8 rows), O^T += V^T P^T (16 values of a head, 8 rows), codes
// converted - exactly - on their way into the registers (products of e4m3 numbers, with the queries taken apart into two or
// three, are converted by the hardware's own instructions: as many).  The tensor core's order of the contraction is free as
// long as both operands share it, so that a lane's 16 bytes of a key are its operands of four products, and 16 bytes each of
// four values' rows, bytes interleaved, those of eight.  Units come by cp.async, 512 bytes of a page side by side at a time
// (lanes that copied what they read themselves, 64 bytes of each of eight tokens at a time, took 1.3 times as long), into a
// ring in shared memory of the warp's own: no barriers.  mma.sync and not tcgen05: a unit has one to eight rows of work, and
// the codes pass through registers, since they are converted.
//
// Keys are dealt out over all warps evenly, whatever the sequences' lengths, which are in device memory: each warp counts
// the units of all sequences and takes its share of their row, at least kLeastUnits; it writes an item (sequence, head,
// rows) that lies wholly in its share, and leaves its part of the first and the last else, which a second kernel adds up.
//
// Roundings: queries to fp16 by a power of two per row (exact, but for bf16 values below 2^-28 of the row's largest);
// weights, raised by 2^14, to fp16 as the products' operands: 2^-11 of themselves down to 2^-28 of the largest that the warp
// has seen, below that 2^-39 of it; all else in fp32.  (The output's own rounding is larger: errors against 64 bits 0.0016 -
// 0.0017 in bf16 and 0.00022 in fp16, with weights in fp32 0.0016 - 0.0017 and 0.00021.  With the largest weight as 1, those below
// 2^-14 lost bits and those below 2^-25 were none, while the sum had them: 6 % off where 12000 keys shared 1e-3 of the weight.)
#include <cuda_fp8.h>

#include "flash_common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

// Warps of a CTA by the tiles of 8 rows that each has: of up to 168 and of up to 255 registers.  (One tile, us, eight warps with
// three units in the ring of each / twelve with two: 16 tokens over up to 32001 keys of 4 heads 51.9 / 52.1, one over up to 1501
// of 16 15.1 / 15.3, five with a window of 1001 18.5 / 17.2.  Sixteen with one: 61, 16.6, 20.6.)
constexpr int warps_of(int tiles) { return tiles == 1 ? 12 : 8; }
constexpr int kUnit = 32;          // keys: two blocks of 16
constexpr int kLeastUnits = 2;     // of a warp's share
constexpr float kRaise = 14.f;     // log2 of what weights are raised by (fp16 ends at 2^16)
constexpr float kLower = 1.f / 16384.f;

// What is known of the work before lengths are: the same in both kernels
struct Plan {
  PagedAttention a;
  int group, rows, tiles, tile_rows, warps, words;     // tiles of rows per head; words: of a row's part
  int page_blocks;                                     // log2 of a page's blocks of 16 keys
  int piece_inverse;                                   // 2^16 / (a token's pieces of 16 bytes), rounded up
  float scale_log2;
};

// A sequence's units: those with a key that one of its rows sees
struct Keys {
  int len, count, first_unit, units;
};
__device__ __forceinline__ Keys keys_of(const PagedCache& c, int window, int b) {
  Keys k;
  k.count = c.counts != nullptr ? min(max(c.counts[b], 0), c.n) : c.n;
  const int64_t most = static_cast<int64_t>(c.table_pages) * c.page;
  k.len = c.lengths[b];
  const int seen = static_cast<int>(min(static_cast<int64_t>(max(k.len, 0)), most));
  const int64_t first = window > 0 ? static_cast<int64_t>(k.len) - k.count - window + 1 : 0;
  k.first_unit = first > 0 ? static_cast<int>(min(first, most)) / kUnit : 0;
  k.units = k.count > 0 ? max((seen + kUnit - 1) / kUnit - k.first_unit, 0) : 0;
  return k;
}
__device__ __forceinline__ int64_t warp_sum_long(int64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
// (a division of 64 bits takes some hundred instructions)
__device__ __forceinline__ int64_t quotient(int64_t a, int b) {
  if (a <= 0x7fffffff) return static_cast<int>(a) / b;
  return a / b;
}
// Units of a warp's share, of `units` per item and all sequences
__device__ __forceinline__ int64_t share_of(const Plan& p, int64_t units) {
  const int64_t total = units * p.a.cache.heads * p.tiles;
  return max(quotient(total + p.warps - 1, p.warps), static_cast<int64_t>(kLeastUnits));
}

__device__ __forceinline__ void copy16(uint32_t to, const void* from, bool ok) {
  const int n = ok ? 16 : 0;
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy4(uint32_t to, const void* from, bool ok) {
  const int n = ok ? 4 : 0;
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(n) : "memory");
}
__device__ __forceinline__ void commit_copies() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void wait_copies() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void clear16(uint32_t at) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at), "r"(0) : "memory");
}
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
__device__ __forceinline__ float2 read8f(uint32_t at) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
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
template <bool kWide, int N>
struct Shape {
  static constexpr int kChunks = kWide ? 2 : 1;                   // of 64 values of a key
  static constexpr int kPieces = 4 * kChunks;                     // of 16 bytes of a token
  static constexpr int kBlock = 16 * 16 * kPieces;                // a block's bytes of keys, or of values, in a warp's ring
  static constexpr int kCopies = kPieces / 2;                     // ... of a lane, 16 each
  static constexpr int kScales = 4 * kBlock;                      // where a unit's four scales are
  static constexpr int kStage = kScales + 16;
  static constexpr int kWarps = warps_of(N);
  static constexpr int kStages = kWide ? (N == 2 ? 3 : 2) : (N == 1 ? 4 : 5);
  static constexpr int kTiles = kWide ? 8 : 4;                    // of 16 values of a head
  static constexpr int kValues = kWide ? 16 : 8;                  // consecutive ones that a lane has
  // the queries' operands: in registers for one tile or two, beside the ring for more
  static constexpr bool kSharedQ = N > 2;
  static constexpr int kQuery = kSharedQ ? N * kChunks * 2 * 512 : 0;
  static constexpr int kWarp = kStages * kStage + kQuery;
  static constexpr int kSmem = kWarps * kWarp;
  // where a piece of a token lies in a block
  static __device__ __forceinline__ uint32_t place(int row, int piece) {
    const int order = kWide ? (((row >> 1) & 3) << 1) ^ ((row & 1) << 2) : (row >> 1) & 3;
    return (row * kPieces + (piece ^ order)) * 16;
  }
};

// A place in the row of all units
struct Cursor {
  int b, item, unit;
  Keys keys;
};

// what a warp leaves of the item that it begins with (0) or ends with (1): a row of `words` floats for each row of the tile
__device__ __forceinline__ float* part_of(const Plan& p, int warp, int which, int row) {
  return p.a.scratch + ((static_cast<int64_t>(warp) * 2 + which) * p.tile_rows + row) * p.words;
}

// This warp's first unit and how many it has.  All lanes count the sequences' units together.
__device__ __forceinline__ int begin_share(const Plan& p, int number, Cursor& at) {
  const PagedCache& c = p.a.cache;
  const int lane = threadIdx.x & 31;
  Keys mine{};                     // of sequence `lane`, where there are at most 32
  int64_t sum = 0;
  for (int b = lane; b < c.B; b += 32) {
    mine = keys_of(c, p.a.window, b);
    sum += mine.units;
  }
  const int64_t all = warp_sum_long(sum), items = static_cast<int64_t>(c.heads) * p.tiles, per = share_of(p, all);
  const int64_t target = number * per;
  if (target >= all * items) return 0;
  int64_t before = 0;
  for (int b0 = 0;; b0 += 32) {        // (ends: the target is before the end)
    if (c.B > 32) mine = b0 + lane < c.B ? keys_of(c, p.a.window, b0 + lane) : Keys{};
    int64_t until = mine.units * items;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t x = __shfl_up_sync(0xffffffffu, until, o);
      if (lane >= o) until += x;
    }
    const unsigned past = __ballot_sync(0xffffffffu, before + until > target);
    if (past == 0) {
      before += __shfl_sync(0xffffffffu, until, 31);
      continue;
    }
    const int l = __ffs(past) - 1;
    at.b = b0 + l;
    at.keys.len = __shfl_sync(0xffffffffu, mine.len, l);
    at.keys.count = __shfl_sync(0xffffffffu, mine.count, l);
    at.keys.first_unit = __shfl_sync(0xffffffffu, mine.first_unit, l);
    at.keys.units = __shfl_sync(0xffffffffu, mine.units, l);
    const int64_t in = target - (before + __shfl_sync(0xffffffffu, until, l) - at.keys.units * items);
    at.item = static_cast<int>(quotient(in, at.keys.units));
    at.unit = static_cast<int>(in - static_cast<int64_t>(at.item) * at.keys.units);
    return static_cast<int>(min(per, all * items - target));
  }
}

template <bool kWide, int N, bool kSmallPages, typename T>
__global__ void __launch_bounds__(warps_of(N) * 32, 1) paged_attention_kernel(const Plan p) {
  using S = Shape<kWide, N>;
  extern __shared__ __align__(128) uint8_t s_ring[];
  const PagedCache& c = p.a.cache;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int number = warp * gridDim.x + blockIdx.x;        // (few shares: one to an SM)
  pdl_launch();
  Cursor at;
  int left = begin_share(p, number, at);
  if (left == 0) return;
  int to_issue = left;
  const uint32_t ring = static_cast<uint32_t>(__cvta_generic_to_shared(s_ring)) + warp * S::kWarp;
  const int head_bytes = c.page * c.pitch;
  const int64_t side_bytes = c.heads * static_cast<int64_t>(head_bytes);
  const uint8_t* lane_pages = c.pages + lane * 16;
  const int items = c.heads * p.tiles;

  Cursor in = at;
  auto step = [&](Cursor& x) {
    if (++x.unit < x.keys.units) return;
    x.unit = 0;
    if (++x.item < items) return;
    x.item = 0;
    while (++x.b < c.B) {
      x.keys = keys_of(c, p.a.window, x.b);
      if (x.keys.units > 0) return;
    }
  };
  // the pages of a unit's two blocks of keys; -1: none
  auto page_of = [&](const Cursor& x, int block) {
    const int number = ((x.keys.first_unit + x.unit) * 2 + block) >> p.page_blocks;
    if (kSmallPages && number >= c.table_pages) return -1;         // (of an odd number of blocks)
    const int id = __ldg(c.table + static_cast<int64_t>(x.b) * c.table_pages + number);
    return id >= 0 && id < c.n_pages ? id : -1;
  };
  constexpr int kPages = kSmallPages ? 2 : 1;
  int page[kPages];
#pragma unroll
  for (int i = 0; i < kPages; ++i) page[i] = page_of(in, i);
  unsigned missing = 0;        // two bits for a stage: its blocks that have no page
  // A block's 16 tokens lie side by side in a page: lanes copy 16 bytes side by side, to a row of 128 (64) bytes for each
  // token, whose pieces are in an order of its own, so that neither reading of them meets a bank twice (narrow: values twice).
  const int pieces = c.pitch / 16;
  uint32_t place[S::kCopies];
  int row_of[S::kCopies];
#pragma unroll
  for (int i = 0; i < S::kCopies; ++i) {
    const int piece = i * 32 + lane;
    row_of[i] = piece * p.piece_inverse >> 16;        // piece / pieces; 16 and more: none
    place[i] = S::place(row_of[i], piece - row_of[i] * pieces);
  }
  // (what lies behind a head's width is zeros from here on: the operands reach to 64 or 128 values)
  if (pieces < S::kPieces) {
    for (int i = lane; i < 4 * S::kStages * 16 * (S::kPieces - pieces); i += 32) {
      const int block = i / (16 * (S::kPieces - pieces)), in_block = i - block * 16 * (S::kPieces - pieces);
      const int row = in_block / (S::kPieces - pieces), piece = pieces + in_block - row * (S::kPieces - pieces);
      clear16(ring + block / 4 * S::kStage + block % 4 * S::kBlock + S::place(row, piece));
    }
    __syncwarp();
  }
  // the unit's codes and scales on their way into a stage; the next unit's pages are read ahead
  auto issue = [&](int stage) {
    if (to_issue > 0) {
      --to_issue;
      const int key0 = (in.keys.first_unit + in.unit) * kUnit, h = p.tiles == 1 ? in.item : in.item / p.tiles;
      const uint32_t to = ring + stage * S::kStage;
      missing &= ~(3u << (2 * stage));
      // keys that no row sees are zeros: a hidden code may be a NaN
      const int until = in.keys.len - key0;
      // (the first row's first key; no less than 1 - window: a window may have all 31 bits)
      const int from = p.a.window > 0 ? max(until - in.keys.count, 0) + 1 - p.a.window : 0;
      const bool every = page[0] >= 0 && page[kPages - 1] >= 0 && until >= kUnit && from <= 0;
      const uint8_t* k = nullptr;
#pragma unroll
      for (int block = 0; block < 2; ++block) {
        const int id = page[kSmallPages ? block : 0];
        // (a page without a key that is seen may never have been written, its scales neither)
        const bool known = every || (id >= 0 && (!kSmallPages || (until > 16 * block && from < 16 * block + 16)));
        if (kSmallPages || block == 0) {
          const int64_t side = (static_cast<int64_t>(known ? id : 0) * 2) * c.heads + h;
          k = lane_pages + side * head_bytes + ((key0 + 16 * block) & (c.page - 1)) * c.pitch;
          // keys' and values' scale by one lane each
          if (lane < 2) copy4(to + S::kScales + 8 * block + 4 * lane, c.scales + side + lane * c.heads, known);
        } else {
          k += 16 * c.pitch;
        }
        const uint8_t* v = k + side_bytes;
        const uint32_t k_to = to + 2 * block * S::kBlock, v_to = k_to + S::kBlock;
        if (every) {
#pragma unroll
          for (int i = 0; i < S::kCopies; ++i) {
            if (row_of[i] < 16) {
              copy16(k_to + place[i], k + i * 512);
              copy16(v_to + place[i], v + i * 512);
            }
          }
        } else {
          if (!known) missing |= 1u << (2 * stage + block);
#pragma unroll
          for (int i = 0; i < S::kCopies; ++i) {
            if (row_of[i] < 16) {
              const int key = 16 * block + row_of[i];
              const bool ok = known && key < until && key >= from;
              copy16(k_to + place[i], ok ? k + i * 512 : c.pages, ok);
              copy16(v_to + place[i], ok ? v + i * 512 : c.pages, ok);
            }
          }
        }
      }
      step(in);
      if (to_issue > 0) {
#pragma unroll
        for (int i = 0; i < kPages; ++i) page[i] = page_of(in, i);
      }
    }
    commit_copies();
  };
#pragma unroll 1
  for (int i = 0; i < S::kStages - 1; ++i) issue(i);

  const uint32_t q_at = ring + S::kStages * S::kStage + lane * 16;
  uint32_t q[S::kSharedQ ? 1 : N][S::kChunks][2][4];
  // m: what a row's scores are measured by, kRaise below its largest; l: the raised weights' sum
  float factor[N][2], m[N][2], l[N][2], o[N][S::kTiles][4];
  int last[N][2];                      // the last key that a row sees, less than 0: none
  // where this lane's operands are in a block: of keys g and g + 8, of values' rows 2 t, 2 t + 1 and eight further
  const uint32_t key_at[2] = {S::place(g, t), S::place(g, kWide ? 4 + t : t)};
  const uint32_t value_at[2] = {S::place(2 * t, kWide ? g : g / 2) + (kWide ? 0 : 8 * (g & 1)),
                                S::place(2 * t + 1, kWide ? g : g / 2) + (kWide ? 0 : 8 * (g & 1))};
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
          for (int half = 0; half < 2; ++half) {
            uint32_t w[4];
#pragma unroll
            for (int y = 0; y < 4; ++y) {
              const __half2 pair = __floats2half2_rn(x[j][8 * half + 2 * y] * down, x[j][8 * half + 2 * y + 1] * down);
              w[y] = *reinterpret_cast<const uint32_t*>(&pair);
            }
            if constexpr (S::kSharedQ) {
              asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(q_at + ((i * S::kChunks + j) * 2 + half) * 512),
                           "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
            } else {
#pragma unroll
              for (int y = 0; y < 4; ++y) q[i][j][half][y] = w[y];
            }
          }
        // the two rows whose scores this lane has
        // (an infinite query's row: NaN)
        const float up = top <= 3.402823466e38f ? __uint_as_float(static_cast<uint32_t>(127 + e) << 23) * p.scale_log2
                                                : __uint_as_float(0x7fffffffu);
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          factor[i][k] = __shfl_sync(0xffffffffu, up, (2 * t + k) * 4);
          const int r = row0 + i * 8 + 2 * t + k, tok = r / p.group;
          last[i][k] = r < p.rows && tok < at.keys.count ? at.keys.len - at.keys.count + tok : -1;
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
    __syncwarp();                      // (what a lane reads others have copied)
    const uint32_t base = ring + stage * S::kStage;
    const unsigned gone = (missing >> (2 * stage)) & 3u;
    float s[N][2][4];
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int block = 0; block < 2; ++block) s[i][block][0] = s[i][block][1] = s[i][block][2] = s[i][block][3] = 0.f;
#pragma unroll
    for (int j = 0; j < S::kChunks; ++j) {
      uint4 keys[2][2];
#pragma unroll
      for (int block = 0; block < 2; ++block)
#pragma unroll
        for (int r = 0; r < 2; ++r)
          keys[block][r] = read16(base + 2 * block * S::kBlock + r * 8 * 16 * S::kPieces + (j == 0 ? key_at[0] : key_at[1]));
#pragma unroll
      for (int half = 0; half < 2; ++half) {
        uint2 a[2][2], b[2][2];        // words 2 half and 2 half + 1 of each block's keys g and g + 8
#pragma unroll
        for (int block = 0; block < 2; ++block) {
          const uint4 &k0 = keys[block][0], &k1 = keys[block][1];
          a[block][0] = halves(half == 0 ? k0.x : k0.z);
          a[block][1] = halves(half == 0 ? k0.y : k0.w);
          b[block][0] = halves(half == 0 ? k1.x : k1.z);
          b[block][1] = halves(half == 0 ? k1.y : k1.w);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          uint32_t w[4];
          if constexpr (S::kSharedQ) {
            const uint4 x = read16(q_at + ((i * S::kChunks + j) * 2 + half) * 512);
            w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
          } else {
#pragma unroll
            for (int y = 0; y < 4; ++y) w[y] = q[i][j][half][y];
          }
#pragma unroll
          for (int y = 0; y < 2; ++y)
#pragma unroll
            for (int block = 0; block < 2; ++block)
              product(s[i][block], a[block][y].x, b[block][y].x, a[block][y].y, b[block][y].y, w[2 * y], w[2 * y + 1]);
        }
      }
    }
    float k_scale[2], v_scale[2];
    {
      const float2 x = read8f(base + S::kScales);
      k_scale[0] = k_scale[1] = x.x;
      v_scale[0] = v_scale[1] = x.y * kLower;
      if constexpr (kSmallPages) {
        const float2 y = read8f(base + S::kScales + 8);
        k_scale[1] = y.x;
        v_scale[1] = y.y * kLower;
      }
    }

    const int key0 = (at.keys.first_unit + at.unit) * kUnit;
    // whether every row sees all of the unit's keys
    const bool all = gone == 0 && key0 + kUnit <= at.keys.len - at.keys.count + 1 &&
                     (p.a.window == 0 || key0 > at.keys.len - 1 - p.a.window);
    uint32_t pb[N][2][2];
    bool grown = false;
    float shrink[N][2];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        float x[4], top = -INFINITY;
#pragma unroll
        for (int block = 0; block < 2; ++block)
#pragma unroll
          for (int r = 0; r < 2; ++r) x[2 * block + r] = s[i][block][2 * r + k] * (factor[i][k] * k_scale[block]);
        if (!all) {
          const int from = p.a.window > 0 ? last[i][k] - p.a.window : -1;
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const int key = key0 + g + 8 * y;
            if (!(key <= last[i][k] && key > from) || ((gone >> (y >> 1)) & 1u) != 0) x[y] = -INFINITY;
          }
        }
#pragma unroll
        for (int y = 0; y < 4; ++y) top = fmaxf(top, x[y]);
#pragma unroll
        for (int off = 4; off < 32; off <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, off));
        const float next = fmaxf(m[i][k], top - kRaise), use = next == -INFINITY ? 0.f : next;
        grown |= next > m[i][k];
        shrink[i][k] = exp2f(m[i][k] - use);
        m[i][k] = next;
        float sum = 0.f;
#pragma unroll
        for (int y = 0; y < 4; ++y) {
          const float e = exp2f(x[y] - use);
          sum += e;
          s[i][y >> 1][2 * (y & 1) + k] = e;
        }
        l[i][k] = l[i][k] * shrink[i][k] + sum;
      }
#pragma unroll
      for (int block = 0; block < 2; ++block)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const __half2 h2 = __floats2half2_rn(s[i][block][2 * r], s[i][block][2 * r + 1]);
          pb[i][block][r] = transposed(*reinterpret_cast<const uint32_t*>(&h2));
        }
    }
    if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
      for (int i = 0; i < N; ++i)
#pragma unroll
        for (int j = 0; j < S::kTiles; ++j)
#pragma unroll
          for (int k = 0; k < 4; ++k) o[i][j][k] *= shrink[i][k & 1];
    }
    uint32_t w[2][4][S::kValues / 4];
#pragma unroll
    for (int block = 0; block < 2; ++block)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        // (rows 2 t and 2 t + 1, and eight further)
        const uint32_t v_from = base + (2 * block + 1) * S::kBlock + (r >> 1) * 8 * 16 * S::kPieces + value_at[r & 1];
        if constexpr (kWide) {
          const uint4 x = read16(v_from);
          w[block][r][0] = x.x; w[block][r][1] = x.y; w[block][r][2] = x.z; w[block][r][3] = x.w;
        } else {
          const uint2 x = read8(v_from);
          w[block][r][0] = x.x; w[block][r][1] = x.y;
        }
      }
    __syncwarp();                      // (all lanes have read the stage before)
    issue(stage == 0 ? S::kStages - 1 : stage - 1);
    stage = stage + 1 == S::kStages ? 0 : stage + 1;
#pragma unroll
    for (int j = 0; j < S::kTiles / 2; ++j) {
      // values 4 j .. 4 j + 3 of this lane's, of keys 2 t, 2 t + 1 and eight further
      uint2 a[2], b[2], e[2], f[2];
#pragma unroll
      for (int block = 0; block < 2; ++block) {
        const auto& x = w[block];
        a[block] = halves(bytes(x[0][j], x[1][j], 0x5140));
        b[block] = halves(bytes(x[2][j], x[3][j], 0x5140));
        e[block] = halves(bytes(x[0][j], x[1][j], 0x7362));
        f[block] = halves(bytes(x[2][j], x[3][j], 0x7362));
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float x[4] = {0.f, 0.f, 0.f, 0.f}, y[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int block = 0; block < 2; ++block) {
          product(x, a[block].x, a[block].y, b[block].x, b[block].y, pb[i][block][0], pb[i][block][1]);
          product(y, e[block].x, e[block].y, f[block].x, f[block].y, pb[i][block][0], pb[i][block][1]);
          if (kSmallPages || block == 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              o[i][2 * j][k] = fmaf(x[k], v_scale[block], o[i][2 * j][k]);
              o[i][2 * j + 1][k] = fmaf(y[k], v_scale[block], o[i][2 * j + 1][k]);
              x[k] = y[k] = 0.f;
            }
          }
        }
      }
    }

    --left;
    const bool complete = at.unit + 1 == at.keys.units;
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
          sum *= kLower;
          const int in_tile = i * 8 + 2 * t + k, row = row0 + in_tile;
          if (row >= p.rows) continue;
          const bool none = last[i][k] < 0;         // (masks are not applied where all rows see all keys)
          const float scale = none ? 0.f : whole ? (sum > 0.f ? 1.f / sum : (sum == 0.f ? 0.f : sum)) : 1.f;
          float* part = part_of(p, number, begun == 0 ? 1 : 0, in_tile);
          const int token = row / p.group;
          T* out = static_cast<T*>(p.a.out) +
                   ((static_cast<int64_t>(at.b) * c.n + token) * p.a.q_heads + h * p.group + row - token * p.group) * c.dim;
#pragma unroll
          for (int j = 0; j < S::kValues / 8; ++j) {
            const int d = S::kValues * g + 8 * j;
            float x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = none ? 0.f : o[i][4 * j + e / 2][2 * (e & 1) + k] * scale;
            if (d >= c.dim) continue;
            if (whole) Vec8<T>::store(out + d, x);
            else Vec8<float>::store(part + d, x);
          }
          if (!whole && g == 0) {
            part[c.dim] = none ? -INFINITY : m[i][k];
            part[c.dim + 1] = none ? 0.f : sum;
          }
        }
      fresh = true;
    }
    step(at);
  }
}

// A row's parts added up, where more than one warp had its item; zeros where none had
template <typename T>
__global__ void __launch_bounds__(256) paged_combine_kernel(const Plan p, int tile_rows) {
  const PagedCache& c = p.a.cache;
  __shared__ float s_m[8], s_l[8], s_o[8][128];
  const int items = c.heads * p.tiles;
  const int r = blockIdx.x % tile_rows, at = blockIdx.x / tile_rows;
  const int b = at / items, item = at - b * items;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = item / p.tiles, row = (item - h * p.tiles) * p.tile_rows + r;
  int64_t before = 0, sum_all = 0;
  Keys keys{};
  for (int x = lane; x < c.B; x += 32) {
    const Keys k = keys_of(c, p.a.window, x);
    sum_all += k.units;
    if (x < b) before += k.units;
    if (x == b) keys = k;
  }
  sum_all = warp_sum_long(sum_all);
  before = warp_sum_long(before);
  const int units = __shfl_sync(0xffffffffu, keys.units, b & 31);
  const int64_t per = share_of(p, sum_all);
  const int64_t begin = before * items + static_cast<int64_t>(item) * units;
  const int w0 = static_cast<int>(begin / per), w1 = static_cast<int>((begin + max(units, 1) - 1) / per);
  pdl_wait();
  if (row >= p.rows || (units > 0 && w0 == w1)) return;
  const int token = row / p.group;
  // each warp every eighth part, four values of a head to a lane
  float m = -INFINITY, l = 0.f, o[4] = {0.f, 0.f, 0.f, 0.f};
  const int d = lane * 4;
  if (units > 0) {
#pragma unroll 4
    for (int w = w0 + warp; w <= w1; w += 8) {
      const float* part = part_of(p, w, w == w0 ? 1 : 0, r);
      const float2 ml = *reinterpret_cast<const float2*>(part + c.dim);
      const float4 x = d < c.dim ? *reinterpret_cast<const float4*>(part + d) : make_float4(0.f, 0.f, 0.f, 0.f);
      const float top = fmaxf(m, ml.x), use = top == -INFINITY ? 0.f : top;
      const float f0 = exp2f(m - use), f1 = exp2f(ml.x - use);
      l = l * f0 + ml.y * f1;
      o[0] = o[0] * f0 + x.x * f1;
      o[1] = o[1] * f0 + x.y * f1;
      o[2] = o[2] * f0 + x.z * f1;
      o[3] = o[3] * f0 + x.w * f1;
      m = top;
    }
  }
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

Plan make_plan(const PagedAttention& a) {
  const PagedCache& c = a.cache;
  Plan p;
  p.a = a;
  p.group = a.q_heads / c.heads;
  p.rows = p.group * c.n;
  p.tile_rows = p.rows <= 8 ? 8 : p.rows <= 16 ? 16 : 32;
  p.tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
  p.page_blocks = 0;
  while ((16 << p.page_blocks) < c.page) ++p.page_blocks;
  p.piece_inverse = (65536 + c.pitch / 16 - 1) / (c.pitch / 16);        // (exact for the 128 pieces of a block)
  p.words = c.dim + 4;           // (rows on 16 bytes)
  p.scale_log2 = a.scale * kLog2e;
  // units if all sequences fill their rows of the table
  const int64_t units = static_cast<int64_t>(c.B) * c.heads * p.tiles *
                        ((static_cast<int64_t>(c.table_pages) * c.page + kUnit - 1) / kUnit);
  const int warps = warps_of(p.tile_rows / 8);
  const int64_t ctas = (units + kLeastUnits * warps - 1) / (kLeastUnits * warps);
  p.warps = static_cast<int>(ctas < sm_count() ? (ctas > 0 ? ctas : 1) : sm_count()) * warps;
  return p;
}

template <bool kWide, int N, bool kSmallPages, typename T>
int launch_tiles(const Plan& p, cudaStream_t stream) {
  using S = Shape<kWide, N>;
  static_assert(S::kSmem <= 227 * 1024, "a CTA's shared memory");
  auto kernel = paged_attention_kernel<kWide, N, kSmallPages, T>;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return 3;
  static bool configured[64] = {};
  if (device < 0 || device >= 64) return 3;
  if (!configured[device]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kSmem) != cudaSuccess) return 3;
    configured[device] = true;
  }
  count_launch();
  kernel<<<p.warps / S::kWarps, S::kWarps * 32, S::kSmem, stream>>>(p);
  if (cudaGetLastError() != cudaSuccess) return 4;
  cudaLaunchConfig_t config{};
  const int tile_rows = p.rows < p.tile_rows ? p.rows : p.tile_rows;
  config.gridDim = dim3(static_cast<unsigned>(p.a.cache.B) * p.a.cache.heads * p.tiles * tile_rows);
  config.blockDim = dim3(256);
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&config, paged_combine_kernel<T>, p, tile_rows) == cudaSuccess ? 0 : 4;
}

template <bool kWide, bool kSmallPages, typename T>
int launch_rows(const Plan& p, cudaStream_t stream) {
  if (p.tile_rows == 8) return launch_tiles<kWide, 1, kSmallPages, T>(p, stream);
  if (p.tile_rows == 16) return launch_tiles<kWide, 2, kSmallPages, T>(p, stream);
  return launch_tiles<kWide, 4, kSmallPages, T>(p, stream);
}

template <typename T>
int launch_heads(const Plan& p, cudaStream_t stream) {
  const bool small = p.a.cache.page < kUnit;
  if (p.a.cache.dim > 64) return small ? launch_rows<true, true, T>(p, stream) : launch_rows<true, false, T>(p, stream);
  return small ? launch_rows<false, true, T>(p, stream) : launch_rows<false, false, T>(p, stream);
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
  if (static_cast<int64_t>(c.B) * c.heads * p.tiles * p.tile_rows > 0x7fffffff) return 5;
  return a.bf16 ? launch_heads<__nv_bfloat16>(p, stream) : launch_heads<__half>(p, stream);
}

}  // namespace slapo
