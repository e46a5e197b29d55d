// Token table: lookup with scaling, and its gradient by sorted tokens.
//   out[t] = scale W[id_t]          dW[v] = scale sum of dY[t] over the tokens t with id_t = v
// Ids outside of the table's rows [0, V) (of a shard: the other ranks' tokens) give rows of zeros and no gradient.
//
// The gradient of a table has few rows that anything is added to, some of them (frequent tokens, a padding id)
// from thousands of tokens.  Atomic additions would need an fp32 copy of the whole table, written three times, and
// their order would change the result from run to run.  Here tokens are sorted by id (a stable radix sort, so that
// a row's tokens stay in their order) and each warp adds up eight tokens in sorted order, all of their rows of dY on
// their way at once whichever rows they belong to: a row of one token and one of thousands cost the same per token.
// What belongs to one row is joined over a CTA's eight warps, and over CTAs by a second kernel (an eighth of a row's
// stretches to a warp), each time in order, so that the result is the same every time.
//
// Sorting is latency, not bytes: one cluster of up to eight CTAs does it, with digits of eight bits; per pass each
// warp counts the digits of its stretch (match.any: equal digits of 32 tokens at a time), offsets are added up over
// the warps, the CTAs (distributed shared memory) and the digits, and the warps go over their stretches again and
// place them.  The other clusters of the same launch fill the table's gradient with zeros meanwhile.
//
// Measured (us; lookup, sort and zeros, sums, joins): 16384 tokens, 30528 x 1024 bf16: 9, 20, 10, 5; 8192 tokens, 50304 x 2048:
// 9 (scaled), 35 (the zeros: 5.9 TB/s), 10, 5; both lookups and sums move their bytes at 6 - 7 TB/s, the sort alone is
// latency.
#include <cooperative_groups.h>

#include "common.cuh"
#include "kernels.h"

namespace cg = cooperative_groups;

namespace slapo {

// ------------------------------------------------------------------------ //
// What a thread takes of a row at a time: 16 bytes, or an element where rows do not keep to 16 bytes
template <typename T>
struct RowVec {      // 16 bytes of a row
  static constexpr int kN = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ void zero() { raw = make_uint4(0u, 0u, 0u, 0u); }
  __device__ __forceinline__ void load(const T* p) { raw = __ldg(reinterpret_cast<const uint4*>(p)); }
  __device__ __forceinline__ void store(T* p) const { *reinterpret_cast<uint4*>(p) = raw; }
  __device__ __forceinline__ void get(float (&v)[kN]) const {
    const T* e = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < kN; ++i) v[i] = static_cast<float>(e[i]);
  }
  __device__ __forceinline__ void set(const float (&v)[kN]) {
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < kN; ++i) e[i] = static_cast<T>(v[i]);
  }
};
template <typename T>
struct RowOne {      // an element
  static constexpr int kN = 1;
  T raw;
  __device__ __forceinline__ void zero() { raw = static_cast<T>(0.f); }
  __device__ __forceinline__ void load(const T* p) { raw = *p; }
  __device__ __forceinline__ void store(T* p) const { *p = raw; }
  __device__ __forceinline__ void get(float (&v)[1]) const { v[0] = static_cast<float>(raw); }
  __device__ __forceinline__ void set(const float (&v)[1]) { raw = static_cast<T>(v[0]); }
};

// A warp for each token and 128 vectors of its row, four to a lane.
template <typename T, typename V, typename Id>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const Id* __restrict__ ids, const T* __restrict__ w,
                                                            T* __restrict__ out, int64_t tokens, int vecs,
                                                            int parts, int64_t rows, int64_t row_stride,
                                                            int64_t start, float scale) {
  constexpr int kEach = 4;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5);
  const int64_t t = parts == 1 ? item : item / parts;
  if (t >= tokens) return;
  const int c0 = static_cast<int>(item - t * parts) * 32 * kEach + (threadIdx.x & 31);
  const int64_t row = static_cast<int64_t>(ids[t]) - start;
  const bool own = row >= 0 && row < rows;
  const T* from = w + (own ? row : 0) * row_stride;
  T* to = out + t * vecs * V::kN;
  V v[kEach];
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    v[u].zero();
    if (own && c0 + u * 32 < vecs) v[u].load(from + static_cast<int64_t>(c0 + u * 32) * V::kN);
  }
#pragma unroll
  for (int u = 0; u < kEach; ++u) {
    if (c0 + u * 32 >= vecs) break;
    if (scale != 1.f) {
      float f[V::kN];
      v[u].get(f);
#pragma unroll
      for (int k = 0; k < V::kN; ++k) f[k] *= scale;
      v[u].set(f);
    }
    v[u].store(to + static_cast<int64_t>(c0 + u * 32) * V::kN);
  }
}

// ------------------------------------------------------------------------ //
constexpr int kSortWarps = 32, kSortThreads = 32 * kSortWarps, kDigits = 256, kSortCtas = 8;
// shared memory for a CTA's slice beside 40 KB of counters, at most
constexpr int kSortSlices = 184 * 1024;

struct SortParams {
  const void* ids;
  int64_t start, padding;       // first row of the table, id without a gradient (or one that no token has)
  int n, rows, passes;
  int stretch;                  // tokens of a warp, a multiple of 32
  int slice;                    // ... and of a CTA
  int* key[2];                  // [n] each: rows in sorted order and ...
  int* pos[2];                  // ... where in `ids` they stand
  int2* sorted;                 // [n]: both together, the result
  int* ends;                    // [rows + 1]: the sorted place behind the tokens of each row that has any
  uint8_t* dw;                  // to be filled with zeros
  int64_t bytes;
};

// What the other clusters of the launch do: zeros, 32 bytes at a time
__device__ __forceinline__ void fill_zeros(const SortParams& p, int cta, int ctas) {
  const int64_t me = static_cast<int64_t>(cta) * kSortThreads + threadIdx.x, all = static_cast<int64_t>(ctas) * kSortThreads;
  const uint32_t zero[8] = {0u, 0u, 0u, 0u, 0u, 0u, 0u, 0u};
  uint8_t* first = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(p.dw) + 31) & ~static_cast<uintptr_t>(31));
  const int64_t head = min(p.bytes, static_cast<int64_t>(first - p.dw)), whole = (p.bytes - head) / 32;
#pragma unroll 4
  for (int64_t i = me; i < whole; i += all) store16_raw(first + i * 32, zero);
  const int64_t tail = head + whole * 32;
  if (me < head) p.dw[me] = 0;
  if (me < p.bytes - tail) p.dw[tail + me] = 0;
}

// kShared: between the passes each CTA holds its slice of the tokens in shared memory, and tokens are placed into the
// others' there (two buffers of `slice` rows and places); else they pass through the scratch in global memory.
template <typename Id, bool kShared>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortParams p) {
  extern __shared__ int slices[];
  __shared__ int count[kSortWarps][kDigits];       // of a warp's digits, then where its next token of a digit goes
  __shared__ int quarter[4][kDigits];              // of eight warps' digits each
  __shared__ int total[kDigits];                   // of the CTA's digits
  __shared__ int before[kDigits];                  // tokens with smaller digits, or of earlier CTAs
  __shared__ int carry[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  if (static_cast<int>(blockIdx.x) >= ctas) {
    fill_zeros(p, blockIdx.x - ctas, gridDim.x - ctas);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int64_t begin64 = static_cast<int64_t>(cta * kSortWarps + warp) * p.stretch;
  const int begin = begin64 < p.n ? static_cast<int>(begin64) : p.n;
  const int end = p.n - begin < p.stretch ? p.n : begin + p.stretch;
  const int d0 = threadIdx.x & (kDigits - 1), q0 = threadIdx.x >> 8;      // a digit and eight of the warps
  const int mine0 = cta * p.slice;
  if (kShared && ctas > 1) cluster.sync();       // (the others have begun: their shared memory can be written)
  for (int pass = 0; pass < p.passes; ++pass) {
    // rows and places as the pass before left them (written by other SMs of the cluster)
    const int* src_key = kShared ? slices + ((pass & 1) ^ 1) * 2 * p.slice - mine0 : p.key[(pass & 1) ^ 1];
    const int* src_pos = kShared ? src_key + p.slice : p.pos[(pass & 1) ^ 1];
    const int shift = 8 * pass;
    auto pos_at = [&](int i) -> int { return pass == 0 ? i : kShared ? src_pos[i] : __ldcg(src_pos + i); };
    auto key_at = [&](int i) -> int {
      if (pass > 0) return kShared ? src_key[i] : __ldcg(src_key + i);
      const int64_t id = static_cast<int64_t>(static_cast<const Id*>(p.ids)[i]);
      const int64_t row = id - p.start;
      return row >= 0 && row < p.rows && id != p.padding ? static_cast<int>(row) : p.rows;
    };
    // the first strips of 32 are kept from counting to placing
    constexpr int kKeep = 2;
    int kept_key[kKeep], kept_pos[kKeep];
#pragma unroll
    for (int s = 0; s < kKeep; ++s) {
      const int i = begin + s * 32 + lane;
      kept_key[s] = i < end ? key_at(i) : 0;
      kept_pos[s] = i < end ? pos_at(i) : 0;
    }
#pragma unroll
    for (int d = 0; d < kDigits; d += 32) count[warp][d + lane] = 0;
    __syncwarp();
    for (int i0 = begin, s = 0; i0 < end; i0 += 32, ++s) {
      const int i = i0 + lane;
      const bool ok = i < end;
      const int key = s == 0 ? kept_key[0] : s == 1 ? kept_key[1] : ok ? key_at(i) : 0;
      const int d = ok ? (key >> shift) & (kDigits - 1) : kDigits;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (ok && (same & ((1u << lane) - 1u)) == 0u) count[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    int mine[8], sum = 0;
#pragma unroll
    for (int w = 0; w < 8; ++w) mine[w] = count[q0 * 8 + w][d0];
#pragma unroll
    for (int w = 0; w < 8; ++w) {
      const int c = mine[w];
      mine[w] = sum;
      sum += c;
    }
    quarter[q0][d0] = sum;
    __syncthreads();
    int ahead_of = 0;
#pragma unroll
    for (int q = 0; q < 3; ++q)
      if (q < q0) ahead_of += quarter[q][d0];
    if (q0 == 3) total[d0] = ahead_of + sum;
    cluster.sync();
    if (threadIdx.x < kDigits) {
      int t[kSortCtas], earlier = 0, all = 0;
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) t[c] = c < ctas ? cluster.map_shared_rank(total, c)[threadIdx.x] : 0;
#pragma unroll
      for (int c = 0; c < kSortCtas; ++c) {
        if (c < cta) earlier += t[c];
        all += t[c];
      }
      // exclusive sums over the digits: within the warp, then over the eight warps
      int inclusive = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += x;
      }
      if (lane == 31) carry[warp] = inclusive;
      before[threadIdx.x] = inclusive - all + earlier;
    }
    __syncthreads();
    int add = before[d0] + ahead_of;
#pragma unroll
    for (int w = 0; w < 8; ++w)
      if (w < d0 >> 5) add += carry[w];
#pragma unroll
    for (int w = 0; w < 8; ++w) count[q0 * 8 + w][d0] = mine[w] + add;
    __syncthreads();
    for (int i0 = begin, s = 0; i0 < end; i0 += 32, ++s) {
      const int i = i0 + lane;
      const bool ok = i < end;
      const int key = s == 0 ? kept_key[0] : s == 1 ? kept_key[1] : ok ? key_at(i) : 0;
      const int from = s == 0 ? kept_pos[0] : s == 1 ? kept_pos[1] : ok ? pos_at(i) : 0;
      const int d = ok ? (key >> shift) & (kDigits - 1) : kDigits;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const uint32_t ahead = same & ((1u << lane) - 1u);
      const int to = ok ? count[warp][d] + __popc(ahead) : 0;
      __syncwarp();
      if (ok && ahead == 0u) count[warp][d] = to + __popc(same);
      if (ok) {
        if constexpr (kShared) {
          const int there = to / p.slice;
          int* dst = cluster.map_shared_rank(slices, there) + (pass & 1) * 2 * p.slice + to - there * p.slice;
          dst[0] = key;
          dst[p.slice] = from;
        } else {
          p.key[pass & 1][to] = key;
          p.pos[pass & 1][to] = from;
        }
      }
      __syncwarp();
    }
    if (!kShared) __threadfence();
    cluster.sync();      // (the totals have been read, and what was placed is visible)
  }
  // where each row's tokens end
  const int buffer = (p.passes & 1) ^ 1, last = min(p.n, mine0 + p.slice);
  auto sorted_key = [&](int i) -> int {
    if constexpr (!kShared) return __ldcg(p.key[buffer] + i);
    const int there = i < mine0 + p.slice ? cta : cta + 1;
    return cluster.map_shared_rank(slices, there)[buffer * 2 * p.slice + i - there * p.slice];
  };
  for (int i = mine0 + threadIdx.x; i < last; i += kSortThreads) {
    const int k = sorted_key(i);
    if (i == p.n - 1 || sorted_key(i + 1) != k) p.ends[k] = i + 1;
    p.sorted[i] = make_int2(k, kShared ? slices[(buffer * 2 + 1) * p.slice + i - mine0] : __ldcg(p.pos[buffer] + i));
  }
  if (kShared && ctas > 1) cluster.sync();      // (nobody reads here any more)
}

struct EmbedGradParams {
  const void* dy;
  void* dw;
  const int2* sorted;   // rows and places of the tokens
  const int* ends;
  float* part;          // [stretches][2][cols]: of rows that go over stretches of 64 tokens, the sums of the row that a
                        // stretch begins in the middle of, and of the one that goes on behind it
  int n, rows;
  int64_t cols;
  int vecs, chunks;     // of a row, and 32 of them to a chunk
  float scale;
};

constexpr int kGradWarps = 8, kGradEach = 8, kGradStretch = kGradWarps * kGradEach;

template <typename T, typename V>
__device__ __forceinline__ void store_row(const EmbedGradParams& p, int row, int c, const float (&sum)[V::kN]) {
  float x[V::kN];
#pragma unroll
  for (int k = 0; k < V::kN; ++k) x[k] = sum[k] * p.scale;
  V out;
  out.set(x);
  if (c < p.vecs) out.store(static_cast<T*>(p.dw) + row * p.cols + static_cast<int64_t>(c) * V::kN);
}

template <typename V>
__device__ __forceinline__ void store_part(const EmbedGradParams& p, float* part, int c, const float (&sum)[V::kN]) {
  if (c >= p.vecs) return;
#pragma unroll
  for (int k = 0; k < V::kN; ++k) part[static_cast<int64_t>(c) * V::kN + k] = sum[k];
}

// A CTA takes a stretch of 64 sorted tokens and 32 vectors of their rows, a warp eight of the tokens.
template <typename T, typename V>
__global__ void __launch_bounds__(32 * kGradWarps) embedding_sum_kernel(const EmbedGradParams p) {
  __shared__ float heads[kGradWarps][32 * V::kN];     // sums of the row that a warp begins in the middle of
  __shared__ int head_ends[kGradWarps];               // whether that row ends within the warp
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stretch = static_cast<int>(blockIdx.x / p.chunks), chunk = static_cast<int>(blockIdx.x) - stretch * p.chunks;
  const int base = stretch * kGradStretch + warp * kGradEach;
  const int c = chunk * 32 + lane;
  // lanes 0 .. 9: the tokens from the one before to the one behind; ids without a row come last
  const int place = base - 1 + lane;
  int2 token = make_int2(p.rows, 0);
  if (lane < kGradEach + 2 && place >= 0 && place < p.n) token = p.sorted[place];
  int row = __shfl_sync(0xffffffffu, token.x, 1);
  const bool any = row < p.rows;                      // (of the warp's tokens)
  const bool began = row == __shfl_sync(0xffffffffu, token.x, 0) && any;      // before the warp
  bool head = began;
  bool open = false;                                  // a row goes on behind the warp that did not begin before it
  float sum[V::kN];
#pragma unroll
  for (int k = 0; k < V::kN; ++k) sum[k] = 0.f;
  if (any) {
    const T* dy = static_cast<const T*>(p.dy) + static_cast<int64_t>(min(c, p.vecs - 1)) * V::kN;
    V v[kGradEach];
#pragma unroll
    for (int u = 0; u < kGradEach; ++u)      // (behind the last token: the first row of dY, which is not used)
      v[u].load(dy + static_cast<int64_t>(__shfl_sync(0xffffffffu, token.y, u + 1)) * p.cols);
#pragma unroll
    for (int u = 0; u < kGradEach; ++u) {
      const int next = __shfl_sync(0xffffffffu, token.x, u + 2);
      if (row < p.rows) {
        float f[V::kN];
        v[u].get(f);
#pragma unroll
        for (int k = 0; k < V::kN; ++k) sum[k] += f[k];
      }
      if (u + 1 == kGradEach || next != row) {      // (uniform: the warp's part of the row ends)
        const bool ends = next != row;
        if (row < p.rows) {
          if (head) {
#pragma unroll
            for (int k = 0; k < V::kN; ++k) heads[warp][k * 32 + lane] = sum[k];
            if (lane == 0) head_ends[warp] = ends;
          } else if (ends) {
            store_row<T, V>(p, row, c, sum);
          } else {
            open = true;
          }
        }
        if (ends) {
#pragma unroll
          for (int k = 0; k < V::kN; ++k) sum[k] = 0.f;
          head = false;
          row = next;
        }
      }
    }
  }
  __syncthreads();
  // What goes over warps: a row that begins in a warp is its to join; one that began before the CTA the first's.
  auto join = [&](int w) -> bool {      // adds heads from warp w on to where the row ends; whether it does
    for (; w < kGradWarps; ++w) {
#pragma unroll
      for (int k = 0; k < V::kN; ++k) sum[k] += heads[w][k * 32 + lane];
      if (head_ends[w]) return true;
    }
    return false;
  };
  float* part = p.part + static_cast<int64_t>(stretch) * 2 * p.cols;
  if (open) {
    if (join(warp + 1)) store_row<T, V>(p, row, c, sum);
    else store_part<V>(p, part + p.cols, c, sum);
  }
  if (warp == 0 && began) {
#pragma unroll
    for (int k = 0; k < V::kN; ++k) sum[k] = heads[0][k * 32 + lane];
    if (!head_ends[0]) join(1);
    store_part<V>(p, part, c, sum);
  }
}

// A row that goes over stretches, by the CTA of the one that it begins in, an eighth of them to a warp
template <typename T, typename V>
__global__ void __launch_bounds__(32 * kGradWarps) embedding_join_kernel(const EmbedGradParams p) {
  __shared__ float sums[kGradWarps][32 * V::kN];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stretch = static_cast<int>(blockIdx.x / p.chunks), chunk = static_cast<int>(blockIdx.x) - stretch * p.chunks;
  const int first = stretch * kGradStretch, behind = first + kGradStretch;
  if (behind >= p.n) return;
  const int row = p.sorted[behind].x, inside = p.sorted[behind - 1].x;
  const int before = first > 0 ? p.sorted[first - 1].x : -1;
  if (inside != row || row >= p.rows || before == row) return;
  const int c = chunk * 32 + lane;
  const int last = (p.ends[row] - 1) / kGradStretch, each = (last - stretch + kGradWarps) / kGradWarps;
  const int from = stretch + warp * each, to = min(last + 1, from + each);
  float sum[V::kN];
#pragma unroll
  for (int k = 0; k < V::kN; ++k) sum[k] = 0.f;
#pragma unroll 4
  for (int s = from; s < to; ++s) {
    const float* part = p.part + (static_cast<int64_t>(s) * 2 + (s == stretch ? 1 : 0)) * p.cols +
                        static_cast<int64_t>(min(c, p.vecs - 1)) * V::kN;
#pragma unroll
    for (int k = 0; k < V::kN; ++k) sum[k] += part[k];
  }
#pragma unroll
  for (int k = 0; k < V::kN; ++k) sums[warp][k * 32 + lane] = sum[k];
  __syncthreads();
  if (warp != 0) return;
#pragma unroll
  for (int k = 0; k < V::kN; ++k) {
#pragma unroll
    for (int w = 1; w < kGradWarps; ++w) sum[k] += sums[w][k * 32 + lane];
  }
  store_row<T, V>(p, row, c, sum);
}

// ------------------------------------------------------------------------ //
#define DISPATCH_DTYPE(dtype, ...)                                   \
  switch (dtype) {                                                   \
    case 0: { using T = __nv_bfloat16; __VA_ARGS__; break; }         \
    case 1: { using T = __half; __VA_ARGS__; break; }                \
    default: { using T = float; __VA_ARGS__; break; }                \
  }

template <typename T, typename Id>
static int lookup(const void* ids, const void* w, void* out, int64_t tokens, int64_t cols, int64_t rows,
                  int64_t row_stride, int64_t start, float scale, bool wide, cudaStream_t stream) {
  const int vecs = static_cast<int>(wide ? cols / RowVec<T>::kN : cols), parts = (vecs + 127) / 128;
  const int64_t blocks = (tokens * parts + 7) / 8;
  if (blocks > 0x7fffffff) return 1;
  count_launch();
  if (wide)
    embedding_fwd_kernel<T, RowVec<T>, Id><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
        static_cast<const Id*>(ids), static_cast<const T*>(w), static_cast<T*>(out), tokens, vecs, parts, rows,
        row_stride, start, scale);
  else
    embedding_fwd_kernel<T, RowOne<T>, Id><<<static_cast<unsigned>(blocks), 256, 0, stream>>>(
        static_cast<const Id*>(ids), static_cast<const T*>(w), static_cast<T*>(out), tokens, vecs, parts, rows,
        row_stride, start, scale);
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

static bool on16(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

int launch_embedding_fwd(const void* ids, bool ids64, const void* w, void* out, int64_t tokens, int64_t rows,
                         int64_t cols, int64_t row_stride, int64_t start, float scale, int dtype,
                         cudaStream_t stream) {
  if (tokens <= 0 || cols <= 0) return 0;
  if (cols > 0x7fffffff) return 1;
  int rc = 1;
  DISPATCH_DTYPE(dtype, {
    const bool wide = cols * sizeof(T) % 16 == 0 && row_stride * sizeof(T) % 16 == 0 && on16(w, out);
    if (ids64) rc = lookup<T, int64_t>(ids, w, out, tokens, cols, rows, row_stride, start, scale, wide, stream);
    else rc = lookup<T, int>(ids, w, out, tokens, cols, rows, row_stride, start, scale, wide, stream);
  });
  return rc;
}

EmbedGradPlan embedding_bwd_plan(int64_t tokens, int64_t rows, int64_t cols) {
  EmbedGradPlan p{};
  auto pad = [](int64_t n) { return (n + 31) / 32 * 32; };      // (128 bytes)
  p.sorted = pad(tokens);
  p.ends = pad(rows + 1);
  p.stretches = (tokens + kGradStretch - 1) / kGradStretch;
  p.part = p.stretches > 1 ? p.stretches * 2 * cols : 0;
  return p;
}

int launch_embedding_bwd(const void* ids, bool ids64, const void* dy, void* dw, int32_t* scratch,
                         const EmbedGradPlan& plan, int64_t tokens, int64_t rows, int64_t cols, int64_t start,
                         int64_t padding, float scale, int dtype, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if (tokens > kEmbedGradTokens || rows > 0x7ffffff0 || cols > 0x7fffffff) return 1;
  const size_t element = dtype == 2 ? 4 : 2;
  const bool wide = cols * element % 16 == 0 && on16(dy, dw);
  const int64_t vecs = wide ? cols * element / 16 : cols, chunks = (vecs + 31) / 32;
  const int64_t blocks = plan.stretches * chunks;
  if (blocks > 0x7fffffff) return 1;
  SortParams s{};
  s.ids = ids; s.start = start; s.padding = padding;
  s.n = static_cast<int>(tokens); s.rows = static_cast<int>(rows);
  for (int i = 0; i < 2; ++i) {
    s.key[i] = scratch + i * 2 * plan.sorted;
    s.pos[i] = s.key[i] + plan.sorted;
  }
  s.ends = scratch + 4 * plan.sorted;
  s.passes = 1;
  while (s.passes < 4 && (rows >> (8 * s.passes)) != 0) ++s.passes;
  s.sorted = reinterpret_cast<int2*>(s.key[s.passes & 1]);      // (over what the last pass has read)
  // a warp's stretch: two rounds of 32 tokens at least, then as many CTAs of the cluster as that leaves work for
  int ctas = 1;
  while (ctas < kSortCtas && static_cast<int64_t>(ctas) * kSortWarps * 64 < tokens) ctas *= 2;
  const int64_t warps = static_cast<int64_t>(ctas) * kSortWarps;
  s.stretch = static_cast<int>(((tokens + warps - 1) / warps + 31) / 32 * 32);
  const int64_t slice = s.stretch * static_cast<int64_t>(kSortWarps), bytes = slice * 16;
  const bool shared = bytes <= kSortSlices;
  if (slice > 0x7fffffff) return 1;
  s.slice = static_cast<int>(slice);
  s.dw = static_cast<uint8_t*>(dw);
  s.bytes = rows * cols * static_cast<int64_t>(element);
  // (128 KB of zeros to a CTA: clusters do not fill all SMs, and the last of several rounds costs little)
  const int64_t fillers = (s.bytes + ctas * 131072 - 1) / (ctas * 131072);
  if (ctas * (1 + fillers) > 0x7fffffff) return 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas * (1 + fillers)));
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  auto kernel = ids64 ? (shared ? embedding_sort_kernel<int64_t, true> : embedding_sort_kernel<int64_t, false>)
                      : (shared ? embedding_sort_kernel<int, true> : embedding_sort_kernel<int, false>);
  if (shared) {
    cfg.dynamicSmemBytes = static_cast<size_t>(bytes);
    // (of the current device; cheap beside a launch)
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSortSlices) != cudaSuccess)
      return 3;
  }
  count_launch();
  if (cudaLaunchKernelEx(&cfg, kernel, s) != cudaSuccess) { (void)cudaGetLastError(); return 4; }
  if (tokens == 0) return 0;

  EmbedGradParams g{};
  g.dy = dy; g.dw = dw;
  g.sorted = s.sorted;
  g.ends = s.ends;
  g.part = reinterpret_cast<float*>(scratch + 4 * plan.sorted + plan.ends);
  g.n = s.n; g.rows = s.rows; g.cols = cols; g.scale = scale;
  g.vecs = static_cast<int>(vecs);
  g.chunks = static_cast<int>(chunks);
#define EMBED_GRAD(KERNEL_, GRID_)                                                                \
  count_launch();                                                                                 \
  DISPATCH_DTYPE(dtype, {                                                                         \
    if (wide) KERNEL_<T, RowVec<T>><<<GRID_, 32 * kGradWarps, 0, stream>>>(g);                    \
    else KERNEL_<T, RowOne<T>><<<GRID_, 32 * kGradWarps, 0, stream>>>(g);                         \
  })
  EMBED_GRAD(embedding_sum_kernel, static_cast<unsigned>(blocks));
  if (plan.stretches > 1) { EMBED_GRAD(embedding_join_kernel, static_cast<unsigned>(blocks)); }
#undef EMBED_GRAD
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace slapo
