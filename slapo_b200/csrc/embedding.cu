// Token table: lookup with scaling, and its gradient by sorted tokens.
//   out[t] = scale W[id_t]          dW[v] = scale sum of dY[t] over the tokens t with id_t = v, in their order
// Ids outside of the table's rows [0, V) (of a shard: the other ranks' tokens) give rows of zeros and no gradient.
//
// The gradient of a table has few rows that anything is added to, some of them (frequent tokens, a padding id)
// from thousands of tokens.  Atomic additions would need an fp32 copy of the whole table, written three times, and
// their order would change the result from run to run.  Here tokens are sorted by id (a stable radix sort, so that
// a row's tokens stay in their order), each row of dW is written once, from registers, by threads that walk over its
// tokens, and rows with many tokens are summed in shares first: fixed stretches of the sorted order,
// so that the result is the same every time.
//
// Sorting: one cluster of up to eight CTAs with digits of eight bits; per pass each warp counts the digits of
// its stretch (match.any: equal digits of 32 tokens at a time), offsets are added up over the warps, the CTAs
// (distributed shared memory) and the digits, and the warps go over their stretches again and place them.
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

template <typename Id>
__device__ __forceinline__ int64_t table_row(const Id* ids, int64_t t, int64_t start, int64_t rows) {
  const int64_t row = static_cast<int64_t>(ids[t]) - start;
  return row >= 0 && row < rows ? row : -1;
}

// A CTA's threads walk over the vectors of all tokens, four at a time.
template <typename T, typename V, typename Id>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const Id* __restrict__ ids, const T* __restrict__ w,
                                                            T* __restrict__ out, int64_t tokens, int vecs,
                                                            int64_t rows, int64_t row_stride, int64_t start,
                                                            float scale) {
  constexpr int kUnroll = 4;
  const int64_t n = tokens * vecs, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i0 = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i0 < n; i0 += kUnroll * stride) {
    V v[kUnroll];
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = i0 + u * stride;
      v[u].zero();
      if (i < n) {
        const int64_t t = i / vecs, row = table_row(ids, t, start, rows);
        if (row >= 0) v[u].load(w + row * row_stride + (i - t * vecs) * V::kN);
      }
    }
#pragma unroll
    for (int u = 0; u < kUnroll; ++u) {
      const int64_t i = i0 + u * stride;
      if (i >= n) break;
      if (scale != 1.f) {
        float f[V::kN];
        v[u].get(f);
#pragma unroll
        for (int k = 0; k < V::kN; ++k) f[k] *= scale;
        v[u].set(f);
      }
      v[u].store(out + i * V::kN);
    }
  }
}

// ------------------------------------------------------------------------ //
constexpr int kSortWarps = 32, kSortThreads = 32 * kSortWarps, kDigits = 256;

struct SortParams {
  const void* ids;
  int64_t start, padding;       // first row of the table, id without a gradient (or one that no token has)
  int n, rows, passes;
  int stretch;                  // tokens of a warp, a multiple of 32
  int* key[2];                  // [n] each: ids by sorted order and ...
  int* pos[2];                  // ... where in `ids` they stand; the result is in [passes & 1 ^ 1]
  int2* range;                  // [rows + 1]: the sorted places [x, y) of each row's tokens
};

template <typename Id>
__global__ void __launch_bounds__(kSortThreads) embedding_sort_kernel(const SortParams p) {
  __shared__ int count[kSortWarps][kDigits];       // of a warp's digits, then where its next token of a digit goes
  __shared__ int total[kDigits];                   // of the CTA's digits
  __shared__ int before[kDigits];                  // tokens with smaller digits, or of earlier CTAs
  __shared__ int carry[8];
  cg::cluster_group cluster = cg::this_cluster();
  const int cta = static_cast<int>(cluster.block_rank()), ctas = static_cast<int>(cluster.num_blocks());
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int all = ctas * kSortThreads, me = cta * kSortThreads + threadIdx.x;
  for (int v = me; v <= p.rows; v += all) p.range[v] = make_int2(0, 0);

  const int64_t begin64 = static_cast<int64_t>(cta * kSortWarps + warp) * p.stretch;
  const int begin = begin64 < p.n ? static_cast<int>(begin64) : p.n;
  const int end = p.n - begin < p.stretch ? p.n : begin + p.stretch;
  for (int pass = 0; pass < p.passes; ++pass) {
    const int* src_key = p.key[(pass & 1) ^ 1];
    const int* src_pos = p.pos[(pass & 1) ^ 1];
    int* dst_key = p.key[pass & 1];
    int* dst_pos = p.pos[pass & 1];
    const int shift = 8 * pass;
    auto key_at = [&](int i) -> int {
      if (pass > 0) return __ldcg(src_key + i);      // (written by other SMs of the cluster)
      const int64_t id = static_cast<int64_t>(static_cast<const Id*>(p.ids)[i]);
      const int64_t row = id - p.start;
      return row >= 0 && row < p.rows && id != p.padding ? static_cast<int>(row) : p.rows;
    };
    for (int d = lane; d < kDigits; d += 32) count[warp][d] = 0;
    __syncwarp();
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool ok = i < end;
      const int d = ok ? (key_at(i) >> shift) & (kDigits - 1) : kDigits;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      if (ok && (same & ((1u << lane) - 1u)) == 0u) count[warp][d] += __popc(same);
      __syncwarp();
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      int sum = 0;
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) {
        const int c = count[w][threadIdx.x];
        count[w][threadIdx.x] = sum;
        sum += c;
      }
      total[threadIdx.x] = sum;
    }
    cluster.sync();
    if (threadIdx.x < kDigits) {
      int earlier = 0, sum = 0;
      for (int c = 0; c < ctas; ++c) {
        const int t = cluster.map_shared_rank(total, c)[threadIdx.x];
        if (c < cta) earlier += t;
        sum += t;
      }
      // exclusive sums over the digits: within the warp, then over the eight warps
      int inclusive = sum;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, inclusive, o);
        if (lane >= o) inclusive += x;
      }
      if (lane == 31) carry[warp] = inclusive;
      before[threadIdx.x] = inclusive - sum + earlier;
    }
    __syncthreads();
    if (threadIdx.x < kDigits) {
      int add = before[threadIdx.x];
      for (int w = 0; w < warp; ++w) add += carry[w];
#pragma unroll 8
      for (int w = 0; w < kSortWarps; ++w) count[w][threadIdx.x] += add;
    }
    __syncthreads();
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool ok = i < end;
      const int key = ok ? key_at(i) : 0;
      const int d = ok ? (key >> shift) & (kDigits - 1) : kDigits;
      const uint32_t same = __match_any_sync(0xffffffffu, d);
      const uint32_t ahead = same & ((1u << lane) - 1u);
      const int to = ok ? count[warp][d] + __popc(ahead) : 0;
      __syncwarp();
      if (ok && ahead == 0u) count[warp][d] = to + __popc(same);
      if (ok) {
        dst_key[to] = key;
        dst_pos[to] = pass > 0 ? __ldcg(src_pos + i) : i;
      }
      __syncwarp();
    }
    __threadfence();
    cluster.sync();      // (the totals have been read, and what was placed is visible)
  }
  const int* key = p.key[(p.passes & 1) ^ 1];
  for (int i = me; i < p.n; i += all) {
    const int k = __ldcg(key + i);
    if (i == 0 || __ldcg(key + i - 1) != k) p.range[k].x = i;
    if (i == p.n - 1 || __ldcg(key + i + 1) != k) p.range[k].y = i + 1;
  }
}

// Sums over a stretch of sorted places, four rows of dY on their way at a time
template <typename T, typename V>
__device__ __forceinline__ void add_rows(const T* __restrict__ dy, const int* __restrict__ pos, int from, int to,
                                         int64_t cols, int64_t col, float (&sum)[V::kN]) {
  constexpr int kAhead = 4;
  for (int i = from; i < to; i += kAhead) {
    V v[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      v[u].zero();
      if (i + u < to) v[u].load(dy + static_cast<int64_t>(pos[i + u]) * cols + col);
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      float f[V::kN];
      v[u].get(f);
#pragma unroll
      for (int k = 0; k < V::kN; ++k) sum[k] += f[k];
    }
  }
}

struct EmbedGradParams {
  const void* dy;
  void* dw;
  const int* pos;
  const int* key;
  const int2* range;
  float* part;          // [stretches][2][cols]: shares of rows with more than `share` tokens
  int n, share;
  int64_t rows, cols;
  int vecs;
  float scale;
};

// Shares of rows with many tokens: stretch s of `share` sorted places holds the end or the middle of one such row
// (from its first place on: share 0) and the beginning of another (share 1).
template <typename T, typename V>
__global__ void __launch_bounds__(128) embedding_shares_kernel(const EmbedGradParams p) {
  const int c = blockIdx.y * 128 + threadIdx.x;
  const int first = blockIdx.x * p.share, last = min(p.n, first + p.share);
  const int a = p.key[first], b = p.key[last - 1];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int row = which == 0 ? a : b;
    if (row >= p.rows || (which == 1 && b == a)) continue;
    const int2 r = p.range[row];
    if (r.y - r.x <= p.share || c >= p.vecs) continue;
    float sum[V::kN];
#pragma unroll
    for (int k = 0; k < V::kN; ++k) sum[k] = 0.f;
    add_rows<T, V>(static_cast<const T*>(p.dy), p.pos, max(first, r.x), min(last, r.y), p.cols,
                   static_cast<int64_t>(c) * V::kN, sum);
    float* to = p.part + (static_cast<int64_t>(blockIdx.x) * 2 + which) * p.cols + static_cast<int64_t>(c) * V::kN;
#pragma unroll
    for (int k = 0; k < V::kN; ++k) to[k] = sum[k];
  }
}

// Every row of dW, by threads that walk over the vectors of all rows
template <typename T, typename V>
__global__ void __launch_bounds__(256) embedding_rows_kernel(const EmbedGradParams p) {
  const int64_t n = p.rows * p.vecs, stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += stride) {
    const int64_t row = i / p.vecs, col = (i - row * p.vecs) * V::kN;
    const int2 r = p.range[row];
    V out;
    out.zero();
    if (r.y > r.x) {
      float sum[V::kN];
#pragma unroll
      for (int k = 0; k < V::kN; ++k) sum[k] = 0.f;
      if (r.y - r.x <= p.share) {
        add_rows<T, V>(static_cast<const T*>(p.dy), p.pos, r.x, r.y, p.cols, col, sum);
      } else {
        const int s0 = r.x / p.share, s1 = (r.y - 1) / p.share;
#pragma unroll 4
        for (int s = s0; s <= s1; ++s) {
          const int which = s == s0 && r.x > s0 * p.share ? 1 : 0;
          const float* from = p.part + (static_cast<int64_t>(s) * 2 + which) * p.cols + col;
#pragma unroll
          for (int k = 0; k < V::kN; ++k) sum[k] += from[k];
        }
      }
#pragma unroll
      for (int k = 0; k < V::kN; ++k) sum[k] *= p.scale;
      out.set(sum);
    }
    out.store(static_cast<T*>(p.dw) + row * p.cols + col);
  }
}

// ------------------------------------------------------------------------ //
#define DISPATCH_DTYPE(dtype, ...)                                   \
  switch (dtype) {                                                   \
    case 0: { using T = __nv_bfloat16; __VA_ARGS__; break; }         \
    case 1: { using T = __half; __VA_ARGS__; break; }                \
    default: { using T = float; __VA_ARGS__; break; }                \
  }

static int grid_for(int64_t threads, int per_sm) {
  const int64_t blocks = (threads + 255) / 256, cap = static_cast<int64_t>(sm_count()) * per_sm;
  return static_cast<int>(blocks < cap ? blocks : cap);
}

template <typename T, typename Id>
static void lookup(const void* ids, const void* w, void* out, int64_t tokens, int64_t cols, int64_t rows,
                   int64_t row_stride, int64_t start, float scale, bool wide, cudaStream_t stream) {
  const int vecs = static_cast<int>(wide ? cols / RowVec<T>::kN : cols);
  const int grid = grid_for((tokens * vecs + 3) / 4, 8);
  if (wide)
    embedding_fwd_kernel<T, RowVec<T>, Id><<<grid, 256, 0, stream>>>(
        static_cast<const Id*>(ids), static_cast<const T*>(w), static_cast<T*>(out), tokens, vecs, rows, row_stride,
        start, scale);
  else
    embedding_fwd_kernel<T, RowOne<T>, Id><<<grid, 256, 0, stream>>>(
        static_cast<const Id*>(ids), static_cast<const T*>(w), static_cast<T*>(out), tokens, vecs, rows, row_stride,
        start, scale);
}

static bool on16(const void* a, const void* b) {
  return ((reinterpret_cast<uintptr_t>(a) | reinterpret_cast<uintptr_t>(b)) & 15) == 0;
}

int launch_embedding_fwd(const void* ids, bool ids64, const void* w, void* out, int64_t tokens, int64_t rows,
                         int64_t cols, int64_t row_stride, int64_t start, float scale, int dtype,
                         cudaStream_t stream) {
  if (tokens <= 0 || cols <= 0) return 0;
  if (cols > 0x7fffffff) return 1;
  count_launch();
  DISPATCH_DTYPE(dtype, {
    const bool wide = cols * sizeof(T) % 16 == 0 && row_stride * sizeof(T) % 16 == 0 && on16(w, out);
    if (ids64) lookup<T, int64_t>(ids, w, out, tokens, cols, rows, row_stride, start, scale, wide, stream);
    else lookup<T, int>(ids, w, out, tokens, cols, rows, row_stride, start, scale, wide, stream);
  });
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

// Tokens of a share: some sqrt(n), so that a row of all tokens has about as many shares as a share has tokens.
static int share_of(int64_t n) {
  int s = 32;
  while (static_cast<int64_t>(s) * s < n && s < 1024) s *= 2;
  return s;
}

EmbedGradPlan embedding_bwd_plan(int64_t tokens, int64_t rows, int64_t cols) {
  EmbedGradPlan p{};
  auto pad = [](int64_t n) { return (n + 31) / 32 * 32; };      // (128 bytes)
  p.sorted = pad(tokens);
  p.range = pad(2 * (rows + 1));
  p.share = share_of(tokens);
  p.shares = tokens > p.share ? (tokens + p.share - 1) / p.share : 0;
  p.part = p.shares * 2 * cols;
  return p;
}

int launch_embedding_bwd(const void* ids, bool ids64, const void* dy, void* dw, int32_t* scratch,
                         const EmbedGradPlan& plan, int64_t tokens, int64_t rows, int64_t cols, int64_t start,
                         int64_t padding, float scale, int dtype, cudaStream_t stream) {
  if (rows <= 0 || cols <= 0) return 0;
  if (tokens > 0x7fffff00 || rows > 0x7ffffff0 || cols > 0x7fffffff || plan.shares > 0x7fffffff) return 1;
  SortParams s{};
  s.ids = ids; s.start = start; s.padding = padding;
  s.n = static_cast<int>(tokens); s.rows = static_cast<int>(rows);
  s.key[0] = scratch;
  s.key[1] = s.key[0] + plan.sorted;
  s.pos[0] = s.key[1] + plan.sorted;
  s.pos[1] = s.pos[0] + plan.sorted;
  s.range = reinterpret_cast<int2*>(s.pos[1] + plan.sorted);
  s.passes = 1;
  while (s.passes < 4 && (rows >> (8 * s.passes)) != 0) ++s.passes;
  // a warp's stretch: two rounds of 32 tokens at least, then as many CTAs of the cluster as that leaves work for
  int ctas = 1;
  while (ctas < 8 && static_cast<int64_t>(ctas) * kSortWarps * 64 < tokens) ctas *= 2;
  const int64_t warps = static_cast<int64_t>(ctas) * kSortWarps;
  s.stretch = static_cast<int>(((tokens + warps - 1) / warps + 31) / 32 * 32);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(ctas);
  cfg.blockDim = dim3(kSortThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ctas;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  count_launch();
  const cudaError_t err = ids64 ? cudaLaunchKernelEx(&cfg, embedding_sort_kernel<int64_t>, s)
                                : cudaLaunchKernelEx(&cfg, embedding_sort_kernel<int>, s);
  if (err != cudaSuccess) { (void)cudaGetLastError(); return 4; }

  EmbedGradParams g{};
  g.dy = dy; g.dw = dw;
  g.key = s.key[(s.passes & 1) ^ 1];
  g.pos = s.pos[(s.passes & 1) ^ 1];
  g.range = s.range;
  g.part = reinterpret_cast<float*>(scratch + 4 * plan.sorted + plan.range);
  g.n = s.n; g.share = plan.share; g.rows = rows; g.cols = cols; g.scale = scale;
  DISPATCH_DTYPE(dtype, {
    const bool wide = cols * sizeof(T) % 16 == 0 && on16(dy, dw);
    g.vecs = static_cast<int>(wide ? cols / RowVec<T>::kN : cols);
    if (plan.shares > 0) {
      const dim3 grid(static_cast<unsigned>(plan.shares), (g.vecs + 127) / 128);
      if (grid.y > 65535) return 1;
      count_launch();
      if (wide) embedding_shares_kernel<T, RowVec<T>><<<grid, 128, 0, stream>>>(g);
      else embedding_shares_kernel<T, RowOne<T>><<<grid, 128, 0, stream>>>(g);
    }
    count_launch();
    const int grid = grid_for(rows * g.vecs, 16);
    if (wide) embedding_rows_kernel<T, RowVec<T>><<<grid, 256, 0, stream>>>(g);
    else embedding_rows_kernel<T, RowOne<T>><<<grid, 256, 0, stream>>>(g);
  });
  return cudaGetLastError() == cudaSuccess ? 0 : 4;
}

}  // namespace slapo
