// The next token of each row of logits, from a given random number.
//
// A row's order: by logit from the largest, equals by index from the first.  top_k keeps the first k of it, top_p the
// shortest beginning whose mass reaches that share of what top_k kept, min_p what weighs that much of the largest.  The
// token is the first one kept, by index, at which the sum of weights passes the random number times their total.
//
// Weights are exp((x - largest) / temperature) in 64 bits, as multiples of 2^-42: sums of integers do not depend on their
// order, so that the same call gives the same token, and what falls to rounding are 2^-43 of the largest weight.
//
// Bound by latency for few rows and by the arithmetic of the weights for many; HBM is read once.  A cluster of CTAs has a
// row, a slice each in shared memory.  Logits are counted in bins of (largest - x) / temperature, an eighth of a
// factor 2 wide, with their weights where top_p asks for them; the bin in which a limit falls is narrowed by the bits of a key that orders
// logits and indices until at most kList are left, and those are compared with one another.  No sort.
#include <cooperative_groups.h>

#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 512;           // of an eighth in log2 of the weight; the last one has the rest
constexpr int kList = 1024;
constexpr int kIndexBits = 18;
static_assert(kSampleVocab == 1 << kIndexBits, "an index has as many bits");
constexpr double kOne = 4398046511104.0;      // 2^42

struct Shared {
  unsigned long long mass[kBins];
  unsigned count[kBins];
  unsigned long long list_key[kList], list_mass[kList];
  unsigned long long warp_mass[kWarps];
  unsigned warp_count[kWarps];
  // of the CTA, for the cluster to read
  unsigned long long cta_mass;
  unsigned long long border;       // of the elements that a limit keeps, the last one's key
  unsigned cta_top, listed, cta_first;
  // of a decision in the CTA
  unsigned long long above_mass;
  unsigned above_count, in_bin;
  int bin;
};

// larger logits, larger keys; 0: none (NaN, -infinity)
__device__ __forceinline__ unsigned key_of(float x) {
  if (!(x > -INFINITY)) return 0u;
  if (x == 0.f) x = 0.f;            // (-0 and 0 are equals)
  const unsigned b = __float_as_uint(x);
  return (b & 0x80000000u) != 0 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float logit_of(unsigned key) {
  return __uint_as_float((key & 0x80000000u) != 0 ? key ^ 0x80000000u : ~key);
}

struct Row {
  float top;
  double slope;           // log2(e) / temperature
  float bins;             // eight times that
  __device__ __forceinline__ double fraction(unsigned key) const {
    const float x = logit_of(key);
    return x == top ? 1.0 : exp2((static_cast<double>(x) - static_cast<double>(top)) * slope);
  }
  __device__ __forceinline__ unsigned long long weight(unsigned key) const {
    return key == 0u ? 0ull : __double2ull_rn(fraction(key) * kOne);
  }
  // monotone in the key, as each of its steps is
  __device__ __forceinline__ int bin(unsigned key) const {
    const float y = (top - logit_of(key)) * bins;
    return y < kBins - 1 ? static_cast<int>(y) : kBins - 1;      // (no number: infinities)
  }
};

__device__ __forceinline__ unsigned long long warp_total(unsigned long long v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// A row's slice in this CTA's shared memory, in a cluster of CTAs
struct Slice {
  cg::cluster_group cluster;
  Shared& s;
  unsigned* keys;
  int size, first;       // elements, and the index of the first one
  int vocab;
  Row row;

  // larger logits first, then lower indices: unique
  __device__ __forceinline__ unsigned long long place(int i) const {
    return (static_cast<unsigned long long>(keys[i]) << kIndexBits) | static_cast<unsigned>(kSampleVocab - 1 - (first + i));
  }

  // Sums over the cluster of a value of each CTA
  __device__ __forceinline__ unsigned long long everywhere(unsigned long long mine) {
    const unsigned long long w = warp_total(mine);
    if ((threadIdx.x & 31) == 0) s.warp_mass[threadIdx.x >> 5] = w;
    __syncthreads();
    if (threadIdx.x == 0) {
      unsigned long long sum = 0;
      for (int i = 0; i < kWarps; ++i) sum += s.warp_mass[i];
      s.cta_mass = sum;
    }
    cluster.sync();
    unsigned long long sum = 0;
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) sum += cluster.map_shared_rank(&s, r)->cta_mass;
    cluster.sync();
    return sum;
  }

  // Counts (and masses) of all CTAs' bins, and the bin in which a limit falls: the first whose beginning is below
  // the limit and whose end is not.  by_mass: kept while the mass before is less than `limit`; else the count.
  // `count0`, `mass0`: before the first bin.  Returns through s.bin (-1: the limit is not reached), s.above_*.
  __device__ __forceinline__ void border_bin(bool by_mass, unsigned long long limit, unsigned count0,
                                             unsigned long long mass0, int bins) {
    cluster.sync();
    const unsigned ranks = cluster.num_blocks();
    unsigned n = 0;
    unsigned long long m = 0;
    if (static_cast<int>(threadIdx.x) < bins) {
      for (unsigned r = 0; r < ranks; ++r) {
        const Shared* o = cluster.map_shared_rank(&s, r);
        n += o->count[threadIdx.x];
        m += o->mass[threadIdx.x];
      }
    }
    unsigned n_end = n;
    unsigned long long m_end = m;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned a = __shfl_up_sync(0xffffffffu, n_end, o);
      const unsigned long long b = __shfl_up_sync(0xffffffffu, m_end, o);
      if (lane >= o) {
        n_end += a;
        m_end += b;
      }
    }
    if (lane == 31) {
      s.warp_count[warp] = n_end;
      s.warp_mass[warp] = m_end;
    }
    if (threadIdx.x == 0) s.bin = -1;
    __syncthreads();
    n_end += count0;
    m_end += mass0;
    for (int w = 0; w < warp; ++w) {
      n_end += s.warp_count[w];
      m_end += s.warp_mass[w];
    }
    const unsigned n_before = n_end - n;
    const unsigned long long m_before = m_end - m;
    const bool here = n > 0 && (by_mass ? m_before < limit && m_end >= limit : n_before < limit && n_end >= limit);
    if (here) {
      s.bin = threadIdx.x;
      s.above_count = n_before;
      s.above_mass = m_before;
      s.in_bin = n;
    }
    cluster.sync();       // (all have read the others' bins)
  }

  __device__ __forceinline__ void clear_bins() {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.count[i] = 0u;
      s.mass[i] = 0ull;
    }
    __syncthreads();
  }

  // The key of the last element that a limit keeps (0: all): elements in order are kept while the mass (or number) of
  // those before is less than the limit.
  __device__ __forceinline__ unsigned long long border(bool by_mass, unsigned long long limit) {
    clear_bins();
    for (int i = threadIdx.x; i < size; i += kThreads) {
      if (keys[i] == 0u) continue;
      const int b = row.bin(keys[i]);
      atomicAdd(&s.count[b], 1u);
      const unsigned long long w = by_mass ? row.weight(keys[i]) : 0ull;
      if (w != 0ull) atomicAdd(&s.mass[b], w);
    }
    border_bin(by_mass, limit, 0u, 0ull, kBins);
    const int bin = s.bin;
    if (bin < 0) return 0ull;
    unsigned n0 = s.above_count, left = s.in_bin;
    unsigned long long m0 = s.above_mass;
    // narrowed by the bits of the elements' places
    unsigned long long low = 0ull, mask = 0ull;
    for (int done = 0; left > kList && done < 32 + kIndexBits; done += 8) {
      __syncthreads();
      clear_bins();
      const int by = max(32 + kIndexBits - 8 - done, 0), width = min(32 + kIndexBits - done, 8);
      for (int i = threadIdx.x; i < size; i += kThreads) {
        if (keys[i] == 0u || row.bin(keys[i]) != bin) continue;
        const unsigned long long p = place(i);
        if ((p & mask) != low) continue;
        const int b = (1 << width) - 1 - static_cast<int>((p >> by) & ((1u << width) - 1));      // larger ones first
        atomicAdd(&s.count[b], 1u);
        const unsigned long long w = by_mass ? row.weight(keys[i]) : 0ull;
        if (w != 0ull) atomicAdd(&s.mass[b], w);
      }
      border_bin(by_mass, limit, n0, m0, 256);
      n0 = s.above_count;
      m0 = s.above_mass;
      left = s.in_bin;
      low |= static_cast<unsigned long long>((1 << width) - 1 - s.bin) << by;
      mask |= static_cast<unsigned long long>((1 << width) - 1) << by;
    }
    // those that are left, in the first CTA
    Shared* home = cluster.map_shared_rank(&s, 0);
    if (threadIdx.x == 0) {
      s.listed = 0u;
      s.border = ~0ull;
    }
    cluster.sync();
    for (int i = threadIdx.x; i < size; i += kThreads) {
      if (keys[i] == 0u || row.bin(keys[i]) != bin) continue;
      const unsigned long long p = place(i);
      if ((p & mask) != low) continue;
      const unsigned at = atomicAdd(&home->listed, 1u);
      if (at < kList) {
        home->list_key[at] = p;
        home->list_mass[at] = row.weight(keys[i]);
      }
    }
    cluster.sync();
    if (cluster.block_rank() == 0) {
      const int n = static_cast<int>(min(s.listed, static_cast<unsigned>(kList)));
      for (int i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long p = s.list_key[i];
        unsigned before = n0;
        unsigned long long sum = m0;
        for (int j = 0; j < n; ++j) {
          if (s.list_key[j] > p) {
            ++before;
            sum += s.list_mass[j];
          }
        }
        if (by_mass ? sum < limit : before < limit) atomicMin(&s.border, p);
      }
    }
    cluster.sync();
    return home->border;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleCall c, int slice) {
  extern __shared__ __align__(16) unsigned s_keys[];
  __shared__ Shared s;
  cg::cluster_group cluster = cg::this_cluster();
  const int ranks = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
  const int64_t r = blockIdx.x / ranks;
  const T* x = static_cast<const T*>(c.logits) + r * c.row_stride;
  const int first = rank * slice, size = max(0, min(slice, c.vocab - first));
  const float temperature = c.temperature.rows != nullptr ? c.temperature.rows[r] : c.temperature.value;
  const float top_p = c.top_p.rows != nullptr ? c.top_p.rows[r] : c.top_p.value;
  const float min_p = c.min_p.rows != nullptr ? c.min_p.rows[r] : c.min_p.value;
  const int top_k = c.top_k.rows != nullptr ? c.top_k.rows[r] : c.top_k.value;
  const float u = c.uniform[r];

  unsigned top = 0u;
  for (int i = threadIdx.x; i < size; i += kThreads) {
    const unsigned k = key_of(static_cast<float>(x[first + i]));
    s_keys[i] = k;
    top = max(top, k);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((threadIdx.x & 31) == 0) s.warp_count[threadIdx.x >> 5] = top;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 0; w < kWarps; ++w) top = max(top, s.warp_count[w]);
    s.cta_top = top;
    s.cta_first = 0xffffffffu;
  }
  cluster.sync();
  top = 0u;
  for (int o = 0; o < ranks; ++o) top = max(top, cluster.map_shared_rank(&s, o)->cta_top);
  Shared* home = cluster.map_shared_rank(&s, 0);

  const bool greedy = !(temperature > 0.f) || top_k == 1;
  if (top == 0u || greedy) {          // nothing to take, or the first of the largest
    for (int i = threadIdx.x; i < size; i += kThreads)
      if (s_keys[i] == top) atomicMin(&home->cta_first, static_cast<unsigned>(first + i));
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) c.out[r] = top == 0u ? -1 : static_cast<int64_t>(s.cta_first);
    return;
  }
  Row row;
  row.top = logit_of(top);
  row.slope = 1.4426950408889634 / static_cast<double>(temperature);
  row.bins = static_cast<float>(8.0 * row.slope);
  Slice at{cluster, s, s_keys, size, first, c.vocab, row};

  // the last place that is kept
  unsigned long long border = 0ull;
  if (top_k > 0 && top_k < c.vocab) border = at.border(false, static_cast<unsigned long long>(top_k));
  const double least = static_cast<double>(min_p);
  if (top_p < 1.f) {
    unsigned long long mine = 0ull;
    for (int i = threadIdx.x; i < size; i += kThreads)
      if (s_keys[i] != 0u && at.place(i) >= border) mine += row.weight(s_keys[i]);
    const unsigned long long mass = at.everywhere(mine);
    const double share = static_cast<double>(top_p) * static_cast<double>(mass);
    unsigned long long limit = __double2ull_ru(share > 0.0 ? share : 0.0);      // less than the share: less than its ceiling
    if (limit == 0ull) limit = 1ull;                                            // (the largest is kept)
    border = max(border, at.border(true, limit));
  }
  // each warp's stretch of the slice, in the order of the indices
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int stretch = (size + kWarps - 1) / kWarps, w0 = warp * stretch, w1 = min(size, w0 + stretch);
  auto weight = [&](int i) -> unsigned long long {
    const unsigned k = s_keys[i];
    if (k == 0u || at.place(i) < border) return 0ull;
    const double f = row.fraction(k);
    return f >= least || k == top ? __double2ull_rn(f * kOne) : 0ull;
  };
  unsigned long long mine = 0ull;
  for (int i = w0 + lane; i < w1; i += 32) mine += weight(i);
  mine = warp_total(mine);
  __syncthreads();
  if (lane == 0) s.warp_mass[warp] = mine;
  __syncthreads();
  if (threadIdx.x == 0) {
    unsigned long long sum = 0;
    for (int w = 0; w < kWarps; ++w) sum += s.warp_mass[w];
    s.cta_mass = sum;
  }
  cluster.sync();
  unsigned long long before = 0ull, total = 0ull;
  for (int o = 0; o < ranks; ++o) {
    const unsigned long long m = cluster.map_shared_rank(&s, o)->cta_mass;
    if (o < rank) before += m;
    total += m;
  }
  const double share = static_cast<double>(u) * static_cast<double>(total);
  unsigned long long target = share > 0.0 ? __double2ull_rd(share) : 0ull;       // passed: more than it, more than its floor
  if (target >= total) target = total - 1ull;
  for (int w = 0; w < warp; ++w) before += s.warp_mass[w];
  if (before <= target && target < before + mine) {
    for (int i0 = w0; i0 < w1; i0 += 32) {
      const int i = i0 + lane;
      unsigned long long sum = i < w1 ? weight(i) : 0ull;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long a = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += a;
      }
      const unsigned passed = __ballot_sync(0xffffffffu, before + sum > target);
      if (passed != 0u) {
        if (lane == 0) c.out[r] = first + i0 + __ffs(passed) - 1;
        break;
      }
      before += __shfl_sync(0xffffffffu, sum, 31);
    }
  }
  cluster.sync();       // (the others have read this CTA's shared memory)
}

template <typename T>
int launch(const SampleCall& c, cudaStream_t stream) {
  auto kernel = sample_kernel<T>;
  // A slice of the row for each CTA of a cluster: many CTAs where rows are few, none of over 40 000 keys
  int ranks = 1;
  while (ranks < 8 && (c.rows * ranks * 2 <= 2 * sm_count() || (c.vocab + ranks - 1) / ranks > 40000)) ranks *= 2;
  if (c.vocab < 2048) ranks = 1;
  const int slice = (c.vocab + ranks - 1) / ranks;
  const int bytes = slice * 4;
  if (bytes > 190 * 1024) return 6;
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess || device < 0 || device >= 64) return 3;
  static bool configured[64] = {};
  if (!configured[device]) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 190 * 1024) != cudaSuccess) return 3;
    configured[device] = true;
  }
  if (c.rows * ranks > 0x7fffffff) return 5;
  cudaLaunchConfig_t config{};
  config.gridDim = dim3(static_cast<unsigned>(c.rows * ranks));
  config.blockDim = dim3(kThreads);
  config.dynamicSmemBytes = bytes;
  config.stream = stream;
  cudaLaunchAttribute attr{};
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = ranks;
  attr.val.clusterDim.y = 1;
  attr.val.clusterDim.z = 1;
  config.attrs = &attr;
  config.numAttrs = 1;
  count_launch();
  return cudaLaunchKernelEx(&config, kernel, c, slice) == cudaSuccess ? 0 : 4;
}

}  // namespace

int launch_sample(const SampleCall& c, cudaStream_t stream) {
  if (c.rows == 0) return 0;
  if (c.vocab < 1 || c.vocab > kSampleVocab) return 1;
  switch (c.dtype) {
    case 0: return launch<__nv_bfloat16>(c, stream);
    case 1: return launch<__half>(c, stream);
    case 2: return launch<float>(c, stream);
    default: return 2;
  }
}

}  // namespace slapo
