// The next token of each row of logits, from a given random number.
//
// A row's order: by logit from the largest, equals by index from the first.  top_k keeps the first k of it, top_p the
// shortest beginning whose mass reaches that share of what top_k kept, min_p what weighs that much of the largest.  The
// token is the first one kept, by index, at which the sum of weights passes the random number times their total.
//
// Weights are exp((x - largest) / temperature) in 64 bits, to 2^-44 of themselves, as multiples of 2^-42: sums of integers
// do not depend on their order, so that the same call gives the same token.
//
// Bound by latency: for few rows some five barriers of a cluster and twenty of a CTA; many rows come in waves of 74 in clusters of
// four CTAs, each of which waits the same, beside the arithmetic of the weights where top_p needs all.  HBM is read once.
// A cluster of CTAs has a row, a slice each in shared memory.  For top_k the largest logit of each thread is
// counted in bins of (largest - x) / temperature, an eighth of a factor 2 wide, and what comes before the end of the bin of the
// top_k-th goes to the first CTA, which sorts it and finishes the row by itself; the others leave.  top_p without top_k needs all
// weights in the bins; where what lies before the end of the bin in which its limit falls is at most kList tokens, the first CTA
// finishes as well.  Else that bin is narrowed by the bits of a key that orders logits and indices until at most kList
// are left, which are sorted, and the cluster sums weights once more.
// 8 x 50304 bf16 with top_k 50 and top_p 0.95 14.3 us (sorted by torch operators 438), 256 x 50272 fp32 61 (2250).
#include <cooperative_groups.h>

#include <cmath>

#include "common.cuh"
#include "generate.h"
#include "kernels.h"

namespace slapo {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512;
constexpr int kRanks = 8;            // CTAs of a cluster, at most
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 512;           // of an eighth in log2 of the weight; the last one has the rest
constexpr int kList = 1024;
constexpr int kIndexBits = 18;
static_assert(kSampleVocab == 1 << kIndexBits, "an index has as many bits");
constexpr double kOne = 4398046511104.0;      // 2^42

struct Shared {
  unsigned mass[3][kBins];             // 14, 14 and 15 bits of the weights: of 2^15 elements, no overflow
  unsigned count[kBins];
  double powers[64];
  unsigned long long list[kList], sorted[kList];       // places (see Slice::place)
  unsigned long long warp_mass[kWarps];
  unsigned warp_count[kWarps];
  // of the CTA, for the cluster to read
  unsigned long long cta_mass;
  unsigned long long border;       // of the elements that a limit keeps, the last one's place
  unsigned cta_top, listed, cta_first;
  unsigned rank_of[256];
  // of a decision in the CTA
  unsigned long long above_mass, total_mass;
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

// 2^(-i / 64)
struct Powers {
  double at[64];
};

struct Row {
  float top;
  double top_wide;
  double slope;           // log2(e) / temperature
  float bins;             // eight times that
  const double* powers;   // in shared memory
  // A float as a double, by its bits: the conversion runs at a quarter of the products' rate.  (0 and what is below the
  // normal numbers become some 2^-127.)
  static __device__ __forceinline__ double wide(float x) {
    const unsigned b = __float_as_uint(x);
    return __hiloint2double(static_cast<int>((b & 0x80000000u) | (((b & 0x7fffffffu) >> 3) + 0x38000000u)),
                            static_cast<int>(b << 29));
  }
  // exp(-(top - x) / temperature) as 2^-n 2^(-i / 64) e^-g, |g| <= ln 2 / 128, by a table and the series of e^-g up to
  // its fourth power (Tang, Table-driven implementation of the exponential function, ACM TOMS 15, 1989): off by 2^-44.  Eleven
  // operations in 64 bits; exp2() and the conversions around it took twice the time.
  __device__ __forceinline__ double fraction(unsigned key) const {
    const float x = logit_of(key);
    if (x == top) return 1.0;
    const double y = (top_wide - wide(x)) * slope;
    if (!(y < 44.0)) return 0.0;
    constexpr double kMagic = 6755399441055744.0;      // 1.5 2^52: what is added to it is rounded to an integer
    const double t = fma(y, 64.0, kMagic);
    const int n = __double2loint(t);
    const double r = fma(y, 64.0, -(t - kMagic));
    constexpr double kL = 0.010830424696249145;        // ln 2 / 64
    double e = fma(r, kL * kL * kL * kL / 24.0, -kL * kL * kL / 6.0);
    e = fma(r, e, kL * kL / 2.0);
    e = fma(r, e, -kL);
    e = fma(r, e, 1.0) * powers[n & 63];
    return __hiloint2double(__double2hiint(e) - ((n >> 6) << 20), __double2loint(e));
  }
  static __device__ __forceinline__ unsigned long long held(double fraction) {
    return static_cast<unsigned long long>(__double_as_longlong(fma(fraction, kOne, 4503599627370496.0))) & 0xfffffffffffffull;
  }
  __device__ __forceinline__ unsigned long long weight(unsigned key) const { return key == 0u ? 0ull : held(fraction(key)); }
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

// What a limit is: kept while the number of those before is less than `count`, or, by mass, their mass less than a
// share of all
struct Limit {
  bool by_mass;
  unsigned count;
  double share;
  unsigned long long mass;         // by mass: known, or 0: the share of all bins' masses
};
// less than the share of a mass: less than its ceiling, and the largest is kept
__device__ __forceinline__ unsigned long long mass_limit(double share, unsigned long long mass) {
  const double x = share * static_cast<double>(mass);
  const unsigned long long limit = __double2ull_ru(x > 0.0 ? x : 0.0);
  return limit == 0ull ? 1ull : limit;
}

// A row's slice in this CTA's shared memory, in a cluster of CTAs
struct Slice {
  cg::cluster_group cluster;
  Shared& s;
  unsigned* keys;
  int size, first;       // elements, and the index of the first one
  Row row;

  // larger logits first, then lower indices: unique
  __device__ __forceinline__ unsigned long long place(int i) const {
    return (static_cast<unsigned long long>(keys[i]) << kIndexBits) | static_cast<unsigned>(kSampleVocab - 1 - (first + i));
  }
  static __device__ __forceinline__ unsigned key_at(unsigned long long place) {
    return static_cast<unsigned>(place >> kIndexBits);
  }
  static __device__ __forceinline__ int index_at(unsigned long long place) {
    return kSampleVocab - 1 - static_cast<int>(place & (kSampleVocab - 1));
  }

  // Elements of a thread that goes through the slice in the order of the indices: an odd number, so that a warp's meet
  // every bank once
  __device__ __forceinline__ int stretch() const { return ((size + kThreads - 1) / kThreads) | 1; }

  // The least key whose bin is `bin` or one before, found by the lanes of each warp together: comparing keys costs a
  // fifth of a bin's number.  `top`: the row's largest key.
  __device__ __forceinline__ unsigned least_key(int bin, unsigned top) const {
    const unsigned lane = threadIdx.x & 31;
    auto in = [&](unsigned key) { return key >= top || (key != 0u && row.bin(key) <= bin); };      // (no keys above the top)
    unsigned base = 0u;                     // at most what is looked for, which is within 32 probes
#pragma unroll 1
    for (int shift = 27; shift > 0; shift -= 5) {
      const unsigned votes = __ballot_sync(0xffffffffu, in(base + (lane << shift)));
      const unsigned from = votes == 0u ? 32u : __ffs(votes) - 1u;
      if (from != 0u) base += (from - 1u) << shift;
    }
    // (six rounds of five bits and two more)
#pragma unroll 1
    for (int i = 0; i < 4; ++i, ++base)
      if (in(base)) break;
    return base;
  }

  // Sums over the cluster of a value of each CTA
  __device__ __forceinline__ unsigned long long everywhere(unsigned long long mine) {
    const unsigned long long w = warp_total(mine);
    __syncthreads();
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

  // A warp's and the block's prefix sums (exclusive), and the block's total
  template <typename V>
  __device__ __forceinline__ V before(V mine, V* warps, V& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    V until = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const V x = __shfl_up_sync(0xffffffffu, until, o);
      if (lane >= o) until += x;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = until;
    __syncthreads();
    V sum = until - mine;
    total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) sum += warps[w];
      total += warps[w];
    }
    return sum;
  }

  // Counts (and masses) of all CTAs' bins, and the bin in which a limit falls: the first whose beginning is below
  // the limit and whose end is not.  `count0`, `mass0`: before the first bin.  Returns through s.bin (-1: the limit is not
  // reached), s.above_*, s.in_bin.  The CTAs' bins can be written again after the cluster's next barrier.
  __device__ __forceinline__ void border_bin(const Limit& limit, unsigned count0, unsigned long long mass0, int bins) {
    cluster.sync();
    const unsigned ranks = cluster.num_blocks();
    unsigned n = 0;
    unsigned long long m = 0;
    if (static_cast<int>(threadIdx.x) < bins) {
      unsigned long long part[3] = {0ull, 0ull, 0ull};
      for (unsigned r = 0; r < ranks; ++r) {
        const Shared* o = cluster.map_shared_rank(&s, r);
        n += o->count[threadIdx.x];
        if (limit.by_mass) {
#pragma unroll
          for (int i = 0; i < 3; ++i) part[i] += o->mass[i][threadIdx.x];
        }
      }
      m = part[0] + (part[1] << 14) + (part[2] << 28);
    }
    if (threadIdx.x == 0) s.bin = -1;
    unsigned all;
    unsigned long long mass;
    const unsigned n_before = count0 + before(n, s.warp_count, all);
    unsigned long long m_before = 0ull;
    mass = 0ull;
    if (limit.by_mass) m_before = mass0 + before(m, s.warp_mass, mass);
    const unsigned long long most = limit.by_mass ? mass_limit(limit.share, limit.mass != 0ull ? limit.mass : mass) : 0ull;
    const bool here = n > 0 && (limit.by_mass ? m_before < most && m_before + m >= most
                                              : n_before < limit.count && n_before + n >= limit.count);
    if (threadIdx.x == 0) s.total_mass = mass;
    if (here) {
      s.bin = threadIdx.x;
      s.above_count = n_before;
      s.above_mass = m_before;
      s.in_bin = n;
    }
    __syncthreads();
  }

  __device__ __forceinline__ void clear_bins(bool masses) {
    for (int i = threadIdx.x; i < kBins; i += kThreads) {
      s.count[i] = 0u;
      if (masses) s.mass[0][i] = s.mass[1][i] = s.mass[2][i] = 0u;
    }
    __syncthreads();
  }
  __device__ __forceinline__ void add(int b, unsigned key, bool by_mass) {
    atomicAdd(&s.count[b], 1u);
    if (!by_mass) return;
    const unsigned long long w = row.weight(key);
    const unsigned part[3] = {static_cast<unsigned>(w) & 0x3fffu, static_cast<unsigned>(w >> 14) & 0x3fffu,
                              static_cast<unsigned>(w >> 28)};
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (part[i] != 0u) atomicAdd(&s.mass[i][b], part[i]);
  }
  // All elements in bins, and the limit's one
  __device__ __forceinline__ void count_bins(const Limit& limit) {
    clear_bins(limit.by_mass);
#pragma unroll 4
    for (int i = threadIdx.x; i < size; i += kThreads)
      if (keys[i] != 0u) add(row.bin(keys[i]), keys[i], limit.by_mass);
    border_bin(limit, 0u, 0ull, kBins);
  }

  // The place of the last element that a limit keeps (0: all), after count_bins
  __device__ __forceinline__ unsigned long long border(const Limit& limit) {
    const int bin = s.bin;
    if (bin < 0) return 0ull;
    unsigned n0 = s.above_count, left = s.in_bin;
    unsigned long long m0 = s.above_mass;
    Limit rest = limit;
    if (limit.by_mass && limit.mass == 0ull) rest.mass = s.total_mass;
    const unsigned long long most = limit.by_mass ? mass_limit(rest.share, rest.mass) : 0ull;
    // narrowed by the bits of the elements' places
    unsigned long long low = 0ull, mask = 0ull;
    for (int done = 0; left > kList && done < 32 + kIndexBits; done += 8) {
      cluster.sync();       // (all have read the bins)
      clear_bins(limit.by_mass);
      const int by = max(32 + kIndexBits - 8 - done, 0), width = min(32 + kIndexBits - done, 8);
      for (int i = threadIdx.x; i < size; i += kThreads) {
        if (keys[i] == 0u || row.bin(keys[i]) != bin) continue;
        const unsigned long long p = place(i);
        if ((p & mask) != low) continue;
        add((1 << width) - 1 - static_cast<int>((p >> by) & ((1u << width) - 1)), keys[i], limit.by_mass);  // larger ones first
      }
      border_bin(rest, n0, m0, 256);
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
      if (at < kList) home->list[at] = p;
    }
    cluster.sync();
    if (cluster.block_rank() == 0) {
      const int n = static_cast<int>(min(s.listed, static_cast<unsigned>(kList)));
      sort_list(n);
      unsigned long long w[2], mine = 0ull, all;
      const int i0 = 2 * threadIdx.x;
#pragma unroll
      for (int j = 0; j < 2; ++j) mine += w[j] = limit.by_mass && i0 + j < n ? row.weight(key_at(s.sorted[i0 + j])) : 0ull;
      unsigned long long sum = m0 + before(mine, s.warp_mass, all);
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        if (i0 + j < n && (limit.by_mass ? sum < most : n0 + i0 + j < limit.count)) atomicMin(&s.border, s.sorted[i0 + j]);
        sum += w[j];
      }
      __syncthreads();
    }
    cluster.sync();
    return home->border;
  }

  // s.sorted: the list's n places, the largest first.  Few of them are counted against one another, more sorted by
  // exchanges (bitonic).
  __device__ __forceinline__ void sort_list(int n) {
    int width = 2;
    while (width < n) width *= 2;
    if (width <= 256) {
      const int i = threadIdx.x & (width - 1), parts = kThreads / width;
      if (threadIdx.x < 256) s.rank_of[threadIdx.x] = 0u;
      __syncthreads();
      if (i < n) {
        const unsigned long long p = s.list[i];
        unsigned larger = 0;
        for (int j = threadIdx.x / width; j < n; j += parts) larger += s.list[j] > p ? 1u : 0u;
        atomicAdd(&s.rank_of[i], larger);
      }
      __syncthreads();
      if (static_cast<int>(threadIdx.x) < n) s.sorted[s.rank_of[threadIdx.x]] = s.list[threadIdx.x];
      __syncthreads();
      return;
    }
    for (int i = threadIdx.x; i < width; i += kThreads) s.sorted[i] = i < n ? s.list[i] : 0ull;
    for (int k = 2; k <= width; k *= 2) {
      for (int j = k / 2; j > 0; j /= 2) {
        __syncthreads();
        for (int i = threadIdx.x; i < width / 2; i += kThreads) {
          const int a = 2 * i - (i & (j - 1)), b = a + j;
          const unsigned long long x = s.sorted[a], y = s.sorted[b];
          if ((x < y) == ((a & k) == 0)) {
            s.sorted[a] = y;
            s.sorted[b] = x;
          }
        }
      }
    }
    __syncthreads();
  }

  // The row by the first CTA alone, from the elements with keys from `least` on: the token (in all threads of the first
  // CTA; -1 in others, which are done and may leave), or kMany in all CTAs where they are more than kList.
  // top_k: 0: all; mass: of all that top_k keeps, or 0: to be summed.
  static constexpr int kMany = -2;
  __device__ __forceinline__ int finish(unsigned least, unsigned top_k, double top_p, double min_p, unsigned long long mass,
                                        double u) {
    // Each CTA's into the first one's list, in the order of the indices: behind those of the CTAs before it, each thread a
    // stretch of the slice.
    const int t0 = threadIdx.x * stretch(), t1 = min(size, t0 + stretch());
    unsigned found = 0, all, lower = 0, n = 0;
#pragma unroll 8
    for (int i = t0; i < t1; ++i) found += keys[i] >= least ? 1u : 0u;
    unsigned to = before(found, s.warp_count, all);
    if (threadIdx.x == 0) s.listed = all;
    cluster.sync();           // (and all have read the others' bins)
    for (unsigned r = 0; r < cluster.num_blocks(); ++r) {
      const unsigned more = cluster.map_shared_rank(&s, r)->listed;
      if (r < cluster.block_rank()) lower += more;
      n += more;
    }
    if (n > kList) return kMany;
    Shared* home = cluster.map_shared_rank(&s, 0);
    if (found != 0u) {
      to += lower;
      for (int i = t0; i < t1; ++i)
        if (keys[i] >= least) home->list[to++] = place(i);
    }
    cluster.sync();           // (the list is whole, and nobody reads another's count any more)
    if (cluster.block_rank() != 0) return -1;
    sort_list(static_cast<int>(n));
    // the kept ones begin the sorted row
    const unsigned i0 = 2 * threadIdx.x;
    const unsigned in_k = top_k > 0 ? min(top_k, n) : n;
    unsigned long long w[2], sum[2], mine = 0ull, total;
    double share[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      share[j] = i0 + j < in_k ? row.fraction(key_at(s.sorted[i0 + j])) : 0.0;
      w[j] = i0 + j < in_k ? Row::held(share[j]) : 0ull;
      mine += w[j];
    }
    sum[0] = before(mine, s.warp_mass, total);
    sum[1] = sum[0] + w[0];
    const unsigned long long most = mass_limit(top_p, mass != 0ull ? mass : total);
    mine = 0ull;
    unsigned kept = 0;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      if (i0 + j < in_k && (i0 + j == 0 || ((sum[j] < most || !(top_p < 1.0)) && share[j] >= min_p))) {
        mine += w[j];
        ++kept;
      }
    }
    // (how many there are, and their mass, in one sum: at most 2^10 of them, and 2^52)
    unsigned long long both;
    before((mine << 11) | kept, s.warp_mass, both);
    const unsigned kept_all = static_cast<unsigned>(both) & 0x7ffu;
    total = both >> 11;
    const unsigned long long last = s.sorted[kept_all - 1];
    const double share_u = u * static_cast<double>(total);
    unsigned long long target = share_u > 0.0 ? __double2ull_rd(share_u) : 0ull;      // passed: more than it, more than its floor
    if (target >= total) target = total - 1ull;
    mine = 0ull;
#pragma unroll
    for (int j = 0; j < 2; ++j) mine += w[j] = i0 + j < n && s.list[i0 + j] >= last ? row.weight(key_at(s.list[i0 + j])) : 0ull;
    sum[0] = before(mine, s.warp_mass, total);
    sum[1] = sum[0] + w[0];
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (sum[j] <= target && target < sum[j] + w[j]) s.bin = index_at(s.list[i0 + j]);
    __syncthreads();
    return s.bin;
  }
};

template <typename T>
__global__ void __launch_bounds__(kThreads, 2) sample_kernel(const SampleCall c, int slice, const Powers powers) {
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
  int top_at = 0;
  constexpr int V = 16 / sizeof(T);
  const bool vectors = (reinterpret_cast<uintptr_t>(x + first) & 15) == 0;
  const int whole = vectors ? size / V * V : 0;
  if (threadIdx.x < 64) s.powers[threadIdx.x] = powers.at[threadIdx.x];
  constexpr int kAhead = 4;
  for (int i0 = threadIdx.x * V; i0 < whole; i0 += kThreads * V * kAhead) {
    uint4 raw[kAhead];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kThreads * V;
      if (i < whole) raw[k] = __ldcs(reinterpret_cast<const uint4*>(x + first + i));
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int i = i0 + k * kThreads * V;
      if (i >= whole) break;
      const T* v = reinterpret_cast<const T*>(&raw[k]);
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        uint4 w;
        w.x = key_of(static_cast<float>(v[j]));
        w.y = key_of(static_cast<float>(v[j + 1]));
        w.z = key_of(static_cast<float>(v[j + 2]));
        w.w = key_of(static_cast<float>(v[j + 3]));
        *reinterpret_cast<uint4*>(s_keys + i + j) = w;
        const unsigned four = max(max(w.x, w.y), max(w.z, w.w));
        if (four > top) {
          top = four;
          top_at = i + j + (w.x == four ? 0 : w.y == four ? 1 : w.z == four ? 2 : 3);
        }
      }
    }
  }
  for (int i = whole + threadIdx.x; i < size; i += kThreads) {
    const unsigned k = key_of(static_cast<float>(x[first + i]));
    s_keys[i] = k;
    if (k > top) {
      top = k;
      top_at = i;
    }
  }
  const unsigned mine_top = top;        // this thread's largest, the first of its equals at top_at
  top = __reduce_max_sync(0xffffffffu, top);
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
    if (mine_top == top && top != 0u) atomicMin(&home->cta_first, static_cast<unsigned>(first + top_at));
    cluster.sync();
    if (rank == 0 && threadIdx.x == 0) c.out[r] = top == 0u ? -1 : static_cast<int64_t>(s.cta_first);
    return;
  }
  Row row;
  row.top = logit_of(top);
  row.top_wide = static_cast<double>(row.top);
  row.powers = s.powers;
  row.slope = 1.4426950408889634 / static_cast<double>(temperature);
  row.bins = static_cast<float>(8.0 * row.slope);
  Slice at{cluster, s, s_keys, size, first, row};

  // the last place that is kept
  unsigned long long border = 0ull;
  const double least = static_cast<double>(fminf(min_p, 1.f));        // (the largest is kept, and its equals)
  bool binned = false;
  if (top_k > 0 && top_k < c.vocab) {
    const Limit limit{false, static_cast<unsigned>(top_k), 0.0, 0ull};
    // The threads' largest ones first: what comes before the end of the bin of their top_k-th has top_k tokens at least, and
    // few more, the largest being spread over the threads.  (All logits in bins: 256 x 50272 with top_k 50, now 58 us, took 7 us more.)
    at.clear_bins(false);
    if (mine_top != 0u) at.add(row.bin(mine_top), mine_top, false);
    at.border_bin(limit, 0u, 0ull, kBins);
    int token = Slice::kMany;
    if (s.bin >= 0) token = at.finish(at.least_key(s.bin, top), static_cast<unsigned>(top_k), top_p, least, 0ull, u);
    if (token != Slice::kMany) {
      if (rank == 0 && threadIdx.x == 0) c.out[r] = token;
      return;
    }
    cluster.sync();         // (all have read the bins)
    at.count_bins(limit);
    border = at.border(limit);
    binned = true;
  }
  if (top_p < 1.f) {
    Limit limit{true, 0u, static_cast<double>(top_p), 0ull};
    if (binned) {
      unsigned long long mine = 0ull;
      for (int i = threadIdx.x; i < size; i += kThreads)
        if (s_keys[i] != 0u && at.place(i) >= border) mine += row.weight(s_keys[i]);
      limit.mass = at.everywhere(mine);
    }
    at.count_bins(limit);
    if (!binned && s.bin >= 0 && s.above_count + s.in_bin <= kList) {
      const int token = at.finish(at.least_key(s.bin, top), 0u, top_p, least, s.total_mass, u);
      if (rank == 0 && threadIdx.x == 0) c.out[r] = token;
      return;
    }
    border = max(border, at.border(limit));
  }
  // each thread a stretch of the slice, in the order of the indices
  const int stretch = at.stretch(), t0 = threadIdx.x * stretch, t1 = min(size, t0 + stretch);
  const unsigned border_key = Slice::key_at(border);
  auto weight = [&](int i) -> unsigned long long {
    const unsigned k = s_keys[i];
    if (k < border_key || k == 0u || (k == border_key && at.place(i) < border)) return 0ull;
    const double f = row.fraction(k);
    return f >= least ? Row::held(f) : 0ull;
  };
  unsigned long long mine = 0ull, all;
#pragma unroll 4
  for (int i = t0; i < t1; ++i) mine += weight(i);
  unsigned long long before = at.before(mine, s.warp_mass, all);
  if (threadIdx.x == 0) s.cta_mass = all;
  cluster.sync();
  unsigned long long total = 0ull;
  for (int o = 0; o < ranks; ++o) {
    const unsigned long long m = cluster.map_shared_rank(&s, o)->cta_mass;
    if (o < rank) before += m;
    total += m;
  }
  cluster.barrier_arrive();       // (this CTA reads the others' shared memory no more)
  const double share = static_cast<double>(u) * static_cast<double>(total);
  unsigned long long target = share > 0.0 ? __double2ull_rd(share) : 0ull;
  if (target >= total) target = total - 1ull;
  // the thread in whose stretch it is passed; its warp goes through that together
  const unsigned here = __ballot_sync(0xffffffffu, before <= target && target < before + mine);
  if (here != 0u) {
    const int lane = threadIdx.x & 31, owner = __ffs(here) - 1;
    const int i1 = __shfl_sync(0xffffffffu, t1, owner);
    before = __shfl_sync(0xffffffffu, before, owner);
    for (int i0 = __shfl_sync(0xffffffffu, t0, owner); i0 < i1; i0 += 32) {
      const int i = i0 + lane;
      unsigned long long sum = i < i1 ? weight(i) : 0ull;
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
  cluster.barrier_wait();
}

template <typename T>
int launch(const SampleCall& c, cudaStream_t stream) {
  auto kernel = sample_kernel<T>;
  // A slice of the row for each CTA of a cluster: many CTAs where rows are few, and slices of which two CTAs' fit an SM (256 x
  // 50272 with settings of their own in 2 / 4 / 8 CTAs a row: 100 / 82 / 127 us, when the rest took longer).  Short rows are
  // not worth a cluster's barriers.
  int ranks = 1;
  while (ranks < kRanks && (c.rows * ranks * 2 <= 2 * sm_count() || (c.vocab + ranks - 1) / ranks > 16384)) ranks *= 2;
  if (c.vocab < 2048) ranks = 1;
  const int slice = ((c.vocab + ranks - 1) / ranks + 7) / 8 * 8;        // (vectors)
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
  static const Powers powers = [] {
    Powers p;
    for (int i = 0; i < 64; ++i) p.at[i] = std::exp2(-i / 64.0);
    return p;
  }();
  return cudaLaunchKernelEx(&config, kernel, c, slice, powers) == cudaSuccess ? 0 : 4;
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
